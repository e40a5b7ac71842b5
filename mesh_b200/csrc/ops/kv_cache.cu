// Rows of a key/value cache, in bf16 or in 8-bit codes: written, read back, moved.
//
// A row of head_dim values of one token and head is stored as int8 codes c and one fp32 scale: with a = max |x|,
// scale = a / 127 and c = 127 x / a rounded to the nearest integer, ties to even.  One scale per row and not per group of
// columns: attention then multiplies a key's score and a value's probability by it once, and the codes themselves are the
// operands of the products.  A row that holds a NaN or an infinity gets the scale NaN: whoever reads it sees that.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cstring>
#include "draft_api.h"
#include "../device/ptx.cuh"
#include "../runtime/host_common.h"

namespace mesh {
namespace kv {

constexpr int THREADS = 256;

// Everything that is read here may have been written by the kernel before, which may still run when this one starts: plain loads behind
// the wait, and no __restrict__, with which the compiler would take the read-only path, that knows no such order.

// 8 consecutive bf16.  ALIGNED: the address is a multiple of 16 bytes.
template <bool ALIGNED>
__device__ __forceinline__ uint4 load8(const __nv_bfloat16* p) {
  if (ALIGNED) return *reinterpret_cast<const uint4*>(p);
  uint4 r;
  unsigned short* h = reinterpret_cast<unsigned short*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = reinterpret_cast<const unsigned short*>(p)[i];
  return r;
}

// A row's scale, from the bf16 bits of its largest magnitude.
__device__ __forceinline__ float scale_of(uint32_t top) { return top >= 0x7f80u ? __int_as_float(0x7fc00000) : __uint_as_float(top << 16) / 127.f; }

__device__ __forceinline__ unsigned long long pair(float lo, float hi) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Codes of eight values of a row whose largest magnitude has the bf16 bits `top`.
//
// The quotient 127 x / a has a numerator of 15 bits and a denominator of 8, so it is either exactly half way between two
// integers or further than 2^-17 of its size from there.  A product q with the rounded reciprocal is off by 2^-23 of its size, which
// is good enough except half way.  The remainder v - q a is exact, and q plus remainder times reciprocal is then the quotient itself,
// which fp32 holds, so the sum with 1.5 2^23 goes to the even neighbour.  Five operations for two values; a division, or a
// comparison for the half way ones, costs more than the memory does (16000 rows: 127 us).
__device__ __forceinline__ uint2 encode8(const uint4& x, uint32_t top) {
  if (top >= 0x7f80u || top == 0) return make_uint2(0, 0);              // a NaN or an infinity in the row
  const float a0 = __uint_as_float(top << 16);
  const float lift = a0 < 1e-18f ? 0x1p66f : 1.f;        // keeps 1 / a finite and the remainder in range; exact
  const float a = a0 * lift * 0x1p-7f, inv = __frcp_rn(a), f = lift * (127.f / 128.f);
  const unsigned long long a2 = pair(-a, -a), inv2 = pair(inv, inv), f2 = pair(f, f), magic = pair(12582912.f, 12582912.f);
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t code[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned long long v = mul2(pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u)), f2);      // x 127 / 128, exact
    const unsigned long long q = mul2(v, inv2);
    const unsigned long long t = add2(fma2(fma2(q, a2, v), inv2, q), magic);
    code[2 * i] = (uint32_t)t;                           // the low bits of each half are the nearest integer
    code[2 * i + 1] = (uint32_t)(t >> 32);
  }
  uint2 r;
  r.x = __byte_perm(__byte_perm(code[0], code[1], 0x0040), __byte_perm(code[2], code[3], 0x0040), 0x5410);
  r.y = __byte_perm(__byte_perm(code[4], code[5], 0x0040), __byte_perm(code[6], code[7], 0x0040), 0x5410);
  return r;
}

__device__ __forceinline__ uint32_t largest(const uint4& x) {
  const uint32_t m = 0x7fff7fffu;
  const uint32_t t = __vmaxu2(__vmaxu2(x.x & m, x.y & m), __vmaxu2(x.z & m, x.w & m));
  return max(t & 0xffffu, t >> 16);
}

struct Strides { long long b, t, h; };

// HD / 8 lanes share a row: 16 bytes of the key and 16 of the value each.  Memory bounds it with bf16 rows (4 sequences of 16000, 8 KV
// heads of 128: 79 us, 6.6 TB/s read and written); with 8-bit ones, 87 us, 4.6 TB/s, the trip of each row's maximum through its lanes
// and the codes' arithmetic stand between loads and stores.  Two rows a thread take 83 us there and, for the single token of a step,
// 2.9 instead of 2.2: one row a thread for all sizes (read_kernel has both forms).
template <int HD, bool Q8, bool ALIGNED>
__global__ void __launch_bounds__(THREADS) append_kernel(MeshKvCache c, const __nv_bfloat16* k, const __nv_bfloat16* v,
                                                         Strides ks, Strides vs, const int* pos,
                                                         const int* counts, int T) {
  constexpr int LANES = HD / 8;
  griddep_launch_dependents();
  griddep_wait();
  const unsigned row = blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES;       // (b, t, h), h fastest; fewer than 2^31
  const int lane = threadIdx.x % LANES;
  const unsigned bt = row / (unsigned)c.kv_heads, h = row - bt * c.kv_heads;
  const long long b = bt / (unsigned)T, t = bt - (unsigned)b * T;
  long long at = -1;
  uint4 kx = make_uint4(0, 0, 0, 0), vx = kx;
  if (b < c.B) {
    const long long slot = pos[b] + t;
    if (t < (counts ? counts[b] : T) && slot >= 0 && slot < c.max_seq) {
      at = (b * c.kv_heads + h) * c.max_seq + slot;
      kx = load8<ALIGNED>(k + b * ks.b + t * ks.t + h * ks.h + lane * 8);
      vx = load8<ALIGNED>(v + b * vs.b + t * vs.t + h * vs.h + lane * 8);
    }
  }
  if (!Q8) {
    if (at >= 0) {
      reinterpret_cast<uint4*>(c.k)[at * LANES + lane] = kx;
      reinterpret_cast<uint4*>(c.v)[at * LANES + lane] = vx;
    }
    return;
  }
  uint32_t top = largest(kx) | largest(vx) << 16;        // both rows at once
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
  const uint2 kc = encode8(kx, top & 0xffffu), vc = encode8(vx, top >> 16);
  const float scale = scale_of(lane & 1 ? top >> 16 : top & 0xffffu);
  if (at < 0) return;
  reinterpret_cast<uint2*>(c.k)[at * LANES + lane] = kc;
  reinterpret_cast<uint2*>(c.v)[at * LANES + lane] = vc;
  if (lane < 2) (lane ? c.v_scale : c.k_scale)[at] = scale;
}

// Eight codes times their row's scale, rounded once.
__device__ __forceinline__ uint4 decode8(const uint2& x, float scale) {
  uint4 r;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = i < 2 ? x.x : x.y;
    const int lo = (int)(signed char)(w >> (16 * (i & 1))), hi = (int)(signed char)(w >> (16 * (i & 1) + 8));
    h[i] = __floats2bfloat162_rn((float)lo * scale, (float)hi * scale);
  }
  return r;
}

// N rows a thread.  With 8-bit rows a thread has half of the bytes on their way that it has with bf16 ones, so where the grid is large,
// two rows: 8 KV heads of 128, 4 sequences of 16000, 62 us (6.4 TB/s read and written) instead of 70; with 500 rows each one row a
// thread takes half a microsecond less.  Rows of bf16 take as long either way.
constexpr long long TWO = 4096;                          // CTAs, of one row a thread
template <int HD, bool Q8, int N>
__global__ void __launch_bounds__(THREADS) read_kernel(MeshKvCache c, uint4* k_out, uint4* v_out,
                                                       const int* start, const int* counts, int T) {
  constexpr int LANES = HD / 8;
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x % LANES;
  uint4 kx[N], vx[N];
  float k_scale[N], v_scale[N];
  bool there[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const unsigned row = (blockIdx.x * N + i) * (THREADS / LANES) + threadIdx.x / LANES;
    const unsigned bt = row / (unsigned)c.kv_heads, h = row - bt * c.kv_heads;
    const long long b = bt / (unsigned)T, t = bt - (unsigned)b * T;
    there[i] = b < c.B;
    kx[i] = vx[i] = make_uint4(0, 0, 0, 0);
    k_scale[i] = v_scale[i] = 0.f;
    if (!there[i]) continue;
    const long long slot = (long long)start[b] + t;
    if (t >= (counts ? counts[b] : T) || slot < 0 || slot >= c.max_seq) continue;
    const long long at = (b * c.kv_heads + h) * c.max_seq + slot;
    if (Q8) {
      const uint2 kc = reinterpret_cast<const uint2*>(c.k)[at * LANES + lane];
      const uint2 vc = reinterpret_cast<const uint2*>(c.v)[at * LANES + lane];
      kx[i].x = kc.x; kx[i].y = kc.y;
      vx[i].x = vc.x; vx[i].y = vc.y;
      k_scale[i] = c.k_scale[at];
      v_scale[i] = c.v_scale[at];
    } else {
      kx[i] = reinterpret_cast<const uint4*>(c.k)[at * LANES + lane];
      vx[i] = reinterpret_cast<const uint4*>(c.v)[at * LANES + lane];
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (!there[i]) continue;
    const long long row = ((long long)blockIdx.x * N + i) * (THREADS / LANES) + threadIdx.x / LANES;
    k_out[row * LANES + lane] = Q8 ? decode8(make_uint2(kx[i].x, kx[i].y), k_scale[i]) : kx[i];
    v_out[row * LANES + lane] = Q8 ? decode8(make_uint2(vx[i].x, vx[i].y), v_scale[i]) : vx[i];
  }
}

constexpr int KEEP_MOST = 64, KEEP_LAYERS = 64;
struct KeepArgs {
  void* data[KEEP_LAYERS][2];
  float* scale[KEEP_LAYERS][2];
};

// One CTA moves the rows of one (layer, key or value, sequence, head): all of them into registers, a barrier, all out again,
// so an entry may read a slot that another one writes.  At most 64 rows of 512 bytes: 8 x 16 bytes a thread.  One launch for all
// layers, which is what it costs: 6 rows of 8 sequences in 30 layers 3.1 us, 64 rows (62 MB read and written) 9 us.
template <int ROW>                                       // bytes of a row
__global__ void __launch_bounds__(THREADS) keep_kernel(const __grid_constant__ KeepArgs a, const int* pos,
                                                       const int* path, const int* counts, int N,
                                                       int kv_heads, int max_seq) {
  constexpr int LANES = ROW / 16, PER = KEEP_MOST * LANES / THREADS > 0 ? KEEP_MOST * LANES / THREADS : 1;
  griddep_launch_dependents();
  griddep_wait();
  const int h = blockIdx.x % kv_heads, b = blockIdx.x / kv_heads, which = blockIdx.y & 1, layer = blockIdx.y >> 1;
  const long long p = pos[b];
  const int n = min(N, counts ? counts[b] : N);
  const long long base = ((long long)b * kv_heads + h) * max_seq;
  uint4* data = reinterpret_cast<uint4*>(a.data[layer][which]) + base * LANES;
  uint4 r[PER];
  long long to[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = i * THREADS + threadIdx.x, e = j / LANES;
    to[i] = -1;
    if (e >= n) continue;
    const int from = path[(long long)b * N + e];
    const long long src = p + from, dst = p + e;
    if (from < 0 || from == e || p < 0 || src >= max_seq || dst >= max_seq) continue;
    r[i] = data[src * LANES + j % LANES];
    to[i] = dst * LANES + j % LANES;
  }
  float* scale = a.scale[layer][which];
  float s = 0.f;
  long long s_to = -1;
  if (scale && (int)threadIdx.x < n) {
    const int from = path[(long long)b * N + threadIdx.x];
    const long long src = p + from, dst = p + threadIdx.x;
    if (from >= 0 && p >= 0 && src < max_seq && dst < max_seq) {
      s = scale[base + src];
      s_to = base + dst;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (to[i] >= 0) data[to[i]] = r[i];
  if (s_to >= 0) scale[s_to] = s;
}

static int check_cache(const MeshKvCache* c, const char* what) {
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return set_error(-2, "%s: head_dim must be 64, 128 or 256", what);
  if (c->bits != 8 && c->bits != 16) return set_error(-2, "%s: a cache of %d bits", what, c->bits);
  if (c->B < 0 || c->kv_heads < 1 || c->max_seq < 1) return set_error(-2, "%s: empty cache", what);
  if (((uintptr_t)c->k | (uintptr_t)c->v) % 16) return set_error(-2, "%s: the cache must start on a multiple of 16 bytes", what);
  return 0;
}

template <class... P, class... A>
static cudaError_t launch(void (*kern)(P...), dim3 grid, int threads, void* stream, A... args) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, P(args)...);
}

}  // namespace kv
}  // namespace mesh

extern "C" int mesh_kv_append(const MeshKvCache* c, const void* k, const void* v, long long k_sb, long long k_st, long long k_sh,
                              long long v_sb, long long v_st, long long v_sh, const int* pos, const int* counts, int T, void* stream) {
  using namespace mesh;
  if (int rc = kv::check_cache(c, "kv_append")) return rc;
  if (c->B == 0 || T <= 0) return 0;
  const int lanes = c->head_dim / 8, per = kv::THREADS / lanes;
  const long long rows = (long long)c->B * T * c->kv_heads, blocks = (rows + per - 1) / per;
  if (rows + per > 0x7fffffffll) return set_error(-2, "kv_append: too many rows for one call");
  const bool aligned = !((((uintptr_t)k | (uintptr_t)v) % 16) || ((k_sb | k_st | k_sh | v_sb | v_st | v_sh) % 8));
  const kv::Strides ks = {k_sb, k_st, k_sh}, vs = {v_sb, v_st, v_sh};
  const dim3 grid((unsigned)blocks);
#define MESH_APPEND(HD)                                                                                                          \
  MESH_CUDA_OK(kv::launch(c->bits == 8 ? (aligned ? kv::append_kernel<HD, true, true> : kv::append_kernel<HD, true, false>)         \
                                       : (aligned ? kv::append_kernel<HD, false, true> : kv::append_kernel<HD, false, false>),      \
                          grid, kv::THREADS, stream, *c, (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, ks, vs, pos, counts, T))
  switch (c->head_dim) {
    case 64: MESH_APPEND(64); break;
    case 128: MESH_APPEND(128); break;
    default: MESH_APPEND(256); break;
  }
#undef MESH_APPEND
  return 0;
}

extern "C" int mesh_kv_read(const MeshKvCache* c, void* k_out, void* v_out, const int* start, const int* counts, int T, void* stream) {
  using namespace mesh;
  if (int rc = kv::check_cache(c, "kv_read")) return rc;
  if (c->B == 0 || T <= 0) return 0;
  if (((uintptr_t)k_out | (uintptr_t)v_out) % 16) return set_error(-2, "kv_read: the results must start on a multiple of 16 bytes");
  const int per = kv::THREADS / (c->head_dim / 8);
  const long long rows = (long long)c->B * T * c->kv_heads;
  long long blocks = (rows + per - 1) / per;
  const bool two = c->bits == 8 && blocks >= kv::TWO;
  if (two) blocks = (blocks + 1) / 2;
  if (rows + 2 * per > 0x7fffffffll) return set_error(-2, "kv_read: too many rows for one call");
  const dim3 grid((unsigned)blocks);
#define MESH_READ(HD)                                                                                                          \
  MESH_CUDA_OK(kv::launch(two ? kv::read_kernel<HD, true, 2> : c->bits == 8 ? kv::read_kernel<HD, true, 1> : kv::read_kernel<HD, false, 1>, \
                          grid, kv::THREADS, stream, *c, (uint4*)k_out, (uint4*)v_out, start, counts, T))
  switch (c->head_dim) {
    case 64: MESH_READ(64); break;
    case 128: MESH_READ(128); break;
    default: MESH_READ(256); break;
  }
#undef MESH_READ
  return 0;
}

extern "C" int mesh_kv_keep(const MeshKvCache* caches, int n, const int* pos, const int* path, const int* counts, int N, void* stream) {
  using namespace mesh;
  if (N > kv::KEEP_MOST) return set_error(-2, "kv_keep: at most %d rows of a sequence", kv::KEEP_MOST);
  for (int i = 0; i < n; ++i) {
    if (int rc = kv::check_cache(caches + i, "kv_keep")) return rc;
    if (caches[i].B != caches->B || caches[i].kv_heads != caches->kv_heads || caches[i].max_seq != caches->max_seq ||
        caches[i].head_dim != caches->head_dim || caches[i].bits != caches->bits)
      return set_error(-2, "kv_keep: the caches of a group have one geometry");
  }
  if (n < 1 || N < 1 || caches->B == 0) return 0;
  for (int first = 0; first < n; first += kv::KEEP_LAYERS) {
    const int m = n - first < kv::KEEP_LAYERS ? n - first : kv::KEEP_LAYERS;
    kv::KeepArgs a;
    memset(&a, 0, sizeof(a));
    for (int i = 0; i < m; ++i) {
      const MeshKvCache& c = caches[first + i];
      a.data[i][0] = c.k; a.data[i][1] = c.v;
      a.scale[i][0] = c.bits == 8 ? c.k_scale : nullptr;
      a.scale[i][1] = c.bits == 8 ? c.v_scale : nullptr;
    }
    const int row = caches->head_dim * caches->bits / 8;
    auto kern = row == 64 ? kv::keep_kernel<64> : row == 128 ? kv::keep_kernel<128> : row == 256 ? kv::keep_kernel<256> : kv::keep_kernel<512>;
    MESH_CUDA_OK(kv::launch(kern, dim3((unsigned)(caches->B * caches->kv_heads), (unsigned)(2 * m)), kv::THREADS, stream, a, pos, path, counts, N,
                            caches->kv_heads, caches->max_seq));
  }
  return 0;
}
