// Attention of drafted tokens over a cache of bf16 rows or of 8-bit codes.
//
// The T drafts of a sequence and the G query heads that share a KV head are T * G query rows over the same keys: rows
// t * G + g.  A CTA takes 16 of them (one tile of the matrix instruction) and a slice of the keys; its warps take blocks of 16
// keys in turn, each with a ring of its own that cp.async fills, so that nothing but the end of the slice joins them.  Slices
// of a (sequence, KV head) are joined by a second kernel.
//
// Formulas.  A score is s = scale q.k; with 8-bit rows k = ks kc and v = vs vc, where kc, vc are the codes: s = (scale ks) (q.kc),
// and the weight of a value's codes is w = exp(s - m) vs.  The running reference m of a row is the maximum of s + log vs, so
// w <= 1 whatever the scales; the sum of exp(s - m) is kept beside it in fp32.  Codes go through the products as fp16, which
// holds them exactly; so do the queries, after a row is multiplied by the power of two that brings its largest value to
// 2^8..2^9 (what is smaller than 2^-32 of that is lost, less than the products' own rounding in fp32).  w is multiplied
// by 2^14 first (in m), so that fp16 holds it down to 2^-38; its rounding to 11 bits is an eighth of bf16's.  With a bf16 cache
// queries and values are bf16 as they are and w is rounded to bf16, half a step of the result's own type.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <atomic>
#include <cstring>
#include "draft_api.h"
#include "../device/ptx.cuh"
#include "../runtime/host_common.h"

namespace mesh {
namespace draft {

constexpr int ROWS = 16;              // query rows of a tile
constexpr int KEYS = 16;              // keys of a block
constexpr int MOST_SPLITS = 64;

struct Args {
  const __nv_bfloat16* q; __nv_bfloat16* out; long long q_sb, q_st, o_sb, o_st;
  const uint8_t* k; const uint8_t* v; const float* k_scale; const float* v_scale;
  const int* pos; const int* counts; const long long* visible;
  int B, T, q_heads, kv_heads, max_seq, window, splits, tiles;
  float scale_log2;                   // scale * log2(e): exponentials are powers of two
  float* part; float* part_ml;        // [B * kv_heads * tiles][splits][ROWS][HD] and [..][ROWS] {m, l}
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <bool Q8>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (Q8)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two codes as fp16: the bytes of x (already code + 128) that `sel` puts under the exponent of 1024, minus 1152.
__device__ __forceinline__ uint32_t codes2(uint32_t x, uint32_t sel) {
  const uint32_t t = __byte_perm(x, 0x64646464u, sel);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&t), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ uint32_t pack16(bool half, float lo, float hi) {
  if (half) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// What the rows of a sequence see.
struct Seq {
  int pos, count, lo, hi;             // keys of any row: slots [lo, hi)
};
__device__ __forceinline__ Seq sequence(const Args& a, int b) {
  Seq s;
  s.pos = min(max(__ldg(a.pos + b), 0), a.max_seq);
  s.count = a.counts ? min(__ldg(a.counts + b), a.T) : a.T;
  s.hi = min(s.pos + max(s.count, 0), a.max_seq);
  s.lo = a.window > 0 ? max(0, s.pos - a.window + 1) : 0;          // the root's; its descendants see less
  return s;
}

template <int HD, bool Q8>
struct Cfg {
  static constexpr int RB = Q8 ? HD : 2 * HD;             // bytes of a row
  static constexpr int NC = RB / 16;                      // 16-byte chunks of a row
  static constexpr int STAGE = 2 * KEYS * RB + (Q8 ? 2 * KEYS * 4 : 0);
  static constexpr int WARPS = STAGE > 9000 ? 4 : 8;
  static constexpr int STAGES = (200 * 1024 / WARPS) / STAGE > 8 ? 8 : (200 * 1024 / WARPS) / STAGE;
  static constexpr int RING = WARPS * STAGES * STAGE;
  static constexpr int QB = ROWS * HD * 2;
  static constexpr int MERGE = WARPS * ROWS * (HD + 2) * 4;
  static constexpr int SMEM = QB + (RING > MERGE ? RING : MERGE);
  static constexpr int PER = Q8 ? 16 : 8;                 // values of a chunk
  static constexpr int VW = Q8 && HD == 64 ? 8 : PER;     // columns of V a lane takes at a time
};

// Chunk c of row r lies at chunk c ^ swz(r) of the row.  For keys the eight lanes of a phase read four chunks of two
// neighbouring rows, for values two chunks of every other row: both fall on eight different 16-byte banks.
template <int NC>
__device__ __forceinline__ int swz(int r) {
  return NC >= 8 ? (r & 6) ^ ((r & 1) << 2) : (r >> 1) & 3;
}

// Whether the 16 bf16 rows hold neither NaN nor infinity.
template <int RB>
__device__ __forceinline__ bool finite_rows(const uint8_t* rows, int lane) {
  bool bad = false;
  for (int i = lane; i < KEYS * RB / 16; i += 32) {
    const uint4 x = reinterpret_cast<const uint4*>(rows)[i];
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) bad |= (w[j] & 0x7f80u) == 0x7f80u || (w[j] & 0x7f800000u) == 0x7f800000u;
  }
  return !__any_sync(0xffffffffu, bad);
}

template <int HD, bool Q8>
__global__ void __launch_bounds__(Cfg<HD, Q8>::WARPS * 32, 1) attention_kernel(const __grid_constant__ Args a) {
  using C = Cfg<HD, Q8>;
  constexpr int RB = C::RB, NC = C::NC, STAGES = C::STAGES, PER = C::PER, VW = C::VW;
  constexpr int KI = HD / (4 * PER);                      // chunks of a key per lane
  constexpr int NT = HD / 8;                              // column tiles of the output
  extern __shared__ __align__(128) uint8_t smem[];
  uint4* q_s = reinterpret_cast<uint4*>(smem);            // [k step][lane]: operand A of the scores
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = lane >> 2, t4 = lane & 3;
  uint8_t* ring = smem + C::QB + warp * (STAGES * C::STAGE);
  const uint32_t ring_u = smem_u32(ring);
  griddep_launch_dependents();
  griddep_wait();

  const int tile = blockIdx.x, split = blockIdx.y;
  const int hk = blockIdx.z % a.kv_heads, b = blockIdx.z / a.kv_heads;
  const int G = a.q_heads / a.kv_heads;
  const Seq s = sequence(a, b);
  const int n_rows = min(max(s.count, 0) * G - tile * ROWS, ROWS);
  if (n_rows <= 0) return;                                // nothing of this tile is written: the joining kernel knows
  const int per = ((s.hi - s.lo + a.splits - 1) / a.splits + KEYS - 1) / KEYS * KEYS;
  const int k_lo = min(s.lo + split * per, s.hi), k_hi = min(k_lo + per, s.hi);
  const int blocks = (k_hi - k_lo + KEYS - 1) / KEYS;
  const long long base = ((long long)b * a.kv_heads + hk) * a.max_seq;
  const uint8_t* kp = a.k + base * RB;
  const uint8_t* vp = a.v + base * RB;

  auto fetch = [&](int block) {                           // this warp's block-th block into its ring
    const int at = block * C::WARPS + warp;
    if (at < blocks) {
      const int slot0 = k_lo + at * KEYS;
      const uint32_t st = ring_u + (block % STAGES) * C::STAGE;
#pragma unroll
      for (int i = 0; i < KEYS * NC / 32; ++i) {
        const int r = (i * 32 + lane) / NC, c = (i * 32 + lane) % NC;
        const long long src = (long long)min(slot0 + r, k_hi - 1) * RB + c * 16;
        const uint32_t dst = st + r * RB + ((c ^ swz<NC>(r)) << 4);
        cp_async16(dst, kp + src);
        cp_async16(dst + KEYS * RB, vp + src);
      }
      if (Q8) {
        const int slot = min(slot0 + (lane & 15), k_hi - 1);
        cp_async4(st + 2 * KEYS * RB + lane * 4, (lane < 16 ? a.k_scale : a.v_scale) + base + slot);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch(i);

  // ---- queries: row i of the tile as 4 consecutive values per lane and k step, in the order the keys' chunks have them
  float q_unit[2];                                        // what a row was divided by, times the scale
  {
    constexpr int STEPS = HD / 16;
    __shared__ float unit_s[ROWS];
    for (int i = warp; i < ROWS; i += C::WARPS) {         // a warp per row: its largest value
      float top = 0.f;
      const int r = tile * ROWS + i, t = r / G, h = hk * G + r % G;
      if (Q8 && i < n_rows) {
        const __nv_bfloat16* src = a.q + b * a.q_sb + t * a.q_st + (long long)h * HD;
        for (int d = lane; d < HD; d += 32) top = fmaxf(top, fabsf(__bfloat162float(src[d])));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      // the power of two that brings it to 2^8..2^9; bounded, so that neither it nor its inverse leaves fp32
      const int e = top > 0.f ? min(max(8 - ilogbf(top), -110), 110) : 0;
      if (lane == 0) unit_s[i] = Q8 ? ldexpf(1.f, e) : 1.f;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < STEPS * 32; i += C::WARPS * 32) {
      const int step = i / 32, l = i % 32, ln = l >> 2, lt = l & 3;
      const int col = ((step / (PER / 4)) * 4 + lt) * PER + (step % (PER / 4)) * 4;
      uint32_t w[2][2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = ln + 8 * j, r = tile * ROWS + row, t = r / G, h = hk * G + r % G;
        float f[4] = {0.f, 0.f, 0.f, 0.f};
        if (row < n_rows) {
          const __nv_bfloat16* src = a.q + b * a.q_sb + t * a.q_st + (long long)h * HD + col;
#pragma unroll
          for (int x = 0; x < 4; ++x) f[x] = __bfloat162float(src[x]) * unit_s[row];
        }
        w[j][0] = pack16(Q8, f[0], f[1]);
        w[j][1] = pack16(Q8, f[2], f[3]);
      }
      q_s[i] = make_uint4(w[0][0], w[1][0], w[0][1], w[1][1]);
    }
    __syncthreads();
    q_unit[0] = a.scale_log2 / unit_s[n];
    q_unit[1] = a.scale_log2 / unit_s[n + 8];
  }

  // ---- what this lane's two rows see
  int row_lo[2];
  unsigned long long vis[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int t = min((tile * ROWS + n + 8 * j) / G, a.T - 1);
    vis[j] = a.visible ? (unsigned long long)__ldg(a.visible + (long long)b * a.T + t) : t >= 63 ? ~0ull : (2ull << t) - 1;
    row_lo[j] = a.window > 0 ? max(0, s.pos + max(__popcll(vis[j]), 1) - a.window) : 0;
  }
  const int free_lo = a.window > 0 ? max(0, s.pos + 64 - a.window) : 0;      // from here to pos every row sees every key

  float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f};
  float o[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
  constexpr float LIFT = Q8 ? 14.f : 0.f;

  for (int block = 0; block * C::WARPS + warp < blocks; ++block) {
    cp_async_wait<STAGES - 2>();
    __syncwarp();
    fetch(block + STAGES - 1);                            // into the stage that the block before left
    const uint8_t* st = ring + (block % STAGES) * C::STAGE;
    const int slot0 = k_lo + (block * C::WARPS + warp) * KEYS;
    // ---- scores: two tiles of 8 keys
    float c[2][4];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < 4; ++j) c[x][j] = 0.f;
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      uint4 kx[2];
#pragma unroll
      for (int x = 0; x < 2; ++x)
        kx[x] = *reinterpret_cast<const uint4*>(st + (x * 8 + n) * RB + (((4 * i + t4) ^ swz<NC>(x * 8 + n)) << 4));
#pragma unroll
      for (int j = 0; j < PER / 4; ++j) {
        const uint4 qa = q_s[(i * (PER / 4) + j) * 32 + lane];
        const uint32_t qr[4] = {qa.x, qa.y, qa.z, qa.w};
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t w[4] = {kx[x].x, kx[x].y, kx[x].z, kx[x].w};
          if (Q8) {
            const uint32_t u = w[j] ^ 0x80808080u;
            mma<Q8>(c[x], qr, codes2(u, 0x4140), codes2(u, 0x4342));
          } else {
            mma<Q8>(c[x], qr, w[2 * j % 4], w[(2 * j + 1) % 4]);
          }
        }
      }
    }
    // ---- softmax of the lane's 2 rows x 4 keys
    const float* ks = reinterpret_cast<const float*>(st + 2 * KEYS * RB);
    const bool masked = slot0 < free_lo || slot0 + KEYS > min(s.pos, k_hi);
    float top[2] = {-CUDART_INF_F, -CUDART_INF_F}, vscale[4];
    uint32_t hidden = 0;                                  // a bit per score of the lane; a score of -inf need not be hidden
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int key = x * 8 + 2 * t4 + e, slot = slot0 + key;
        const float kscale = Q8 ? ks[key] : 1.f;
        vscale[2 * x + e] = Q8 ? ks[KEYS + key] : 1.f;
        const float up = Q8 ? fmaxf(lg2(vscale[2 * x + e]), -60.f) : 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float v = c[x][2 * j + e] * (q_unit[j] * kscale);
          if (masked) {
            const bool sees = slot < k_hi && (slot < s.pos ? slot >= row_lo[j] : (vis[j] >> (slot - s.pos)) & 1ull);
            if (!sees) {
              v = -CUDART_INF_F;
              hidden |= 1u << (4 * x + 2 * j + e);
            }
          }
          c[x][2 * j + e] = v;
          top[j] = fmaxf(top[j], v + up);
        }
      }
    float alpha[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 1));
      top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 2));
      const float now = fmaxf(m[j], top[j] - LIFT);
      alpha[j] = m[j] == now ? 1.f : ex2(m[j] - now);     // nothing seen before: 0
      m[j] = now;
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        o[i][0] *= alpha[0]; o[i][1] *= alpha[0];
        o[i][2] *= alpha[1]; o[i][3] *= alpha[1];
      }
      l[0] *= alpha[0];
      l[1] *= alpha[1];
    }
    uint32_t pa[4];
    float w_row[2][4];                                    // weights of the lane's keys
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float at = m[j] == -CUDART_INF_F ? 0.f : m[j];
        float p[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          p[e] = ex2(c[x][2 * j + e] - at);
          l[j] += p[e];
          if (Q8) p[e] *= vscale[2 * x + e];
          if (masked && (hidden >> (4 * x + 2 * j + e) & 1u)) p[e] = 0.f;      // a hidden key's scale may be anything
          if (!Q8) w_row[j][2 * x + e] = p[e];
        }
        pa[2 * x + j] = pack16(Q8, p[0], p[1]);
      }
    // ---- values: keys 2 t4, 2 t4 + 1 and those 8 further, VW columns at a time
    const uint8_t* vs = st + KEYS * RB;
    // Zero times a NaN or an infinity is not zero: where a block has keys that some row must not see, and such values, the
    // products are formed one by one.  (8-bit rows keep theirs in the scale, which is not looked at for a hidden key.)
    if (!Q8 && masked && !finite_rows<RB>(vs, lane)) {
#pragma unroll 1
      for (int key = 0; key < KEYS; ++key) {
        const int from = (lane & ~3) | ((key & 7) >> 1);
        float w[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float a0 = __shfl_sync(0xffffffffu, key < 8 ? w_row[j][0] : w_row[j][2], from);
          const float a1 = __shfl_sync(0xffffffffu, key < 8 ? w_row[j][1] : w_row[j][3], from);
          w[j] = key & 1 ? a1 : a0;
        }
        const uint32_t hid = __shfl_sync(0xffffffffu, hidden, from) >> (4 * (key >> 3) + (key & 1));
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int col = ((i / VW) * 8 + 2 * t4 + e) * VW + i % VW;
            const float x = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(vs + key * RB + (((col / 8) ^ swz<NC>(key)) << 4) + col % 8 * 2));
            if (!(hid & 1u)) o[i][e] += w[0] * x;
            if (!(hid & 4u)) o[i][2 + e] += w[1] * x;
          }
      }
      __syncwarp();
      continue;
    }
#pragma unroll
    for (int i = 0; i < NT / VW; ++i) {
      uint32_t w[4][4];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int r = 2 * t4 + (y & 1) + 8 * (y >> 1);
        if (Q8 && VW == 8) {
          const uint2 x = *reinterpret_cast<const uint2*>(vs + r * RB + (((n >> 1) ^ swz<NC>(r)) << 4) + (n & 1) * 8);
          w[y][0] = x.x; w[y][1] = x.y; w[y][2] = w[y][3] = 0;
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(vs + r * RB + (((8 * i + n) ^ swz<NC>(r)) << 4));
          w[y][0] = x.x; w[y][1] = x.y; w[y][2] = x.z; w[y][3] = x.w;
        }
      }
      if (Q8) {
#pragma unroll
        for (int y = 0; y < VW / 4; ++y) {
          const uint32_t r0 = w[0][y] ^ 0x80808080u, r1 = w[1][y] ^ 0x80808080u, r2 = w[2][y] ^ 0x80808080u, r3 = w[3][y] ^ 0x80808080u;
          const uint32_t lo01 = __byte_perm(r0, r1, 0x5140), hi01 = __byte_perm(r0, r1, 0x7362);
          const uint32_t lo23 = __byte_perm(r2, r3, 0x5140), hi23 = __byte_perm(r2, r3, 0x7362);
          mma<Q8>(o[i * VW + 4 * y], pa, codes2(lo01, 0x4140), codes2(lo23, 0x4140));
          mma<Q8>(o[i * VW + 4 * y + 1], pa, codes2(lo01, 0x4342), codes2(lo23, 0x4342));
          mma<Q8>(o[i * VW + 4 * y + 2], pa, codes2(hi01, 0x4140), codes2(hi23, 0x4140));
          mma<Q8>(o[i * VW + 4 * y + 3], pa, codes2(hi01, 0x4342), codes2(hi23, 0x4342));
        }
      } else {
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          mma<Q8>(o[i * VW + 2 * y], pa, __byte_perm(w[0][y], w[1][y], 0x5410), __byte_perm(w[2][y], w[3][y], 0x5410));
          mma<Q8>(o[i * VW + 2 * y + 1], pa, __byte_perm(w[0][y], w[1][y], 0x7632), __byte_perm(w[2][y], w[3][y], 0x7632));
        }
      }
    }
    __syncwarp();                                         // the stage is free for the next fetch
  }
  cp_async_wait<0>();

  // ---- join the warps: the ring's memory holds every warp's output
  __syncthreads();
  float* o_s = reinterpret_cast<float*>(smem + C::QB);    // [warp][row][HD]
  float* ml_s = o_s + C::WARPS * ROWS * HD;               // [warp][row]{m, l}
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    l[j] += __shfl_xor_sync(0xffffffffu, l[j], 1);
    l[j] += __shfl_xor_sync(0xffffffffu, l[j], 2);
    if (t4 == 0) {
      ml_s[(warp * ROWS + n + 8 * j) * 2] = m[j];
      ml_s[(warp * ROWS + n + 8 * j) * 2 + 1] = l[j];
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        o_s[(warp * ROWS + n + 8 * j) * HD + ((i / VW) * 8 + 2 * t4 + e) * VW + i % VW] = o[i][2 * j + e];
  }
  __syncthreads();
  const long long item = ((long long)(b * a.kv_heads + hk) * a.tiles + tile) * a.splits + split;
  for (int i = threadIdx.x; i < n_rows * (HD / 4); i += C::WARPS * 32) {
    const int row = i / (HD / 4), d = i % (HD / 4) * 4;
    float mm = -CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < C::WARPS; ++w) mm = fmaxf(mm, ml_s[(w * ROWS + row) * 2]);
    const float at = mm == -CUDART_INF_F ? 0.f : mm;
    float ll = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < C::WARPS; ++w) {
      const float wt = ex2(ml_s[(w * ROWS + row) * 2] - at);      // 0 for a warp that saw no key; its sum may be NaN
      ll += wt * ml_s[(w * ROWS + row) * 2 + 1];
      const float4 x = *reinterpret_cast<const float4*>(o_s + (w * ROWS + row) * HD + d);
      acc.x += wt * x.x; acc.y += wt * x.y; acc.z += wt * x.z; acc.w += wt * x.w;
    }
    if (a.splits > 1) {
      *reinterpret_cast<float4*>(a.part + (item * ROWS + row) * HD + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (item * ROWS + row) * 2) = make_float2(mm, ll);
    } else {
      const float inv = ll == 0.f ? 0.f : 1.f / ll;
      const int r = tile * ROWS + row;
      __nv_bfloat162 h[2] = {__floats2bfloat162_rn(acc.x * inv, acc.y * inv), __floats2bfloat162_rn(acc.z * inv, acc.w * inv)};
      __nv_bfloat162* dst = reinterpret_cast<__nv_bfloat162*>(a.out + b * a.o_sb + (r / G) * a.o_st + (long long)(hk * G + r % G) * HD + d);
      dst[0] = h[0];
      dst[1] = h[1];
    }
  }
}

// Joins the slices: a warp per query row.
template <int HD>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Args a) {
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31, G = a.q_heads / a.kv_heads;
  const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int rows = a.T * G;
  const int r = (int)(w % rows);
  const long long bh = w / rows;
  const int b = (int)(bh / a.kv_heads), hk = (int)(bh % a.kv_heads);
  if (b >= a.B) return;
  const Seq s = sequence(a, b);
  if (r >= s.count * G) return;
  const long long item = (bh * a.tiles + r / ROWS) * a.splits;
  const int row = r % ROWS;
  float ms[MOST_SPLITS / 32], ls[MOST_SPLITS / 32], mm = -CUDART_INF_F;
#pragma unroll
  for (int i = 0; i < MOST_SPLITS / 32; ++i) {
    const int sp = i * 32 + lane;
    float2 x = make_float2(-CUDART_INF_F, 0.f);
    if (sp < a.splits) x = __ldcg(reinterpret_cast<const float2*>(a.part_ml + ((item + sp) * ROWS + row) * 2));
    ms[i] = x.x; ls[i] = x.y;
    mm = fmaxf(mm, x.x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
  const float at = mm == -CUDART_INF_F ? 0.f : mm;
  float l = 0.f;
#pragma unroll
  for (int i = 0; i < MOST_SPLITS / 32; ++i) {
    ms[i] = ex2(ms[i] - at);
    l += ms[i] * ls[i];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  constexpr int PL = HD / 32;                             // columns of a lane
  float acc[PL];
#pragma unroll
  for (int i = 0; i < PL; ++i) acc[i] = 0.f;
#pragma unroll
  for (int i = 0; i < MOST_SPLITS / 32; ++i)
#pragma unroll 4
    for (int x = 0; x < min(32, a.splits - i * 32); ++x) {
      const float wt = __shfl_sync(0xffffffffu, ms[i], x);
      const float* p = a.part + ((item + i * 32 + x) * ROWS + row) * HD + lane * 2;
#pragma unroll
      for (int y = 0; y < PL / 2; ++y) {
        const float2 v = __ldcg(reinterpret_cast<const float2*>(p + y * 64));
        acc[2 * y] += wt * v.x;
        acc[2 * y + 1] += wt * v.y;
      }
    }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __nv_bfloat16* dst = a.out + b * a.o_sb + (r / G) * a.o_st + (long long)(hk * G + r % G) * HD + lane * 2;
#pragma unroll
  for (int y = 0; y < PL / 2; ++y)
    *reinterpret_cast<__nv_bfloat162*>(dst + y * 64) = __floats2bfloat162_rn(acc[2 * y] * inv, acc[2 * y + 1] * inv);
}

static int tiles_of(const MeshKvCache* c, const MeshDraftAttention* a) {
  return (a->T * (a->q_heads / c->kv_heads) + ROWS - 1) / ROWS;
}

// Slices per (sequence, KV head): enough that every SM has a CTA, at most one per 256 keys of the longest range.
static int splits_of(const MeshKvCache* c, const MeshDraftAttention* a) {
  if (a->splits > 0) return a->splits < MOST_SPLITS ? a->splits : MOST_SPLITS;
  const long long work = (long long)c->B * c->kv_heads * tiles_of(c, a);
  long long keys = c->max_seq;
  if (a->window > 0 && a->window + a->T < keys) keys = a->window + a->T;
  long long n = work > 0 ? sm_count() / work : 1;
  const long long most = (keys + 255) / 256;
  if (n > most) n = most;
  if (n > MOST_SPLITS) n = MOST_SPLITS;
  return n < 1 ? 1 : (int)n;
}

static int check(const MeshKvCache* c, const MeshDraftAttention* a) {
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return set_error(-2, "draft_attention: head_dim must be 64, 128 or 256");
  if (c->bits != 8 && c->bits != 16) return set_error(-2, "draft_attention: a cache of %d bits", c->bits);
  if (c->kv_heads < 1 || c->max_seq < 1 || a->q_heads < 1 || a->q_heads % c->kv_heads)
    return set_error(-2, "draft_attention: query heads must be a multiple of KV heads");
  if (a->T < 0 || a->T > 64) return set_error(-2, "draft_attention: at most 64 drafts per sequence");
  if (a->window < 0 || (a->window > 0 && a->window < a->T))
    return set_error(-2, "draft_attention: a window must be at least as long as the drafts");
  if (!(a->scale > 0.f)) return set_error(-2, "draft_attention: scale must be positive");
  if (((uintptr_t)c->k | (uintptr_t)c->v) % 16) return set_error(-2, "draft_attention: the cache must start on a multiple of 16 bytes");
  return 0;
}

template <class... P>
static cudaError_t launch(void (*kern)(P...), dim3 grid, int threads, int smem, void* stream, const Args& a) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a);
}

template <int HD, bool Q8>
static int run(const Args& p, void* stream) {
  using C = Cfg<HD, Q8>;
  static_assert(C::STAGES >= 3 && C::SMEM <= 227 * 1024, "ring of a warp");
  static std::atomic<unsigned long long> configured{0};   // a bit per device
  int dev = 0;
  MESH_CUDA_OK(cudaGetDevice(&dev));
  if (!(configured.load() >> (dev & 63) & 1)) {
    MESH_CUDA_OK(cudaFuncSetAttribute(attention_kernel<HD, Q8>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    configured.fetch_or(1ull << (dev & 63));
  }
  MESH_CUDA_OK(launch(attention_kernel<HD, Q8>, dim3(p.tiles, p.splits, p.B * p.kv_heads), C::WARPS * 32, C::SMEM, stream, p));
  if (p.splits > 1) {
    const long long rows = (long long)p.B * p.q_heads * p.T;
    MESH_CUDA_OK(launch(join_kernel<HD>, dim3((unsigned)((rows + 7) / 8)), 256, 0, stream, p));
  }
  return 0;
}

}  // namespace draft
}  // namespace mesh

extern "C" long long mesh_draft_attention_scratch(const MeshKvCache* c, const MeshDraftAttention* a) {
  using namespace mesh::draft;
  if (check(c, a)) return -1;
  const int splits = splits_of(c, a);
  if (splits <= 1) return 0;
  return (long long)c->B * c->kv_heads * tiles_of(c, a) * splits * ROWS * (c->head_dim + 2);
}

extern "C" int mesh_draft_attention(const MeshKvCache* c, const MeshDraftAttention* a, void* stream) {
  using namespace mesh;
  using namespace mesh::draft;
  if (int rc = check(c, a)) return rc;
  if (c->B == 0 || a->T == 0) return 0;
  if ((long long)c->B * c->kv_heads > 65535) return set_error(-2, "draft_attention: more than 65535 sequences times KV heads");
  if (((uintptr_t)a->q % 2) || ((uintptr_t)a->out % 4) || a->o_sb % 2 || a->o_st % 2)
    return set_error(-2, "draft_attention: rows of the output must start on a multiple of 4 bytes");
  Args p;
  memset(&p, 0, sizeof(p));
  p.q = (const __nv_bfloat16*)a->q; p.out = (__nv_bfloat16*)a->out;
  p.q_sb = a->q_sb; p.q_st = a->q_st; p.o_sb = a->o_sb; p.o_st = a->o_st;
  p.k = (const uint8_t*)c->k; p.v = (const uint8_t*)c->v; p.k_scale = c->k_scale; p.v_scale = c->v_scale;
  p.pos = a->pos; p.counts = a->counts; p.visible = a->visible;
  p.B = c->B; p.T = a->T; p.q_heads = a->q_heads; p.kv_heads = c->kv_heads; p.max_seq = c->max_seq; p.window = a->window;
  p.splits = splits_of(c, a);
  p.tiles = tiles_of(c, a);
  p.scale_log2 = a->scale * 1.4426950408889634f;
  if (p.splits > 1) {
    if (!a->scratch) return set_error(-2, "draft_attention: no scratch memory");
    const long long items = (long long)c->B * c->kv_heads * p.tiles * p.splits;
    p.part = a->scratch;
    p.part_ml = a->scratch + items * ROWS * c->head_dim;
  }
  switch (c->head_dim * 2 + (c->bits == 8)) {
    case 128: return run<64, false>(p, stream);
    case 129: return run<64, true>(p, stream);
    case 256: return run<128, false>(p, stream);
    case 257: return run<128, true>(p, stream);
    case 512: return run<256, false>(p, stream);
    default: return run<256, true>(p, stream);
  }
}
