// Penalties for repeated tokens, biases and a grammar mask on logits, and the greedy choice among what is left, in one pass.
//
// A row's vocabulary is cut over the CTAs of a cluster, a CTA's share into pieces of at most 16384 ids.  Before a piece is
// streamed, a bit per id is set for every id of the history and the bias list, and the logits of the listed ids are fetched.  Eight
// warps then stream the logits and treat the listed ids like forbidden ones, while two gather what the lists say: sums of bits before each
// word of the bitmap number the listed ids, and a word per listed id holds how often it was generated (16 bits),
// whether it stands in the history at all (1 bit) and 1 + its last place in the bias list (15 bits).  When both are done the
// adjusted logits of the listed ids are put in.  Shared memory grows with the lists, not with the vocabulary.
//
// 128 rows of 262144 fp32 with a mask, the result kept: 50.6 us without lists (5.4 TB/s), 65 with some 2300 listed ids a row: the trips
// to memory before a stream begins, which other CTAs' streams hide only in part.  With the penalties' arithmetic in the
// stream, where one lane of most warps has a listed id, 76 us; with the words gathered before the stream, four CTAs
// of 512 threads to an SM, 71.  Sixteen CTAs a row where they pay: 8 rows of 262144, the token alone, 6.2 us against 7.5 with eight.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <atomic>
#include <cstring>
#include "draft_api.h"
#include "../device/ptx.cuh"
#include "../runtime/host_common.h"

namespace mesh {
namespace constrain {

constexpr int STREAM = 256, LIST = 64, THREADS = STREAM + LIST, WARPS = THREADS / 32;
constexpr int PIECE = 16384, WORDS = PIECE / 32, WPT = WORDS / LIST;       // bitmap words of a list thread
constexpr int AT_ONCE = 2;                                  // vectors of a thread under way
constexpr int LISTS = WORDS * 4 + WORDS * 2, ENTRY = 4 + 4 + 2;            // bytes: bitmap and numbers; a listed id
constexpr int ONE_CTA_VOCAB = 4096, EIGHT_CTA_VOCAB = 65536;
constexpr uint32_t COUNT = 0xffffu, SEEN = 0x10000u;
constexpr int BIAS_SHIFT = 17;

__device__ __forceinline__ void better(float& v, int& i, float ov, int oi) {
  if (ov > v || (ov == v && oi < i)) { v = ov; i = oi; }
}

template <bool HALF>
__device__ __forceinline__ float load1(const void* row, int c) {
  return HALF ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[c]) : reinterpret_cast<const float*>(row)[c];
}
template <bool HALF>
__device__ __forceinline__ void store1(void* row, int c, float v) {
  if (HALF) reinterpret_cast<__nv_bfloat16*>(row)[c] = __float2bfloat16_rn(v);
  else reinterpret_cast<float*>(row)[c] = v;
}
// 16 bytes of logits: 4 fp32 or 8 bf16.
template <bool HALF> struct Vec { static constexpr int N = HALF ? 8 : 4; };
template <bool HALF>
__device__ __forceinline__ void widen(const uint4& x, float (&f)[Vec<HALF>::N]) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (HALF) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      f[i] = __uint_as_float(w[i]);
    }
}
template <bool HALF>
__device__ __forceinline__ uint4 narrow(const float (&f)[Vec<HALF>::N]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (HALF) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      w[i] = __float_as_uint(f[i]);
    }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

struct Row {
  const int* history; int hist, prompt;
  const int* bias_ids; const float* bias; int nbias;
  float repetition, presence, frequency;
  bool repeats;
};

__device__ __forceinline__ float adjust(float x, uint32_t word, const Row& r) {
  const uint32_t n = word & COUNT;
  if (r.repeats && (n || (word & SEEN))) x = x > 0.f ? __fdiv_rn(x, r.repetition) : __fmul_rn(x, r.repetition);
  if (n) x = __fsub_rn(__fsub_rn(x, __fmul_rn(r.frequency, (float)n)), r.presence);
  if (word >> BIAS_SHIFT) x = __fadd_rn(x, r.bias[(word >> BIAS_SHIFT) - 1]);
  return x;
}

__device__ __forceinline__ int number_of(const uint32_t* listed, const uint16_t* number, unsigned id) {
  return number[id >> 5] + __popc(listed[id >> 5] & ((1u << (id & 31)) - 1));
}

// f(i, place in the piece) for the entries of a list that lie in the piece, by threads thread of threads: several loads at a
// time, a trip to L2 for all of them and not for each.
template <class F>
__device__ __forceinline__ void each(const int* list, int n, unsigned first, unsigned size, int thread, int threads, F f) {
  for (int i0 = thread; i0 < n; i0 += 4 * threads) {
    unsigned id[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) id[i] = i0 + i * threads < n ? (unsigned)list[i0 + i * threads] - first : ~0u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (id[i] < size) f(i0 + i * threads, id[i]);
  }
}
__device__ __forceinline__ void list_sync() { asm volatile("bar.sync 1, %0;" ::"n"(LIST) : "memory"); }

template <bool HALF, int CTAS>
__global__ void __launch_bounds__(THREADS, 6) constrain_kernel(const __grid_constant__ MeshLogits a, int vectors, int entries) {
  constexpr int N = Vec<HALF>::N, STEP = STREAM * N;      // ids of a vector per stream thread
  extern __shared__ __align__(16) uint8_t smem[];
  uint32_t* listed = reinterpret_cast<uint32_t*>(smem);   // a bit per id of the piece
  uint16_t* number = reinterpret_cast<uint16_t*>(listed + WORDS);      // listed ids before each word
  uint32_t* table = reinterpret_cast<uint32_t*>(number + WORDS);       // [entries] by number: the word of a listed id
  float* raw = reinterpret_cast<float*>(table + entries);              // [entries] in any order: its logit
  uint16_t* ids = reinterpret_cast<uint16_t*>(raw + entries);          // ... and its place in the piece
  __shared__ int warp_sum[LIST / 32], n_listed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_launch_dependents();
  if (CTAS > 1) cluster_arrive_relaxed();                 // waited for before the store into the first CTA's shared memory
  griddep_wait();
  const int row = blockIdx.x / CTAS, part = blockIdx.x % CTAS;
  Row r;
  r.hist = a.history ? (a.history_len ? min(max(a.history_len[row], 0), a.hist) : a.hist) : 0;
  r.history = a.history + (long long)row * a.ldh;
  r.prompt = a.prompt_len ? a.prompt_len[row] : 0;
  r.nbias = a.bias_ids ? (a.bias_len ? min(max(a.bias_len[row], 0), a.nbias) : a.nbias) : 0;
  r.bias_ids = a.bias_ids + (long long)row * a.ldb;
  r.bias = a.bias + (long long)row * a.ldb;
  r.repeats = a.repetition != nullptr;
  r.repetition = a.repetition ? a.repetition[row] : 1.f;
  r.presence = a.presence ? a.presence[row] : 0.f;
  r.frequency = a.frequency ? a.frequency[row] : 0.f;
  const uint8_t* in = reinterpret_cast<const uint8_t*>(a.logits) + (long long)row * a.ldl * (HALF ? 2 : 4);
  uint8_t* out = reinterpret_cast<uint8_t*>(a.out) + (long long)row * a.ldo * (HALF ? 2 : 4);
  const uint32_t* allowed = a.allowed ? a.allowed + (long long)row * a.ldw : nullptr;
  const bool lists = r.hist > 0 || r.nbias > 0, keeps = a.out != nullptr, streams = threadIdx.x < STREAM;
  const int lt = (int)threadIdx.x - STREAM, st = threadIdx.x;

  const int share = ((a.vocab + CTAS - 1) / CTAS + 31) / 32 * 32;        // whole words of the bitmaps
  const int end = min(a.vocab, (part + 1) * share);
  float best = -CUDART_INF_F;
  int bi = 0x7fffffff;
  for (int lo = part * share; lo < end; lo += PIECE) {
    const int hi = min(lo + PIECE, end), whole = vectors ? (hi - lo) / (AT_ONCE * STEP) * (AT_ONCE * STEP) : 0;
    const unsigned first = (unsigned)(a.vocab_offset + lo), size = (unsigned)(hi - lo);
    if (lists) {
      __syncthreads();                                    // the piece before is done with the lists
      for (int i = threadIdx.x; i < WORDS; i += THREADS) listed[i] = 0;
      if (threadIdx.x == 0) n_listed = 0;
      __syncthreads();
      auto mark = [&](int, unsigned id) {
        if (atomicOr(&listed[id >> 5], 1u << (id & 31)) >> (id & 31) & 1u) return;
        ids[atomicAdd(&n_listed, 1)] = (uint16_t)id;
      };
      each(r.history, r.hist, first, size, threadIdx.x, THREADS, mark);
      each(r.bias_ids, r.nbias, first, size, threadIdx.x, THREADS, mark);
      __syncthreads();
      for (int k = threadIdx.x; k < n_listed; k += THREADS) raw[k] = load1<HALF>(in, lo + ids[k]);
      __syncthreads();                                    // from here on the stream may write over them
    }
    if (streams) {
      const uint4* src = reinterpret_cast<const uint4*>(in) + lo / N + st;
      uint4* dst = reinterpret_cast<uint4*>(out) + lo / N + st;
      const uint32_t* allow = allowed + (lo >> 5) + (st * N >> 5);
      const uint32_t* list = listed + (st * N >> 5);
      const int shift = st * N & 31;
      for (int c0 = 0; c0 < whole; c0 += AT_ONCE * STEP) {
        uint4 x[AT_ONCE];
        uint32_t ok[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          x[i] = src[i * STREAM];
          ok[i] = allowed ? allow[i * (STEP / 32)] : ~0u;
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          if (lists) ok[i] &= ~list[i * (STEP / 32)];
          float f[N];
          widen<HALF>(x[i], f);
          const uint32_t mine = ok[i] >> shift;
          float top = -CUDART_INF_F;
#pragma unroll
          for (int e = 0; e < N; ++e) {
            if (!(mine >> e & 1u)) f[e] = -CUDART_INF_F;
            top = fmaxf(top, f[e]);
          }
          if (top > best) {                               // seldom
            const int c = lo + c0 + i * STEP + st * N;
#pragma unroll
            for (int e = 0; e < N; ++e)
              if (f[e] > best) { best = f[e]; bi = c + e; }              // ascending per thread: the first maximum is kept
          }
          if (keeps) dst[i * STREAM] = narrow<HALF>(f);
        }
        src += AT_ONCE * STREAM;
        dst += AT_ONCE * STREAM;
        allow += AT_ONCE * (STEP / 32);
        list += AT_ONCE * (STEP / 32);
      }
      for (int at = whole + st; at < hi - lo; at += STREAM) {            // the rest, and rows at any address
        const int c = lo + at;
        float f = load1<HALF>(in, c);
        if ((allowed && !(allowed[c >> 5] >> (c & 31) & 1u)) || (lists && (listed[at >> 5] >> (at & 31) & 1u))) f = -CUDART_INF_F;
        if (f > best) { best = f; bi = c; }
        if (keeps) store1<HALF>(out, c, f);
      }
    } else if (lists) {
      int n[WPT], sum = 0;                                // a thread's words follow one another
#pragma unroll
      for (int i = 0; i < WPT; ++i) {
        n[i] = sum;
        sum += __popc(listed[lt * WPT + i]);
      }
      int before = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
      }
      if (lane == 31) warp_sum[lt >> 5] = before;
      for (int i = lt; i < n_listed; i += LIST) table[i] = 0;
      list_sync();
      before -= sum;
      if (lt >= 32) before += warp_sum[0];
#pragma unroll
      for (int i = 0; i < WPT; ++i) number[lt * WPT + i] = (uint16_t)(before + n[i]);
      list_sync();
      if (r.nbias) {                                      // before the counts: the largest place wins, whatever the order
        each(r.bias_ids, r.nbias, first, size, lt, LIST,
             [&](int i, unsigned id) { atomicMax(&table[number_of(listed, number, id)], (uint32_t)(i + 1) << BIAS_SHIFT); });
        list_sync();
      }
      each(r.history, r.hist, first, size, lt, LIST, [&](int i, unsigned id) {
        uint32_t* word = &table[number_of(listed, number, id)];
        if (i >= r.prompt) atomicAdd(word, 1u);
        else atomicOr(word, SEEN);
      });
    }
    if (lists) {
      __syncthreads();                                    // the words are whole, and the stream has written -inf there
      for (int k = threadIdx.x; k < n_listed; k += THREADS) {
        const int id = ids[k], c = lo + id;
        if (allowed && !(allowed[c >> 5] >> (c & 31) & 1u)) continue;
        const float v = adjust(raw[k], table[number_of(listed, number, id)], r);
        better(best, bi, v, c);
        if (keeps) store1<HALF>(out, c, v);
      }
    }
  }
  if (!a.tokens) {
    if (CTAS > 1) cluster_wait();
    return;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, best, o);
    const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
    better(best, bi, ov, oi);
  }
  __shared__ float sv[WARPS], pv[CTAS];
  __shared__ int si[WARPS], pi[CTAS];
  if (lane == 0) { sv[warp] = best; si[warp] = bi; }
  __syncthreads();
  if (CTAS > 1) cluster_wait();
  if (warp == 0) {
    best = lane < WARPS ? sv[lane] : -CUDART_INF_F;
    bi = lane < WARPS ? si[lane] : 0x7fffffff;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float ov = __shfl_xor_sync(0xffffffffu, best, o);
      const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
      better(best, bi, ov, oi);
    }
    if (CTAS > 1 && lane == 0) {
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_u32(smem_u32(&pv[part]), 0)), "f"(best) : "memory");
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapa_u32(smem_u32(&pi[part]), 0)), "r"(bi) : "memory");
    }
    __syncwarp();
  }
  if (CTAS > 1) cluster_sync_all();
  if (part != 0 || threadIdx.x != 0) return;
  if (CTAS > 1)
    for (int i = 0; i < CTAS; ++i) {
      if (i == 0) { best = pv[0]; bi = pi[0]; }
      else better(best, bi, pv[i], pi[i]);
    }
  a.tokens[row] = best == -CUDART_INF_F ? -1 : bi + a.vocab_offset;
}

// Listed ids that a piece has room for.
static int entries_of(const MeshLogits* a) {
  const int listed = a->hist + a->nbias;
  return listed < PIECE ? (listed + 1) / 2 * 2 : PIECE;
}
static int smem_of(int entries) { return entries > 0 ? LISTS + entries * ENTRY : 0; }

template <bool HALF, int CTAS>
static cudaError_t configure(int dev) {
  static std::atomic<unsigned long long> configured{0};   // a bit per device
  if (configured.load() >> (dev & 63) & 1) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(constrain_kernel<HALF, CTAS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_of(PIECE));
  if (e == cudaSuccess && CTAS > 8) e = cudaFuncSetAttribute(constrain_kernel<HALF, CTAS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) configured.fetch_or(1ull << (dev & 63));
  return e;
}

// Whether the current device can run a cluster of sixteen with this much shared memory a CTA: it is no size that every device has, and the
// CTAs need so many SMs of one group with that room.  Asked once for every 16 KB.
template <bool HALF>
static bool sixteen_fit(int smem) {
  constexpr int STEP = 16 * 1024;
  static std::atomic<int> known[64][(LISTS + PIECE * ENTRY) / STEP + 2];               // 1: no, 2: yes
  int dev = 0, n = 0;
  bool ok = cudaGetDevice(&dev) == cudaSuccess;
  std::atomic<int>& k = known[dev & 63][(smem + STEP - 1) / STEP];
  if (ok && k.load()) return k.load() == 2;
  const int most = smem_of(PIECE), asked = (smem + STEP - 1) / STEP * STEP;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(16);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = asked < most ? asked : most;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 16;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  ok = ok && configure<HALF, 16>(dev) == cudaSuccess && cudaOccupancyMaxActiveClusters(&n, constrain_kernel<HALF, 16>, &cfg) == cudaSuccess;
  if (!ok) {
    cudaGetLastError();                                   // eight will do
    return false;
  }
  k.store(n > 0 ? 2 : 1);
  return n > 0;
}

template <bool HALF, int CTAS>
static int run(const MeshLogits* a, void* stream) {
  int dev = 0;
  MESH_CUDA_OK(cudaGetDevice(&dev));
  MESH_CUDA_OK((configure<HALF, CTAS>(dev)));
  const int entries = entries_of(a), smem = smem_of(entries);
  const int vectors = !((uintptr_t)a->logits % 16) && a->ldl % Vec<HALF>::N == 0 && !((uintptr_t)a->out % 16) && a->ldo % Vec<HALF>::N == 0;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)(a->rows * CTAS));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CTAS;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CTAS > 1 ? 2 : 1;
  MESH_CUDA_OK(cudaLaunchKernelEx(&cfg, constrain_kernel<HALF, CTAS>, *a, vectors, entries));
  return 0;
}

}  // namespace constrain
}  // namespace mesh

extern "C" int mesh_constrain_logits(const MeshLogits* a, void* stream) {
  using namespace mesh;
  using namespace mesh::constrain;
  if (a->rows < 0 || a->rows > (1 << 20)) return set_error(-2, "constrain_logits: rows must be 0..2^20");
  if (a->vocab < 1 || a->vocab > (1 << 30)) return set_error(-2, "constrain_logits: vocabulary must be 1..2^30");
  if (a->hist > 65535) return set_error(-2, "constrain_logits: a history of at most 65535 tokens");
  if (a->nbias > 32767) return set_error(-2, "constrain_logits: at most 32767 biases");
  if (!a->out && !a->tokens) return set_error(-2, "constrain_logits: nothing asked for");
  if (a->rows == 0) return 0;
  const int smem = smem_of(entries_of(a));
  const int ctas = a->vocab <= ONE_CTA_VOCAB ? 1 : a->vocab <= EIGHT_CTA_VOCAB || !(a->half ? sixteen_fit<true>(smem) : sixteen_fit<false>(smem)) ? 8 : 16;
#define MESH_CONSTRAIN(HALF) (ctas == 1 ? run<HALF, 1>(a, stream) : ctas == 8 ? run<HALF, 8>(a, stream) : run<HALF, 16>(a, stream))
  return a->half ? MESH_CONSTRAIN(true) : MESH_CONSTRAIN(false);
#undef MESH_CONSTRAIN
}
