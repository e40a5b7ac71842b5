// Penalties for repeated tokens, biases and a grammar mask on logits, and the greedy choice among what is left, in one pass.
//
// A row's vocabulary is cut over the CTAs of a cluster; a CTA goes through its slice in pieces of 16384 ids.  What the history and the
// bias list say about a piece stands in a table in shared memory, a word per id: times the id was generated (16 bits), whether
// it stands in the history at all (1 bit), 1 + its last place in the bias list (15 bits); and a bit per id says that the word
// is set, so that only words of listed ids are ever cleared, written or read.  The loads of a piece's logits are under way
// while the lists are gone through.
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

constexpr int THREADS = 1024, PIECE = 16384, VEC = 4, PER = PIECE / (THREADS * VEC);
constexpr int MOST_CTAS = 8;
constexpr int SMEM = PIECE * 4 + PIECE / 8;
constexpr uint32_t COUNT = 0xffffu, SEEN = 0x10000u;
constexpr int BIAS_SHIFT = 17;

__device__ __forceinline__ void better(float& v, int& i, float ov, int oi) {
  if (ov > v || (ov == v && oi < i)) { v = ov; i = oi; }
}

// Four logits from column c of a row; what lies behind the last column reads as -inf.  (No read-only loads: the result may be
// written over the logits.)
template <bool HALF>
__device__ __forceinline__ float4 load4(const void* row, int c, int vocab, bool vec) {
  float f[4];
  if (vec && c + 4 <= vocab) {
    if (!HALF) return *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(row) + c);
    const uint2 x = *reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(row) + c);
    f[0] = __uint_as_float(x.x << 16); f[1] = __uint_as_float(x.x & 0xffff0000u);
    f[2] = __uint_as_float(x.y << 16); f[3] = __uint_as_float(x.y & 0xffff0000u);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      f[i] = c + i >= vocab ? -CUDART_INF_F
             : HALF         ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[c + i])
                            : reinterpret_cast<const float*>(row)[c + i];
  }
  return make_float4(f[0], f[1], f[2], f[3]);
}
template <bool HALF>
__device__ __forceinline__ void store4(void* row, int c, int vocab, bool vec, const float4& v) {
  const float f[4] = {v.x, v.y, v.z, v.w};
  if (vec && c + 4 <= vocab) {
    if (!HALF) {
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(row) + c) = v;
    } else {
      uint2 x;
      __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&x);
      h[0] = __floats2bfloat162_rn(v.x, v.y);
      h[1] = __floats2bfloat162_rn(v.z, v.w);
      *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(row) + c) = x;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (c + i < vocab) {
      if (HALF) reinterpret_cast<__nv_bfloat16*>(row)[c + i] = __float2bfloat16_rn(f[i]);
      else reinterpret_cast<float*>(row)[c + i] = f[i];
    }
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
  if (word >> BIAS_SHIFT) x = __fadd_rn(x, __ldg(r.bias + (word >> BIAS_SHIFT) - 1));
  return x;
}

template <bool HALF, int CTAS>
__global__ void __launch_bounds__(THREADS) constrain_kernel(const __grid_constant__ MeshLogits a, int vec_in, int vec_out) {
  extern __shared__ __align__(16) uint8_t smem[];
  uint32_t* table = reinterpret_cast<uint32_t*>(smem);
  uint32_t* listed = table + PIECE;                       // a bit per id of the piece
  griddep_launch_dependents();
  if (CTAS > 1) cluster_arrive_relaxed();                 // waited for before the store into the first CTA's shared memory
  griddep_wait();
  const int row = blockIdx.x / CTAS, part = blockIdx.x % CTAS;
  Row r;
  r.hist = a.history ? (a.history_len ? min(max(__ldg(a.history_len + row), 0), a.hist) : a.hist) : 0;
  r.history = a.history + (long long)row * a.ldh;
  r.prompt = a.prompt_len ? __ldg(a.prompt_len + row) : 0;
  r.nbias = a.bias_ids ? (a.bias_len ? min(max(__ldg(a.bias_len + row), 0), a.nbias) : a.nbias) : 0;
  r.bias_ids = a.bias_ids + (long long)row * a.ldb;
  r.bias = a.bias + (long long)row * a.ldb;
  r.repeats = a.repetition != nullptr;
  r.repetition = a.repetition ? __ldg(a.repetition + row) : 1.f;
  r.presence = a.presence ? __ldg(a.presence + row) : 0.f;
  r.frequency = a.frequency ? __ldg(a.frequency + row) : 0.f;
  const uint8_t* in = reinterpret_cast<const uint8_t*>(a.logits) + (long long)row * a.ldl * (HALF ? 2 : 4);
  uint8_t* out = reinterpret_cast<uint8_t*>(a.out) + (long long)row * a.ldo * (HALF ? 2 : 4);
  const uint32_t* allowed = a.allowed ? a.allowed + (long long)row * a.ldw : nullptr;
  const bool lists = r.hist > 0 || r.nbias > 0;

  const int pieces = (a.vocab + PIECE - 1) / PIECE, per = (pieces + CTAS - 1) / CTAS;
  float best = -CUDART_INF_F;
  int bi = 0x7fffffff;
  for (int piece = part * per; piece < min(pieces, (part + 1) * per); ++piece) {
    const int lo = piece * PIECE;
    const unsigned first = (unsigned)(a.vocab_offset + lo), size = (unsigned)min(PIECE, a.vocab - lo);
    float4 x[PER];
    uint32_t bits[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = lo + (i * THREADS + threadIdx.x) * VEC;
      bits[i] = ~0u;
      x[i] = make_float4(-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F);
      if (c < a.vocab) {
        x[i] = load4<HALF>(in, c, a.vocab, vec_in);
        if (allowed) bits[i] = __ldg(allowed + (c >> 5)) >> (c & 31);
      }
    }
    if (lists) {
      __syncthreads();                                    // the piece before is done with the table
      if (threadIdx.x < PIECE / 32) listed[threadIdx.x] = 0;
      for (int i = threadIdx.x; i < r.hist; i += THREADS) {
        const unsigned id = (unsigned)__ldg(r.history + i) - first;
        if (id < size) table[id] = 0;
      }
      for (int i = threadIdx.x; i < r.nbias; i += THREADS) {
        const unsigned id = (unsigned)__ldg(r.bias_ids + i) - first;
        if (id < size) table[id] = 0;
      }
      __syncthreads();
      if (r.nbias) {                                      // before the counts: the largest place wins, whatever the order
        for (int i = threadIdx.x; i < r.nbias; i += THREADS) {
          const unsigned id = (unsigned)__ldg(r.bias_ids + i) - first;
          if (id < size) {
            atomicMax(&table[id], (uint32_t)(i + 1) << BIAS_SHIFT);
            atomicOr(&listed[id >> 5], 1u << (id & 31));
          }
        }
        __syncthreads();
      }
      for (int i = threadIdx.x; i < r.hist; i += THREADS) {
        const unsigned id = (unsigned)__ldg(r.history + i) - first;
        if (id < size) {
          if (i >= r.prompt) atomicAdd(&table[id], 1u);
          else atomicOr(&table[id], SEEN);
          atomicOr(&listed[id >> 5], 1u << (id & 31));
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = (i * THREADS + threadIdx.x) * VEC, c = lo + at;
      if (c >= a.vocab) continue;
      float f[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
      if (lists) {
        const uint32_t l = listed[at >> 5] >> (at & 31) & 15u;
        if (l) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (l >> e & 1u) f[e] = adjust(f[e], table[at + e], r);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (!(bits[i] >> e & 1u)) f[e] = -CUDART_INF_F;
        if (f[e] > best) { best = f[e]; bi = c + e; }     // ascending per thread: the first maximum is kept
      }
      if (a.out) store4<HALF>(out, c, a.vocab, vec_out, make_float4(f[0], f[1], f[2], f[3]));
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
  __shared__ float sv[32], pv[CTAS];
  __shared__ int si[32], pi[CTAS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) { sv[warp] = best; si[warp] = bi; }
  __syncthreads();
  if (CTAS > 1) cluster_wait();
  if (warp == 0) {
    best = sv[lane];
    bi = si[lane];
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

template <bool HALF, int CTAS>
static int run(const MeshLogits* a, void* stream) {
  static std::atomic<unsigned long long> configured{0};   // a bit per device
  int dev = 0;
  MESH_CUDA_OK(cudaGetDevice(&dev));
  if (!(configured.load() >> (dev & 63) & 1)) {
    MESH_CUDA_OK(cudaFuncSetAttribute(constrain_kernel<HALF, CTAS>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    configured.fetch_or(1ull << (dev & 63));
  }
  const int size = HALF ? 2 : 4;
  const int vec_in = !((uintptr_t)a->logits % (4 * size)) && a->ldl % 4 == 0;
  const int vec_out = !((uintptr_t)a->out % (4 * size)) && a->ldo % 4 == 0;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)(a->rows * CTAS));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM;
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
  MESH_CUDA_OK(cudaLaunchKernelEx(&cfg, constrain_kernel<HALF, CTAS>, *a, vec_in, vec_out));
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
  const int ctas = a->vocab <= PIECE ? 1 : MOST_CTAS;
  if (a->half) return ctas > 1 ? run<true, MOST_CTAS>(a, stream) : run<true, 1>(a, stream);
  return ctas > 1 ? run<false, MOST_CTAS>(a, stream) : run<false, 1>(a, stream);
}
