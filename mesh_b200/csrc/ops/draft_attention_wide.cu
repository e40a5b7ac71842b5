// Attention of drafts with many query rows (which: `wide` in draft_attention.cu) on the 5th-generation tensor cores.
//
// A tile is 128 query rows of one (sequence, KV head); a CTA goes through its stretches of 64-key blocks (how the work is cut and
// the formulas: draft_attention.cuh, draft_attention.cu).  Warps 0-15: softmax, in two groups that take the blocks in turn, in each
// two threads per query row with half of the block's keys.  Warps 16-21: keys and values, a warp per 4 KB of a tile, into the 128-byte
// swizzle of the operands: bf16 rows by cp.async; 8-bit codes copied in bulk to places of the warp's own and widened to
// fp16 from there.  Warps 22 and 23: the products S = Q K^T, up to three blocks ahead, and O += P V, by one elected lane each.
// Tensor memory holds the queries (operand A of the first product, 16 bits), S of four blocks (heads of 256: two), of each of
// which P (16 bits, operand A of the second) overwrites the first half, and O, which is rescaled only when a row's maximum
// has grown by more than 2^8: the reference point of a row goes from group to group through shared memory.
//
// Codes are widened once per 128 rows: as operands of a product in 8 bits the queries and probabilities would have to be rounded to 8
// bits too.  Queries in tensor memory leave shared memory to the rings and its bandwidth to their stores and reads.  The
// roles are chains of short steps, each a few instructions behind the one before, so there are many warps of few registers; and
// they run different code on the same SM, so it is kept short.  The first form, with one group of softmax threads and scores read
// twice from tensor memory, took 165 us for 64 drafts x 4 heads over four contexts of 20000-32704 keys of 256 in 8 bits; this one takes
// 126 (29 at the tensor cores' rate).  Slower on the way: tiles held in registers ahead of their turn and everything inlined (112 KB of code,
// one fetch in six missed the cache); all loader threads at every tile; blocks of 128 keys with the queries in shared memory.
// What bounds it is the way of a block through the roles, some 4300 clocks for 64 keys of 256, of which the products need 1000: of 121
// us for 16 drafts over 8 contexts of 8000-16000 keys of 128 in 8 bits 92 were left without the softmax, 112 without the widened codes' stores.
#include "draft_attention.cuh"

namespace mesh {
namespace draft {
namespace {

constexpr int TT = WIDE_ROWS, KB = WIDE_UNIT;               // rows of a tile, keys of a block
constexpr int GROUP = 256, SOFT = 2 * GROUP, LOAD_WARPS = 6, THREADS = SOFT + 32 * LOAD_WARPS + 64;
constexpr int LOAD_WARP = SOFT / 32, S_WARP = LOAD_WARP + LOAD_WARPS, O_WARP = S_WARP + 1;
constexpr int SCALES = 8;                                   // blocks whose scales are kept: stages and buffers of S together
constexpr int CHUNK = 4096, PIECES = CHUNK / (32 * 16);     // bytes of stored rows a warp takes at a time; 16-byte pieces of a lane

template <int HD, bool Q8>
struct Wide {
  static constexpr int TILE = KB * HD * 2;
  // No more than pays, for the first-level cache's sake: heads of 256 in bf16 with three stages 62.2 us, with two 60.5 (64 drafts of 4
  // sequences over 6000-12000 keys); of 128 in 8 bits with four 99.2, with three 97.8, in bf16 86.3 and 88.1 (16 drafts of 8).
  static constexpr int STAGES = HD == 256 ? 2 : HD == 128 && Q8 ? 3 : 4;
  static constexpr int NB = HD < 256 ? 4 : 2;               // blocks whose S is in tensor memory
  static constexpr int RB = Q8 ? HD : 2 * HD, NC = RB / 16;           // bytes and 16-byte pieces of a stored row
  static constexpr int CPT = KB * RB / CHUNK;               // chunks of a tile
  // Chunks of bf16 rows that a warp has under way.  While it waits for a place, the product that frees it waits for tiles of at least
  // 2 STAGES - 1 before: what the warp has not handed over must be younger.
  static constexpr int BEHIND = CPT >= 4 ? 3 : 2;
  static_assert(Q8 || (BEHIND - 1) * LOAD_WARPS <= (2 * STAGES - 2) * CPT, "a loader would wait for what it has not handed over");
  // Chunks of codes that a warp has under way: a third would take memory from the first-level cache, which holds what the softmax warps have
  // no registers for (64 drafts over 20000-32704 keys of 256: 125 us, 136 with three, 134 with two and the memory of three).
  static constexpr int RAWS = Q8 ? 2 : 0;
  static constexpr int N_BARS = 1 + 4 * STAGES + 3 * NB + 2 + SCALES + RAWS * LOAD_WARPS;
  static constexpr int SCALE_BYTES = Q8 ? SCALES * 3 * KB * 4 : 0;
  static constexpr int SMEM = 2 * STAGES * TILE + RAWS * LOAD_WARPS * CHUNK + SCALE_BYTES + 8 * N_BARS + 64 + 1024;
  static constexpr int S_COL = 0, O_COL = NB * KB, Q_COL = O_COL + HD;  // columns of tensor memory
};

// Once, not in every role: its divisions are long.
__device__ __noinline__ bool next_stretch(const Args& a, Walk& w, Stretch& x) { return next(a, w, x); }

// The waits' slow path, once: a bounded wait, see mbar_wait.
__device__ __noinline__ bool wait_on(uint32_t bar, uint32_t parity, volatile int* abort_smem, Status* st, int site) {
  return mbar_wait(bar, parity, abort_smem, st, site);
}
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_smem, Status* st, int site) {
  bool ok = mbar_try_wait(bar, parity);
  if (!__all_sync(0xffffffffu, ok)) ok = __all_sync(0xffffffffu, wait_on(bar, parity, abort_smem, st, site));
  return ok;
}
// Until more than n blocks are over, bounded alike.  For a converged warp, whose lanes leave together: one of them looks for all.
__device__ __noinline__ bool wait_over(const volatile int* over, int n, volatile int* abort_smem, Status* st) {
  const unsigned long long t0 = globaltimer_ns();
  for (uint32_t it = 1;; ++it) {
    int end = 0;                                            // 1: over, 2: given up
    if ((threadIdx.x & 31) == 0) {
      const int now = *over;
      if (now > n) {
        end = 1;
      } else if (*abort_smem) {
        end = 2;
      } else if ((it & 0x3fu) == 0) {
        const bool canceled = status_aborted(st);
        if (canceled || globaltimer_ns() - t0 > MESH_WAIT_LIMIT_NS) {
          *abort_smem = 1;
          status_record(st, canceled ? MESH_CANCELED : MESH_TIMEOUT, SITE_SMEM_EMPTY, n, now, it);
          end = 2;
        }
      }
    }
    end = __shfl_sync(0xffffffffu, end, 0);
    if (end) return end == 1;
  }
}
// A role that gave up: its copies and products under way, each a phase of a barrier, have to be over before the CTA ends.  Bounded too,
// and whatever the others do.
__device__ __noinline__ void drain(uint32_t bar, uint32_t parity) {
  const unsigned long long t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity))
    if (globaltimer_ns() - t0 > MESH_WAIT_LIMIT_NS) return;
}
// 16 bytes, or zeros where `there` is false.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// two fp32 at a time
struct F2 { unsigned long long v; };
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack(F2 a, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

__device__ __forceinline__ int blocks_of(const Stretch& x) { return (x.k_hi - x.k_lo + KB - 1) / KB; }
// Whether some row may not see some key of the block.
__device__ __forceinline__ bool masked_block(const Args& a, const Stretch& x, int slot0) {
  return (a.window > 0 && slot0 < x.s.pos + 64 - a.window) || slot0 + KB > min(x.s.pos, x.k_hi);
}
// Bits of the slots first .. first + 32 that a row sees.
__device__ __forceinline__ uint32_t below(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; }
__device__ __forceinline__ uint32_t seen(const Stretch& x, int row_lo, unsigned long long vis, int first) {
  const int d = first - x.s.pos;
  const uint32_t past = below(-d) & ~below(row_lo - first);
  const uint32_t drafts = d >= 64 ? 0u : d >= 0 ? (uint32_t)(vis >> d) : d > -32 ? (uint32_t)(vis << -d) : 0u;
  return (past | drafts) & below(x.k_hi - first);
}
__device__ __forceinline__ bool not_finite(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t w) {
  return ((w & 0x7f80u) == 0x7f80u ? 0u : w & 0xffffu) | ((w & 0x7f800000u) == 0x7f800000u ? 0u : w & 0xffff0000u);
}

// Where the tiles of keys and values lie.  Per stretch they come in the order the products take them: K0 K1 V0 K2 V1 ... V(last).
struct Tiles {                                             // (the walk apart: what a call takes the address of stays in memory)
  Stretch x;
  int first = 0, blocks = 0, n0 = 0, stretch = -1;        // tiles before this stretch, its blocks, blocks before it, stretches with keys
  long long at = 0;                                       // row of its first slot
  bool key = false;
  int j = 0;                                              // block within the stretch
  // Tile o of all, not before the last one asked for; false behind the last.
  __device__ __forceinline__ bool find(const Args& a, Walk& walk, int o) {
    while (o - first >= 2 * blocks) {
      first += 2 * blocks;
      n0 += blocks;
      blocks = 0;
      Stretch y;
      if (!next_stretch(a, walk, y)) return false;
      x = y;
      blocks = blocks_of(x);
      stretch += blocks > 0;
      at = ((long long)x.b * a.kv_heads + x.hk) * a.max_seq + x.k_lo;
    }
    o -= first;
    key = o == 0 || ((o & 1) && o < 2 * blocks - 1);
    j = key ? (o + 1) / 2 : o == 2 * blocks - 1 ? blocks - 1 : o / 2 - 1;
    return true;
  }
  __device__ __forceinline__ int n() const { return n0 + j; }                              // block of all
  __device__ __forceinline__ int slot() const { return x.k_lo + j * KB; }
  __device__ __forceinline__ int rows() const { return x.k_hi - slot(); }                  // of the tile, if fewer than KB
};

template <int HD, bool Q8>
__global__ void __launch_bounds__(THREADS, 1) wide_kernel(const __grid_constant__ Args a) {
  using C = Wide<HD, Q8>;
  constexpr uint32_t FP16 = Q8 ? (1u << 7) | (1u << 10) : 0u;              // operands in fp16 instead of bf16
  constexpr int STAGES = C::STAGES, NC = C::NC, NB = C::NB;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t sK = base, sV = sK + STAGES * C::TILE, sRaw = sV + STAGES * C::TILE, sScale = sRaw + C::RAWS * LOAD_WARPS * CHUNK, bars = sScale + C::SCALE_BYTES;
  float* scale_s = reinterpret_cast<float*>(gen + (sScale - base));        // [buffer]{key scale, lg2 of the value scale, value scale}[key]
  auto bar = [&](int i) { return bars + 8u * i; };
  constexpr int Q_FULL = 0, K_FULL = 1, K_EMPTY = K_FULL + STAGES, V_FULL = K_EMPTY + STAGES, V_EMPTY = V_FULL + STAGES,
                S_FULL = V_EMPTY + STAGES, P_FULL = S_FULL + NB, O_DONE = P_FULL + NB, M_READY = O_DONE + NB, SC_FULL = M_READY + 2, RAW_FULL = SC_FULL + SCALES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gen + (bars - base) + 8 * C::N_BARS);
  volatile int* abort_smem = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // [8]: stretch + 1 whose values had to be cleaned.  Only stretches with keys count: loaders are at most 5 of them ahead.
  volatile int* spoilt_s = reinterpret_cast<volatile int*>(tmem_slot + 2);
  __shared__ Walk walk_s;
  __shared__ float top_s[2][2][2][TT];                      // [group][its block & 1][half][row]
  __shared__ float m_s[2][TT], sum_s[4][TT];                // [group][row]: reference points; [group, half][row]
  __shared__ float2 ml_s[TT];                               // of a cluster's part
  __shared__ volatile int over_s;                           // blocks whose second product is over
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = a.q_heads / a.kv_heads;

  if (threadIdx.x == 0) {
    mbar_init(bar(Q_FULL), SOFT);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar(K_FULL + s), C::CPT);
      mbar_init(bar(V_FULL + s), C::CPT);
      mbar_init(bar(K_EMPTY + s), 1);
      mbar_init(bar(V_EMPTY + s), 1);
    }
    for (int s = 0; s < NB; ++s) {
      mbar_init(bar(S_FULL + s), 1);
      mbar_init(bar(P_FULL + s), GROUP);
      mbar_init(bar(O_DONE + s), 1);
    }
    for (int s = 0; s < 2; ++s) mbar_init(bar(M_READY + s), GROUP);
    over_s = 0;
    for (int s = 0; s < SCALES; ++s) mbar_init(bar(SC_FULL + s), 1);
    for (int s = 0; s < C::RAWS * LOAD_WARPS; ++s) mbar_init(bar(RAW_FULL + s), 1);
    *abort_smem = 0;
    for (int s = 0; s < 8; ++s) spoilt_s[s] = 0;
    fence_mbar_init();
  }
  if (warp == O_WARP) {
    tmem_alloc<1>(smem_u32(tmem_slot), 512);
    tmem_relinquish<1>();
  }
  griddep_wait();
  griddep_launch_dependents();
  if (warp == 0) begin_walk(a, &walk_s);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  Walk walk = walk_s;
  Stretch x;
  bool ok = true;

  if (warp >= LOAD_WARP && warp < S_WARP) {
    // ------------------------------------------------------------------ keys and values
    // Chunk q of all is warp q mod LOAD_WARPS's.
    Tiles t;
    const int w0 = warp - LOAD_WARP;
    // A warp may pass a place's phases unseen, and a wait could be answered by the phase before the one it means: so the one two phases
    // back must be known to be over, which it nearly always is.
    auto place_free = [&]() {
      const int n = t.n();
      if (n < STAGES) return true;
      if (n >= 2 * STAGES && !__all_sync(0xffffffffu, over_s > n - 2 * STAGES) && !wait_over(&over_s, n - 2 * STAGES, abort_smem, a.status)) return false;
      return wait_warp(bar((t.key ? K_EMPTY : V_EMPTY) + n % STAGES), (n / STAGES - 1) & 1, abort_smem, a.status, SITE_SMEM_EMPTY);
    };
    if (Q8) {
      constexpr int RAWS = C::RAWS ? C::RAWS : 1;
      Tiles ahead;
      Walk ahead_walk = walk;
      const uint32_t own = sRaw + w0 * (RAWS * CHUNK), own_full = bar(RAW_FULL) + 8 * w0 * RAWS;
      // Starts the copy of a chunk; what lies behind the last slot is not read, and behind the last chunk nothing: a place's phase ends at once.
      auto fetch = [&](int q, int place) {
        const bool there = ahead.find(a, ahead_walk, q / C::CPT);
        const int part = q % C::CPT, bytes = there ? min(max(ahead.rows() * C::RB - part * CHUNK, 0), CHUNK) : 0;
        if (lane == 0) {
          mbar_expect_tx(own_full + 8 * place, bytes);
          if (bytes)
            bulk_load_1d(own + place * CHUNK, (ahead.key ? a.k : a.v) + (ahead.at + ahead.j * KB) * C::RB + part * CHUNK, bytes, own_full + 8 * place);
        }
      };
#pragma unroll 1
      for (int i = 0; i < RAWS; ++i) fetch(w0 + i * LOAD_WARPS, i);
      int place = 0, phase = 0;
#pragma unroll 1
      for (int q = w0; ok && t.find(a, walk, q / C::CPT); q += LOAD_WARPS) {
        const int part = q % C::CPT, s = t.n() % STAGES, rows = t.rows();
        const bool scales = t.key && part == 0;
        float f[4];                                       // scales of keys lane, lane + 32 and their values
        if (scales) {
          const long long row = t.at + t.j * KB + lane;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            f[i] = lane + 32 * i < rows ? __ldcg(a.k_scale + row + 32 * i) : 0.f;
            f[2 + i] = lane + 32 * i < rows ? __ldcg(a.v_scale + row + 32 * i) : 0.f;
          }
        }
        ok = wait_warp(own_full + 8 * place, phase, abort_smem, a.status, SITE_SMEM_FULL) && place_free();
        if (!ok) break;
        const uint8_t* src = gen + (own - base) + place * CHUNK;
        uint8_t* dst = gen + ((t.key ? sK : sV) + s * C::TILE - base);
#pragma unroll 4
        for (int i = 0; i < PIECES; ++i) {
          // the eight lanes of a phase store to eight different 16-byte banks: four pieces of each of two rows that follow one another
          const int at = NC == 4 ? lane : NC == 8 ? (lane & 19) | (lane & 4) << 1 | (lane & 8) >> 1 : (lane & 3) | (lane & 4) << 2 | (lane & 24) >> 1;
          const int idx = part * (CHUNK / 16) + i * 32 + at, r = idx / NC, c = idx % NC;
          uint4 v = *reinterpret_cast<const uint4*>(src + (i * 32 + at) * 16);
          if (r >= rows) v = make_uint4(0, 0, 0, 0);
          uint8_t* p = dst + (c >> 2) * (KB * 128) + r * 128;
          const uint32_t w[4] = {v.x ^ 0x80808080u, v.y ^ 0x80808080u, v.z ^ 0x80808080u, v.w ^ 0x80808080u};
          const uint4 lo = make_uint4(codes2(w[0], 0x4140), codes2(w[0], 0x4342), codes2(w[1], 0x4140), codes2(w[1], 0x4342));
          const uint4 hi = make_uint4(codes2(w[2], 0x4140), codes2(w[2], 0x4342), codes2(w[3], 0x4140), codes2(w[3], 0x4342));
          const int c0 = 2 * (c & 3);
          *reinterpret_cast<uint4*>(p + ((c0 ^ (r & 7)) << 4)) = lo;
          *reinterpret_cast<uint4*>(p + (((c0 + 1) ^ (r & 7)) << 4)) = hi;
        }
        if (scales) {
          float* sc = scale_s + (t.n() % SCALES) * 3 * KB + lane;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            sc[32 * i] = f[i];
            sc[KB + 32 * i] = fmaxf(lg2(f[2 + i]), -60.f);
            sc[2 * KB + 32 * i] = f[2 + i];
          }
        }
        fence_proxy_async_smem();                         // of the stores, for the products; of the reads, for the next copy
        __syncwarp();
        if (lane == 0) {
          if (scales) mbar_arrive(bar(SC_FULL + t.n() % SCALES));
          mbar_arrive(bar((t.key ? K_FULL : V_FULL) + s));
        }
        fetch(q + RAWS * LOAD_WARPS, place);
        if (++place == RAWS) {
          place = 0;
          phase ^= 1;
        }
      }
      for (int i = 0; !ok && i < RAWS; ++i) {
        drain(own_full + 8 * place, phase);
        if (++place == RAWS) {
          place = 0;
          phase ^= 1;
        }
      }
    } else {
      // What a chunk under way needs when it is handed over: its barrier, and for values of a masked block where they lie.
      uint32_t full[C::BEHIND] = {}, clean[C::BEHIND] = {};
      int of[C::BEHIND] = {};
      bool more = true;
      int under_way = 0;
#pragma unroll 1
      for (int q = w0; ok && (more || under_way > 0); q += LOAD_WARPS) {
        if (full[C::BEHIND - 1]) {
          asm volatile("cp.async.wait_group %0;" ::"n"(C::BEHIND - 1) : "memory");
          if (clean[C::BEHIND - 1]) {
            // zero times a NaN or an infinity is not zero: hidden keys must not hold any.  Rows that see them get them at the end.
            bool spoilt = false;
#pragma unroll 1
            for (int i = 0; i < PIECES; ++i) {
              const int idx = i * 32 + lane, c = idx % NC, r0 = (clean[C::BEHIND - 1] - base) / 128, r = idx / NC;
              uint4* p = reinterpret_cast<uint4*>(gen + (clean[C::BEHIND - 1] - base) + (c >> 3) * (KB * 128) + r * 128 + (((c & 7) ^ ((r0 + r) & 7)) << 4));
              const uint4 v = *p;
              if (not_finite(v.x) || not_finite(v.y) || not_finite(v.z) || not_finite(v.w)) {
                *p = make_uint4(finite_or_zero(v.x), finite_or_zero(v.y), finite_or_zero(v.z), finite_or_zero(v.w));
                spoilt = true;
              }
            }
            if (spoilt) spoilt_s[of[C::BEHIND - 1] & 7] = of[C::BEHIND - 1] + 1;
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(full[C::BEHIND - 1]);
          --under_way;
        }
        uint32_t new_full = 0, new_clean = 0;
        if (more) more = t.find(a, walk, q / C::CPT);
        if (more) {
          const int part = q % C::CPT, s = t.n() % STAGES, rows = t.rows();
          const uint32_t dst = (t.key ? sK : sV) + s * C::TILE;
          const uint8_t* src = (t.key ? a.k : a.v) + (t.at + t.j * KB) * C::RB;
          ok = place_free();
          if (!ok) break;
#pragma unroll 4
          for (int i = 0; i < PIECES; ++i) {
            const int idx = part * (CHUNK / 16) + i * 32 + lane, r = idx / NC, c = idx % NC;
            copy16(dst + (c >> 3) * (KB * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4), src + (r < rows ? idx * 16 : 0), r < rows);
          }
          new_full = bar((t.key ? K_FULL : V_FULL) + s);
          ++under_way;
          if (!t.key && masked_block(a, t.x, t.slot())) new_clean = dst + part * (CHUNK / C::RB) * 128;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll
        for (int i = C::BEHIND - 1; i > 0; --i) {
          full[i] = full[i - 1];
          clean[i] = clean[i - 1];
          of[i] = of[i - 1];
        }
        full[0] = new_full;
        clean[0] = new_clean;
        of[0] = t.stretch;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");      // nothing is under way, unless this warp gave up
    }
  } else if (warp == S_WARP) {
    // ------------------------------------------------------------------ S = Q K^T (warp-uniform, one elected lane issues)
    constexpr uint32_t idesc = umma_idesc_bf16(TT, KB, 0, 0) & ~FP16;
    const bool leader = elect_one();
    const uint64_t dk0 = umma_smem_desc(sK, 16, 1024);
    int n = 0, visit = 0;                                 // blocks and stretches done
    for (Stretch y; ok && next_stretch(a, walk, y);) {
      const int blocks = blocks_of(y);
      if (blocks == 0) continue;
      ok = wait_warp(bar(Q_FULL), visit++ & 1, abort_smem, a.status, SITE_SMEM_FULL);
      const int first = n;
      if (lane == 0) over_s = n;
#pragma unroll 1
      for (; ok && n < first + blocks; ++n) {
        // This S overwrites the P that the product NB blocks back reads: that one's end is waited for.  (So by the time a block's
        // scores are there, that product is over: a wait for the end of a product, on one of NB barriers in turn, cannot be
        // answered by the phase before.)
        if (n >= first + NB) {
          ok = wait_warp(bar(O_DONE + n % NB), (n / NB - 1) & 1, abort_smem, a.status, SITE_TMEM_EMPTY);
          if (lane == 0) over_s = n - NB + 1;
        }
        const int s = n % STAGES;
        ok = ok && wait_warp(bar(K_FULL + s), (n / STAGES) & 1, abort_smem, a.status, SITE_SMEM_FULL);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          const uint32_t d = tmem + C::S_COL + n % NB * KB;
          const uint64_t dk = dk0 + (uint32_t)(s * (C::TILE >> 4));
#pragma unroll
          for (int k = 0; k < HD / 16; ++k)
            umma_f16_ts(d, tmem + C::Q_COL + k * 8, dk + ((k / 4) * (KB * 128) + (k % 4) * 32) / 16, idesc, k ? 1u : 0u);
          umma_commit(bar(K_EMPTY + s));
          umma_commit(bar(S_FULL + n % NB));
        }
        __syncwarp();
      }
    }
    if (!ok && n > 0) drain(bar(S_FULL + (n - 1) % NB), (n - 1) / NB & 1);
  } else if (warp == O_WARP) {
    // ------------------------------------------------------------------ O += P V
    constexpr uint32_t idesc = umma_idesc_bf16(TT, HD, 0, 1) & ~FP16;                       // B = V is MN-major
    const bool leader = elect_one();
    const uint64_t dv0 = umma_smem_desc(sV, KB * 128, 1024);
    int n = 0;
    for (Stretch y; ok && next_stretch(a, walk, y);) {
      const int first = n, blocks = blocks_of(y);
#pragma unroll 1
      for (; ok && n < first + blocks; ++n) {
        const int s = n % STAGES;
        ok = wait_warp(bar(V_FULL + s), (n / STAGES) & 1, abort_smem, a.status, SITE_SMEM_FULL);
        ok = ok && wait_warp(bar(P_FULL + n % NB), n / NB & 1, abort_smem, a.status, SITE_TMEM_FULL);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          const uint32_t p = tmem + C::S_COL + n % NB * KB;
          const uint64_t dv = dv0 + (uint32_t)(s * (C::TILE >> 4));
#pragma unroll
          for (int k = 0; k < KB / 16; ++k) umma_f16_ts(tmem + C::O_COL, p + k * 8, dv + k * 128, idesc, k ? 1u : n > first ? 1u : 0u);
          umma_commit(bar(V_EMPTY + s));
          umma_commit(bar(O_DONE + n % NB));
        }
        __syncwarp();
      }
    }
    if (!ok && n > 0) drain(bar(O_DONE + (n - 1) % NB), (n - 1) / NB & 1);
  } else if (warp < LOAD_WARP) {
    // ------------------------------------------------------------------ softmax: two threads per query row = TMEM lane
    constexpr float LIFT = Q8 ? 6.f : 0.f;                // with the 2^8 that a reference may lag behind, w stays below 2^14
    constexpr int HALF = KB / 2;                          // keys of a thread
    const int row = threadIdx.x & 127, half = threadIdx.x >> 7 & 1, group = threadIdx.x / GROUP, quarter = threadIdx.x >> 7;
    const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    auto both = [&] { asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(GROUP) : "memory"); };      // halves of a group
    auto all = [] { asm volatile("bar.sync 3, %0;" ::"n"(SOFT) : "memory"); };
    int n = 0, stretch = -1;                              // blocks of the stretches before
    // Every warp of these passes the same barriers whatever happens: a wait that ran out makes the others run out, it ends no loop.
    for (Stretch y; next_stretch(a, walk, y);) {
      x = y;
      const int blocks = blocks_of(x), r = x.tile * TT + row, t = min(r / G, a.T - 1), h = x.hk * G + r % G;
      const bool real = row < x.n_rows;
      float unit = 1.f;
      stretch += blocks > 0;
      if (blocks > 0) {                                   // a quarter of a row of Q into its place
        const __nv_bfloat16* src = a.q + x.b * a.q_sb + t * a.q_st + (long long)h * HD + quarter * (HD / 4);
        const bool vec = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
        auto piece = [&](int c) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (real) {
            if (vec) {
              v = *reinterpret_cast<const uint4*>(src + c * 8);
            } else {
              const unsigned short* u = reinterpret_cast<const unsigned short*>(src + c * 8);
              v = make_uint4(u[0] | (uint32_t)u[1] << 16, u[2] | (uint32_t)u[3] << 16, u[4] | (uint32_t)u[5] << 16, u[6] | (uint32_t)u[7] << 16);
            }
          }
          return v;
        };
        if (Q8) {
          float top = 0.f;
#pragma unroll 2
          for (int c = 0; c < HD / 32; ++c) {
            const uint4 v = piece(c);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xffff0000u))));
          }
          sum_s[quarter][row] = top;
          all();
          top = fmaxf(fmaxf(sum_s[0][row], sum_s[1][row]), fmaxf(sum_s[2][row], sum_s[3][row]));
          unit = ldexpf(1.f, top > 0.f ? min(max(8 - ilogbf(top), -110), 110) : 0);
        }
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          const uint4 v = piece(c);
          uint32_t w[4] = {v.x, v.y, v.z, v.w};
          if (Q8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack16(true, __uint_as_float(w[i] << 16) * unit, __uint_as_float(w[i] & 0xffff0000u) * unit);
          }
          __syncwarp();
          asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(lane_addr + C::Q_COL + quarter * (HD / 8) + c * 4),
                       "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
        }
        tmem_st_wait();
        tc_fence_before();                                // and O of the stretch before has been read
        mbar_arrive(bar(Q_FULL));
      }
      const float q_unit = a.scale_log2 / unit;
      const unsigned long long vis = a.visible ? (unsigned long long)__ldcg(a.visible + (long long)x.b * a.T + t) : t >= 63 ? ~0ull : (2ull << t) - 1;
      const int row_lo = a.window > 0 ? max(0, x.s.pos + max(__popcll(vis), 1) - a.window) : 0;
      const bool works = (warp & 3) * 32 < x.n_rows;            // some row of this warp is real
      const F2 unit2 = f2(q_unit, q_unit);
      const int before = n;
      float m = -CUDART_INF_F, l = 0.f;                   // the point that l is relative to
      for (int j = (n & 1) ^ group; j < blocks; j += 2) {
        const int n = before + j;
        ok = ok && wait_warp(bar(S_FULL + n % NB), n / NB & 1, abort_smem, a.status, SITE_TMEM_FULL);
        if (Q8) ok = ok && wait_warp(bar(SC_FULL + n % SCALES), (n / SCALES) & 1, abort_smem, a.status, SITE_SMEM_FULL);
        tc_fence_after();
        const uint32_t s_addr = lane_addr + C::S_COL + n % NB * KB;
        const int slot0 = x.k_lo + j * KB;
        const bool masked = masked_block(a, x, slot0);
        const float4* ks = reinterpret_cast<const float4*>(scale_s + (n % SCALES) * 3 * KB + half * HALF);
        uint32_t v[32], see = ~0u;                        // scores times the keys' scales; the keys that the row sees
        if (works) {
          tmem_ld_32x32(s_addr + half * HALF, v);
          tmem_ld_wait();
          if (Q8) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 k4 = ks[i / 4];
              float f0, f1;
              unpack(mul2(f2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), f2(k4.x, k4.y)), f0, f1);
              v[i] = __float_as_uint(f0);
              v[i + 1] = __float_as_uint(f1);
              unpack(mul2(f2(__uint_as_float(v[i + 2]), __uint_as_float(v[i + 3])), f2(k4.z, k4.w)), f0, f1);
              v[i + 2] = __float_as_uint(f0);
              v[i + 3] = __float_as_uint(f1);
            }
          }
          if (masked) {
            see = seen(x, row_lo, vis, slot0 + half * HALF);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(see >> i & 1u)) v[i] = 0xff800000u;   // -inf: exp2 gives an exact zero
          }
          float part[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            float f[4] = {__uint_as_float(v[i]), __uint_as_float(v[i + 1]), __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3])};
            if (Q8) {
              const float4 u4 = ks[KB / 4 + i / 4];
              unpack(fma2(f2(f[0], f[1]), unit2, f2(u4.x, u4.y)), f[0], f[1]);
              unpack(fma2(f2(f[2], f[3]), unit2, f2(u4.z, u4.w)), f[2], f[3]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) part[e] = fmaxf(part[e], f[e]);
          }
          float top = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
          if (!Q8) top *= q_unit;
          top_s[group][n >> 1 & 1][half][row] = top;
        }
        both();                                           // and every score is in registers: P may overwrite them
        if (!works) mbar_arrive(bar(M_READY + group));
        if (works) {
          const float top = fmaxf(top_s[group][n >> 1 & 1][0][row], top_s[group][n >> 1 & 1][1][row]);
          float alpha = 1.f, now = -CUDART_INF_F;         // the point that the other group left for the block before
          if (j > 0) {
            ok = ok && wait_warp(bar(M_READY + (group ^ 1)), (n - 1) >> 1 & 1, abort_smem, a.status, SITE_SMEM_FULL);
            now = m_s[group ^ 1][row];
          }
          if (top - LIFT > now + 8.f) {                   // also the first block with a visible key (now = -inf)
            alpha = ex2(now - (top - LIFT));
            now = top - LIFT;
          }
          if (half == 0) m_s[group][row] = now;
          // By both halves: the other group may write its next points, and pass its barrier's next phase, only when every thread here has
          // read the last ones.
          mbar_arrive(bar(M_READY + group));
          if (m != now) {
            l *= ex2(m - now);                            // nothing summed yet: 0
            m = now;
          }
          // tcgen05.ld / .st are warp-collective: the decision must be the same for all rows of a warp.  Never for the first
          // block: its product overwrites O.
          if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
            ok = ok && wait_warp(bar(O_DONE + (n - 1) % NB), (n - 1) / NB & 1, abort_smem, a.status, SITE_TMEM_EMPTY);
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {           // half of the columns each
              uint32_t o[16];
              const uint32_t at = lane_addr + C::O_COL + half * (HD / 2) + c * 16;
              tmem_ld_32x16(at, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st_32x16(at, o);
            }
          }
          const float off = m == -CUDART_INF_F ? 0.f : -m;
          const F2 off2 = f2(off, off);
          F2 sum2[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float p0, p1;
            unpack(fma2(f2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), unit2, off2), p0, p1);
            F2 p = f2(ex2(p0), ex2(p1));
            sum2[(i / 2) & 1] = add2(sum2[(i / 2) & 1], p);
            if (Q8) {
              const float4 v4 = ks[2 * KB / 4 + i / 4];
              p = mul2(p, i & 2 ? f2(v4.z, v4.w) : f2(v4.x, v4.y));
            }
            unpack(p, p0, p1);
            w[i / 2] = pack16(Q8, p0, p1);
          }
          if (Q8 && masked) {                             // a hidden key's scale may be anything
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] &= (see >> (2 * i) & 1u ? 0xffffu : 0u) | (see >> (2 * i + 1) & 1u ? 0xffff0000u : 0u);
          }
          tmem_st_32x16(s_addr + half * (HALF / 2), w);
          float s0, s1;
          unpack(add2(sum2[0], sum2[1]), s0, s1);
          l += s0 + s1;
          tmem_st_wait();
        }
        tc_fence_before();
        mbar_arrive(bar(P_FULL + n % NB));
      }
      n += blocks;
      // ---- the stretch's result: final, or a share of it; a quarter of the columns each
      if (blocks > 0) {
        ok = ok && wait_warp(bar(O_DONE + (n - 1) % NB), (n - 1) / NB & 1, abort_smem, a.status, SITE_TMEM_FULL);
        tc_fence_after();
      }
      all();                                              // every point that is waited for has been read
      if (half == 0) m_s[group][row] = m;
      sum_s[quarter][row] = l;
      all();
      {                                                   // the later point of the two; sums of both groups brought to it
        const float m0 = m_s[0][row], m1 = m_s[1][row], ref = fmaxf(m0, m1), at = ref == -CUDART_INF_F ? 0.f : ref;
        l = (sum_s[0][row] + sum_s[1][row]) * ex2(m0 - at) + (sum_s[2][row] + sum_s[3][row]) * ex2(m1 - at);
        m = ref;
      }
      all();                                              // they have been read
      if (!ok || !works) continue;
      const bool spoilt = !Q8 && blocks > 0 && spoilt_s[stretch & 7] == stretch + 1;
      const float inv = !x.whole ? 1.f : l == 0.f ? 0.f : 1.f / l;
      __nv_bfloat16* dst = a.out + x.b * a.o_sb + t * a.o_st + (long long)h * HD;
      const bool vec = (reinterpret_cast<uintptr_t>(dst) & 15) == 0;
#pragma unroll 1
      for (int c = quarter * (HD / 64); c < (quarter + 1) * (HD / 64); ++c) {
        uint32_t o[16];
        if (blocks > 0) {
          tmem_ld_32x16(lane_addr + C::O_COL + c * 16, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = 0;
        }
        if (spoilt) {                                     // seldom: values of the masked blocks that are not finite
          const __nv_bfloat16* v0 = reinterpret_cast<const __nv_bfloat16*>(a.v) + ((long long)x.b * a.kv_heads + x.hk) * a.max_seq * HD + c * 16;
          for (int slot = x.k_lo; slot < x.k_hi; ++slot) {
            if (!masked_block(a, x, x.k_lo + (slot - x.k_lo) / KB * KB)) continue;
            if (!(seen(x, row_lo, vis, slot) & 1u)) continue;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float f = __bfloat162float(v0[(long long)slot * HD + i]);
              o[i] = __float_as_uint(__uint_as_float(o[i]) + (fabsf(f) < CUDART_INF_F ? 0.f : f));
            }
          }
          __syncwarp();
        }
        // the loads above are warp-collective: every lane takes part, only the stores depend on the row being real
        if (real && x.whole) {
          uint32_t w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = pack16(false, __uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
          uint32_t* p = reinterpret_cast<uint32_t*>(dst + c * 16);
          if (vec) {
            reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
            reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = w[i];
          }
        } else if (real && a.cluster) {                   // the only stretch: the rings are not used again
#pragma unroll
          for (int i = 0; i < 4; ++i)
            reinterpret_cast<float4*>(gen)[(c * 4 + i) * TT + row] =
                make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
        } else if (real) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            a.part[((long long)x.slot * (HD / 4) + c * 4 + i) * TT + row] =
                make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
        }
        __syncwarp();
      }
      if (!x.whole && real && quarter == 0) (a.cluster ? ml_s[row] : a.part_ml[(long long)x.slot * TT + row]) = make_float2(m, l);
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == O_WARP) {
    tc_fence_after();
    tmem_dealloc<1>(tmem, 512);
  }
  // ---- a cluster's item that was cut: each CTA joins some groups of 8 columns
  const int ranks = walk_s.ranks;
  if (ranks <= 1) return;                                   // the same in all CTAs of the cluster; 0 without clusters
  cluster_sync_all();
  const Item item = item_of_cluster(a);
  const int n_rows = min(sequence(a, item.b).count * G - item.tile * TT, TT);
  for (int e = threadIdx.x; e < TT * ((HD / 8 + a.cluster - 1) / a.cluster); e += THREADS) {
    const int row = e % TT, i = 2 * (e / TT * a.cluster + blockIdx.x % a.cluster), r = item.tile * TT + row;
    if (row >= n_rows || i >= HD / 4) continue;
    float m = -CUDART_INF_F, l = 0.f;
    for (int c = 0; c < ranks; ++c) m = fmaxf(m, cluster_load2(smem_u32(ml_s + row), c).x);
    const float ref = m == -CUDART_INF_F ? 0.f : m;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int c = 0; c < ranks; ++c) {
      const float2 ml = cluster_load2(smem_u32(ml_s + row), c);
      const float4 u = cluster_load4(base + (i * TT + row) * 16, c), v = cluster_load4(base + ((i + 1) * TT + row) * 16, c);
      const float wt = ex2(ml.x - ref);
      l += wt * ml.y;
      acc[0] += wt * u.x; acc[1] += wt * u.y; acc[2] += wt * u.z; acc[3] += wt * u.w;
      acc[4] += wt * v.x; acc[5] += wt * v.y; acc[6] += wt * v.z; acc[7] += wt * v.w;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + item.b * a.o_sb + (r / G) * a.o_st + (long long)(item.hk * G + r % G) * HD + i * 4);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = pack16(false, acc[2 * j] * inv, acc[2 * j + 1] * inv);
    if ((reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) dst[j] = w[j];
    }
  }
  cluster_sync_all();                                       // the others have read this CTA's part
}

// Joins the shares of the items that were cut, a thread per row and 8 columns.  SPLIT: a CTA per item and 8 columns, four groups of threads
// that take the shares in turn (few items in many shares); else one per item and 32 columns, a group for 8 of them.
constexpr int GROUPS = 4;
template <int HD, bool SPLIT>
__global__ void __launch_bounds__(GROUPS * TT) wide_join_kernel(const __grid_constant__ Args a) {
  constexpr int EACH = SPLIT ? GROUPS : 1;                // groups among which an item's shares are dealt
  __shared__ int c_s[3];
  __shared__ float2 ml_s[GROUPS][TT];
  __shared__ float4 o_s[GROUPS][2][TT];
  const int warp = threadIdx.x >> 5, row = threadIdx.x % TT, group = threadIdx.x / TT, G = a.q_heads / a.kv_heads;
  const int tile = blockIdx.x % a.tiles, hk = blockIdx.x / a.tiles % a.kv_heads, b = blockIdx.x / a.tiles / a.kv_heads;
  const int i = SPLIT ? blockIdx.y * 2 : blockIdx.y * 8 + group * 2;       // group of 4 columns
  // All wait: what comes after this kernel relies on the one before it.  And none looks at the lengths before: they are older than
  // that kernel, but only the wait keeps a read from finding what its line held before them.
  griddep_launch_dependents();
  griddep_wait();
  if (warp == 0) shares_of_item(a, b, hk, tile, c_s);
  __syncthreads();
  const int c0 = c_s[0], c1 = c_s[1], odd = c_s[2];
  if (c0 == c1) return;                                   // whole in one CTA, or not there
  const int n_rows = min(sequence(a, b).count * G - tile * TT, TT);
  float m = -CUDART_INF_F, l = 0.f;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (row < n_rows) {
#pragma unroll 4
    for (int c = c0 + (SPLIT ? group : 0); c <= c1; c += EACH) {
      const long long slot = 2 * c + (c == c0 ? odd : 0);
      const float2 x = __ldcg(a.part_ml + slot * TT + row);
      const float4 u = __ldcg(a.part + (slot * (HD / 4) + i) * TT + row), v = __ldcg(a.part + (slot * (HD / 4) + i + 1) * TT + row);
      const float now = fmaxf(m, x.x), ref = now == -CUDART_INF_F ? 0.f : now, old = ex2(m - ref), wt = ex2(x.x - ref);
      m = now;
      l = l * old + wt * x.y;
      acc[0] = acc[0] * old + wt * u.x; acc[1] = acc[1] * old + wt * u.y; acc[2] = acc[2] * old + wt * u.z; acc[3] = acc[3] * old + wt * u.w;
      acc[4] = acc[4] * old + wt * v.x; acc[5] = acc[5] * old + wt * v.y; acc[6] = acc[6] * old + wt * v.z; acc[7] = acc[7] * old + wt * v.w;
    }
  }
  ml_s[group][row] = make_float2(m, l);
  o_s[group][0][row] = make_float4(acc[0], acc[1], acc[2], acc[3]);
  o_s[group][1][row] = make_float4(acc[4], acc[5], acc[6], acc[7]);
  __syncthreads();
  // pairs of columns, those of a row by neighbouring threads
  constexpr int PAIRS = SPLIT ? 4 : 16;
  for (int e = threadIdx.x; e < TT * PAIRS; e += GROUPS * TT) {
    const int out_row = e / PAIRS, pair = e % 4, g0 = SPLIT ? 0 : e % PAIRS / 4, r = tile * TT + out_row;
    if (out_row >= n_rows) continue;
    float mm = -CUDART_INF_F, ll = 0.f, s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int g = 0; g < EACH; ++g) mm = fmaxf(mm, ml_s[g0 + g][out_row].x);
    const float ref = mm == -CUDART_INF_F ? 0.f : mm;
#pragma unroll
    for (int g = 0; g < EACH; ++g) {
      const float wt = ex2(ml_s[g0 + g][out_row].x - ref);
      const float2 v = reinterpret_cast<const float2*>(&o_s[g0 + g][pair >> 1][out_row])[pair & 1];
      ll += wt * ml_s[g0 + g][out_row].y;
      s0 += wt * v.x;
      s1 += wt * v.y;
    }
    const float inv = ll == 0.f ? 0.f : 1.f / ll;
    *reinterpret_cast<uint32_t*>(a.out + b * a.o_sb + (r / G) * a.o_st + (long long)(hk * G + r % G) * HD + blockIdx.y * (SPLIT ? 8 : 32) + (g0 * 4 + pair) * 2) =
        pack16(false, s0 * inv, s1 * inv);
  }
}

template <int HD, bool Q8>
int run(const Args& p, void* stream) {
  using C = Wide<HD, Q8>;
  static_assert(HD * TT * 4 <= 2 * C::STAGES * C::TILE, "a cluster's part takes the rings' place");
  static_assert(C::SMEM <= 222 * 1024 && C::CPT * CHUNK == KB * C::RB && C::Q_COL + HD / 2 <= 512 && SCALES >= C::STAGES + C::NB, "shared memory of a CTA");
  static std::atomic<unsigned long long> configured{0};   // a bit per device
  int dev = 0;
  MESH_CUDA_OK(cudaGetDevice(&dev));
  if (!(configured.load() >> (dev & 63) & 1)) {
    MESH_CUDA_OK(cudaFuncSetAttribute(wide_kernel<HD, Q8>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    configured.fetch_or(1ull << (dev & 63));
  }
  MESH_CUDA_OK(launch(wide_kernel<HD, Q8>, dim3(grid_of(p)), THREADS, C::SMEM, stream, p));
  if (p.part) {
    const unsigned items = (unsigned)(p.B * p.kv_heads * p.tiles);
    if (p.shares > 8ll * items) MESH_CUDA_OK(launch(wide_join_kernel<HD, true>, dim3(items, HD / 8), GROUPS * TT, 0, stream, p));
    else MESH_CUDA_OK(launch(wide_join_kernel<HD, false>, dim3(items, HD / 32), GROUPS * TT, 0, stream, p));
  }
  return 0;
}

}  // namespace

int wide_clusters(int head_dim, bool q8, int ranks) {
#define MESH_CLUSTERS(HD, Q8) clusters_at_once<THREADS, Wide<HD, Q8>::SMEM>(wide_kernel<HD, Q8>, ranks)
  if (q8) return head_dim == 64 ? MESH_CLUSTERS(64, true) : head_dim == 128 ? MESH_CLUSTERS(128, true) : MESH_CLUSTERS(256, true);
  return head_dim == 64 ? MESH_CLUSTERS(64, false) : head_dim == 128 ? MESH_CLUSTERS(128, false) : MESH_CLUSTERS(256, false);
#undef MESH_CLUSTERS
}

int run_wide(const Args& p, int head_dim, bool q8, void* stream) {
  switch (head_dim * 2 + q8) {
    case 128: return run<64, false>(p, stream);
    case 129: return run<64, true>(p, stream);
    case 256: return run<128, false>(p, stream);
    case 257: return run<128, true>(p, stream);
    case 512: return run<256, false>(p, stream);
    default: return run<256, true>(p, stream);
  }
}

}  // namespace draft
}  // namespace mesh
