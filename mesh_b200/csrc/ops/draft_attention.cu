// Attention of drafted tokens over a cache of bf16 rows or of 8-bit codes.
//
// The T drafts of a sequence and the G query heads that share a KV head are T * G query rows over the same keys: rows
// t * G + g.  An item is 16 of them (one tile of the matrix instruction) with all keys that any of them sees.  The items' keys, in
// units of 16 a warp, are laid end to end and cut into one share per CTA, all alike: lengths differ from sequence to sequence,
// and whole items (or equal slices of each) left most SMs waiting for the longest (282 us of a case that now takes 143).  Only
// the device knows the lengths, so every CTA finds its share itself.  A CTA's warps take blocks of 16 keys in turn, each
// with a ring of its own that cp.async fills, so that nothing but the end of an item joins them.  Items that were cut are
// joined by a second kernel.
//
// Formulas.  A score is s = scale q.k; with 8-bit rows k = ks kc and v = vs vc, where kc, vc are the codes: s = (scale ks) (q.kc),
// and the weight of a value's codes is w = exp(s - m) vs; the sum of exp(s - m) is kept beside it in fp32.  The reference m of a
// row follows the maximum of s + log vs, whatever the scales are, and is moved, and the output with it, only when that has
// grown by more than 2^8: with every new maximum most blocks of 16 rows rescaled their output (59 us now, 68 then, 4 drafts).
// Codes go through the products as fp16, which holds them exactly; so do the queries, after a row is multiplied by the power of two
// that brings its largest value to 2^8..2^9 (what is smaller than 2^-32 of that is lost, less than the products' own rounding
// in fp32).  w is multiplied by 2^6 first (in m), so it stays below 2^14 and fp16 holds it in full down to 2^-20, in part down to
// 2^-30, of the largest; its rounding to 11 bits is an eighth of bf16's.  With a bf16 cache queries and values are bf16 as they are
// and w is rounded to bf16, half a step of the result's own type: over a window of 512 keys results are off by 0.0022 (root of the mean
// square, relative), and by 0.0017, their own rounding, with weights in fp32 (as the decode step's attention has them).  A second product
// with what the rounding leaves makes up for that, but takes 1 to 10 % more time (33 drafts of heads of 64 11.6 us instead of 10.8, the
// window 16.1 instead of 15.4, 16 drafts in the other kernel 96 instead of 87), and turns an infinite value that is seen into a NaN.
//
// Measured: 16 sequences of 4000 to 32767 keys, 8 KV heads of 128 in 8 bits, 4 query heads each, one token: 142 us, 4.4 TB/s of keys
// and values.  What bounds it is the issue of instructions (2.4 a clock and SM), 525 of a warp for a block of 16 keys: some 176 widen
// the codes of both sides; most of the others are spent on 16 rows of scores, weights and output of which 4 hold a query.  32 keys a
// block took the same time, with a few registers spilled.  With bf16 rows (8 x 12000 keys) 72 us, 5.6 TB/s: memory.
#include "draft_attention.cuh"

namespace mesh {
namespace draft {

constexpr int ROWS = 16;              // query rows of a tile
constexpr int KEYS = 16;              // keys of a block

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

template <int HD, bool Q8>
struct Cfg {
  static constexpr int NT = HD / 8;                       // column tiles of the output
  static constexpr int RB = Q8 ? HD : 2 * HD, NC = RB / 16;           // bytes and 16-byte chunks of a row
  static constexpr int STAGE = 2 * KEYS * RB + (Q8 ? 2 * KEYS * 4 : 0);
  // As many warps as their registers allow (half of a warp's are the output's), four where a block is 16 KB.  Heads of 128 in 8 bits:
  // With 12 warps 151 us, with 8 162; two warps to a block with half of the columns each, 16 in all, 185.
  static constexpr int WARPS = STAGE > 9000 ? 4 : HD == 256 ? 8 : HD == 128 ? 12 : 16;
  static constexpr int ROOM = 200 * 1024 / WARPS, STAGES = ROOM / STAGE > 8 ? 8 : ROOM / STAGE;
  static constexpr int RING = WARPS * STAGES * STAGE;
  static constexpr int QB = ROWS * HD * 2;
  static constexpr int UNIT = WARPS * KEYS;               // keys of a unit of work
  static constexpr int OUT_PITCH = HD + 8;                // of a row of the result in shared memory
  static constexpr int MERGE = WARPS * ROWS * HD * 4;
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

// The column that n' = 0..7 of output tile i is: the tiles are values i % VW of the column groups n' of group i / VW.
template <int VW>
__device__ __forceinline__ int column(int i, int n) { return ((i / VW) * 8 + n) * VW + i % VW; }

template <int HD, bool Q8>
__global__ void __launch_bounds__(Cfg<HD, Q8>::WARPS * 32, 1) attention_kernel(const __grid_constant__ Args a) {
  using C = Cfg<HD, Q8>;
  constexpr int RB = C::RB, NC = C::NC, STAGES = C::STAGES, PER = C::PER, VW = C::VW, NT = C::NT;
  constexpr int KI = HD / (4 * PER);                      // chunks of a key per lane
  extern __shared__ __align__(128) uint8_t smem[];
  uint4* q_s = reinterpret_cast<uint4*>(smem);            // [k step][lane]: operand A of the scores
  __shared__ float unit_s[ROWS], weight_s[C::WARPS][ROWS], m_s[ROWS], l_s[ROWS];
  __shared__ float2 ml_s[C::WARPS][ROWS];
  __shared__ Walk walk_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = lane >> 2, t4 = lane & 3;
  uint8_t* ring = smem + C::QB + warp * (STAGES * C::STAGE);
  const uint32_t ring_u = smem_u32(ring);
  const int G = a.q_heads / a.kv_heads;
  griddep_wait();
  griddep_launch_dependents();

  if (warp == 0) begin_walk(a, &walk_s);
  __syncthreads();
  Walk walk = walk_s;
  for (Stretch y; next(a, walk, y);) {
  const Stretch x = y;
  const Seq s = x.s;
  const int b = x.b, hk = x.hk, tile = x.tile, n_rows = x.n_rows, k_lo = x.k_lo, k_hi = x.k_hi;
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

  // ---- queries: 4 consecutive values of a row are two words of a lane and k step, in the order the keys' chunks have them
  for (int i = warp; i < ROWS; i += C::WARPS) {
    const int r = tile * ROWS + i, t = r / G, h = hk * G + r % G;
    const __nv_bfloat16* src = a.q + b * a.q_sb + t * a.q_st + (long long)h * HD;
    const bool vec = (reinterpret_cast<uintptr_t>(src) & 7) == 0;
    constexpr int PARTS = (HD + 127) / 128;
    uint2 x[PARTS];
    float top = 0.f;
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      x[p] = make_uint2(0, 0);
      const int col = p * 128 + lane * 4;
      if (i < n_rows && col < HD) {
        if (vec) {
          x[p] = *reinterpret_cast<const uint2*>(src + col);
        } else {
          const unsigned short* u = reinterpret_cast<const unsigned short*>(src + col);
          x[p] = make_uint2(u[0] | (uint32_t)u[1] << 16, u[2] | (uint32_t)u[3] << 16);
        }
      }
      top = fmaxf(fmaxf(top, fmaxf(fabsf(__uint_as_float(x[p].x << 16)), fabsf(__uint_as_float(x[p].x & 0xffff0000u)))),
                  fmaxf(fabsf(__uint_as_float(x[p].y << 16)), fabsf(__uint_as_float(x[p].y & 0xffff0000u))));
    }
    float up = 1.f;
    if (Q8) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      // the power of two that brings it to 2^8..2^9; bounded, so that neither it nor its inverse leaves fp32
      up = ldexpf(1.f, top > 0.f ? min(max(8 - ilogbf(top), -110), 110) : 0);
    }
    if (lane == 0) unit_s[i] = up;
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      const int col = p * 128 + lane * 4;
      if (col < HD) {
        const int chunk = col / PER, step = chunk / 4 * (PER / 4) + col % PER / 4;
        uint32_t* w = reinterpret_cast<uint32_t*>(q_s + step * 32 + (i & 7) * 4 + chunk % 4) + (i >> 3);
        if (Q8) {
          w[0] = pack16(true, __uint_as_float(x[p].x << 16) * up, __uint_as_float(x[p].x & 0xffff0000u) * up);
          w[2] = pack16(true, __uint_as_float(x[p].y << 16) * up, __uint_as_float(x[p].y & 0xffff0000u) * up);
        } else {
          w[0] = x[p].x;
          w[2] = x[p].y;
        }
      }
    }
  }
  __syncthreads();
  const float q_unit[2] = {a.scale_log2 / unit_s[n], a.scale_log2 / unit_s[n + 8]};

  // ---- what this lane's two rows see
  int row_lo[2];
  unsigned long long vis[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int t = min((tile * ROWS + n + 8 * j) / G, a.T - 1);
    vis[j] = a.visible ? (unsigned long long)a.visible[(long long)b * a.T + t] : t >= 63 ? ~0ull : (2ull << t) - 1;
    row_lo[j] = a.window > 0 ? max(0, s.pos + max(__popcll(vis[j]), 1) - a.window) : 0;
  }
  const int free_lo = a.window > 0 ? max(0, s.pos + 64 - a.window) : 0;      // from here to pos every row sees every key

  float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f};
  float o[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
  constexpr float LIFT = Q8 ? 6.f : 0.f, LAG = 8.f;

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
    // The reference moves only when some score has grown by more than 2^LAG (also at the first key that is seen)
    if (__any_sync(0xffffffffu, top[0] - LIFT > m[0] + LAG || top[1] - LIFT > m[1] + LAG)) {
      float alpha[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 1));
        top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 2));
        const float now = top[j] - LIFT > m[j] + LAG ? top[j] - LIFT : m[j];
        alpha[j] = m[j] == now ? 1.f : ex2(m[j] - now);   // nothing seen before: 0
        m[j] = now;
      }
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

  // ---- join the warps: the ring's memory holds every warp's output as its fragments lie, [warp][tile of 8 columns][lane]
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    l[j] += __shfl_xor_sync(0xffffffffu, l[j], 1);
    l[j] += __shfl_xor_sync(0xffffffffu, l[j], 2);
    if (t4 == 0) ml_s[warp][n + 8 * j] = make_float2(m[j], l[j]);
  }
  __syncthreads();                                        // every warp is done with its ring
  float4* o_s = reinterpret_cast<float4*>(smem + C::QB);
#pragma unroll
  for (int i = 0; i < NT; ++i) o_s[(warp * NT + i) * 32 + lane] = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
  if (threadIdx.x < ROWS) {
    const int r = threadIdx.x;
    float mm = -CUDART_INF_F, ll = 0.f;
#pragma unroll
    for (int w = 0; w < C::WARPS; ++w) mm = fmaxf(mm, ml_s[w][r].x);
    const float ref = mm == -CUDART_INF_F ? 0.f : mm;
#pragma unroll
    for (int w = 0; w < C::WARPS; ++w) {
      const float wt = ex2(ml_s[w][r].x - ref);           // 0 for a warp that saw no key; its sum may be NaN
      weight_s[w][r] = wt;
      ll += wt * ml_s[w][r].y;
    }
    m_s[r] = mm;
    l_s[r] = ll;
  }
  __syncthreads();
  const bool whole = x.whole;
  const int slot = x.slot;
  __nv_bfloat16* row_s = reinterpret_cast<__nv_bfloat16*>(smem);          // the queries' memory and, after a barrier, more
  constexpr int TURNS = (NT + C::WARPS - 1) / C::WARPS;   // tiles of the output that a warp sums
  float4 sum[TURNS];
#pragma unroll
  for (int y = 0; y < TURNS; ++y) {
    const int i = y * C::WARPS + warp;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < NT) {
#pragma unroll
      for (int w = 0; w < C::WARPS; ++w) {
        const float w0 = weight_s[w][n], w1 = weight_s[w][n + 8];
        const float4 v = o_s[(w * NT + i) * 32 + lane];
        acc.x += w0 * v.x; acc.y += w0 * v.y; acc.z += w1 * v.z; acc.w += w1 * v.w;
      }
      if (!whole && !a.cluster) a.part[((long long)slot * NT + i) * 32 + lane] = acc;
    }
    sum[y] = acc;
  }
  if (!whole && a.cluster) {                              // for the cluster's CTAs
    __syncthreads();
#pragma unroll
    for (int y = 0; y < TURNS; ++y)
      if (y * C::WARPS + warp < NT) o_s[(y * C::WARPS + warp) * 32 + lane] = sum[y];
    if (threadIdx.x < ROWS) ml_s[0][threadIdx.x] = make_float2(m_s[threadIdx.x], l_s[threadIdx.x]);
  } else if (!whole) {
    if (threadIdx.x < ROWS) a.part_ml[slot * ROWS + threadIdx.x] = make_float2(m_s[threadIdx.x], l_s[threadIdx.x]);
  } else {
    __syncthreads();
    const float i0 = l_s[n] == 0.f ? 0.f : 1.f / l_s[n], i1 = l_s[n + 8] == 0.f ? 0.f : 1.f / l_s[n + 8];
#pragma unroll
    for (int y = 0; y < TURNS; ++y) {
      const int i = y * C::WARPS + warp;
      if (i >= NT) continue;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = column<C::VW>(i, 2 * t4 + e);
        row_s[n * C::OUT_PITCH + col] = __float2bfloat16_rn((e ? sum[y].y : sum[y].x) * i0);
        row_s[(n + 8) * C::OUT_PITCH + col] = __float2bfloat16_rn((e ? sum[y].w : sum[y].z) * i1);
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n_rows * (HD / 2); i += C::WARPS * 32) {
      const int row = i / (HD / 2), d = i % (HD / 2) * 2, r = tile * ROWS + row;
      *reinterpret_cast<__nv_bfloat162*>(a.out + b * a.o_sb + (r / G) * a.o_st + (long long)(hk * G + r % G) * HD + d) =
          *reinterpret_cast<const __nv_bfloat162*>(row_s + row * C::OUT_PITCH + d);
    }
  }
  __syncthreads();                                        // shared memory is the next item's
  }

  // ---- a cluster's item that was cut: each CTA joins some of the tiles of columns
  const int ranks = walk.ranks;
  if (ranks <= 1) return;                                 // the same in all CTAs of the cluster; 0 without clusters
  cluster_sync_all();
  const Item x = item_of_cluster(a);
  const int n_rows = sequence(a, x.b).count * G - x.tile * ROWS;
  const uint32_t o_at = smem_u32(smem + C::QB), ml_at = smem_u32(ml_s);
  for (int i = warp * a.cluster + blockIdx.x % a.cluster; i < NT; i += C::WARPS * a.cluster) {
    float2 u[MOST_RANKS][2];
    float4 v[MOST_RANKS];
    float mm[2] = {-CUDART_INF_F, -CUDART_INF_F}, ll[2] = {0.f, 0.f};
#pragma unroll
    for (int r = 0; r < MOST_RANKS; ++r) {
      if (r >= ranks) break;
      u[r][0] = cluster_load2(ml_at + n * 8, r);
      u[r][1] = cluster_load2(ml_at + (n + 8) * 8, r);
      v[r] = cluster_load4(o_at + (i * 32 + lane) * 16, r);
    }
#pragma unroll
    for (int r = 0; r < MOST_RANKS; ++r) {
      if (r >= ranks) break;
      mm[0] = fmaxf(mm[0], u[r][0].x);
      mm[1] = fmaxf(mm[1], u[r][1].x);
    }
    const float ref[2] = {mm[0] == -CUDART_INF_F ? 0.f : mm[0], mm[1] == -CUDART_INF_F ? 0.f : mm[1]};
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < MOST_RANKS; ++r) {
      if (r >= ranks) break;
      const float w0 = ex2(u[r][0].x - ref[0]), w1 = ex2(u[r][1].x - ref[1]);
      ll[0] += w0 * u[r][0].y;
      ll[1] += w1 * u[r][1].y;
      acc.x += w0 * v[r].x; acc.y += w0 * v[r].y; acc.z += w1 * v[r].z; acc.w += w1 * v[r].w;
    }
    const float i0 = ll[0] == 0.f ? 0.f : 1.f / ll[0], i1 = ll[1] == 0.f ? 0.f : 1.f / ll[1];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int row = n + 8 * y, r = x.tile * ROWS + row;
      if (row >= n_rows) continue;
      __nv_bfloat16* dst = a.out + x.b * a.o_sb + (r / G) * a.o_st + (long long)(x.hk * G + r % G) * HD;
      dst[column<C::VW>(i, 2 * t4)] = __float2bfloat16_rn(y ? acc.z * i1 : acc.x * i0);
      dst[column<C::VW>(i, 2 * t4 + 1)] = __float2bfloat16_rn(y ? acc.w * i1 : acc.y * i0);
    }
  }
  cluster_sync_all();                                     // the others have read this CTA's part
}

// Joins the shares of the items that were cut.  SPLIT: a CTA per item and tile of 8 columns, whose warps take the shares in turn (few items
// in many shares); else a CTA per item, whose warps take the tiles of columns.
template <int HD, bool Q8, bool SPLIT>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Args a) {
  using C = Cfg<HD, Q8>;
  constexpr int NT = HD / 8, EACH = SPLIT ? 8 : 1;        // warps among which an item's shares are dealt
  __shared__ int c_s[3];
  __shared__ float m_s[8][ROWS], l_s[8][ROWS];
  __shared__ float4 o_s[8][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = lane >> 2, t4 = lane & 3, G = a.q_heads / a.kv_heads;
  const int tile = blockIdx.x % a.tiles, hk = blockIdx.x / a.tiles % a.kv_heads, b = blockIdx.x / a.tiles / a.kv_heads;
  // All wait: what comes after this kernel relies on the one before it.  And none looks at the lengths before: they are older than
  // that kernel, but only the wait keeps a read from finding what its line held before them.
  griddep_launch_dependents();
  griddep_wait();
  if (warp == 0) shares_of_item(a, b, hk, tile, c_s);
  __syncthreads();
  const int c0 = c_s[0], c1 = c_s[1], odd = c_s[2];
  if (c0 == c1) return;                                   // whole in one CTA, or not there
  const int n_rows = sequence(a, b).count * G - tile * ROWS;
  for (int i = SPLIT ? blockIdx.y : warp; i < NT; i += SPLIT ? NT : 8) {
    float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f};
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = c0 + (SPLIT ? warp : 0); c <= c1; c += EACH * 4) {
      float2 x[4][2];
      float4 v[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int cc = c + EACH * y;
        const long long slot = 2 * cc + (cc == c0 ? odd : 0);
        x[y][0] = x[y][1] = make_float2(-CUDART_INF_F, 0.f);
        v[y] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (cc <= c1) {
          x[y][0] = __ldcg(a.part_ml + slot * ROWS + n);
          x[y][1] = __ldcg(a.part_ml + slot * ROWS + n + 8);
          v[y] = __ldcg(a.part + (slot * NT + i) * 32 + lane);
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float now = m[j];
#pragma unroll
        for (int y = 0; y < 4; ++y) now = fmaxf(now, x[y][j].x);
        const float ref = now == -CUDART_INF_F ? 0.f : now, old = ex2(m[j] - ref);
        m[j] = now;
        l[j] *= old;
        if (j == 0) { acc.x *= old; acc.y *= old; } else { acc.z *= old; acc.w *= old; }
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float wt = ex2(x[y][j].x - ref);
          l[j] += wt * x[y][j].y;
          if (j == 0) { acc.x += wt * v[y].x; acc.y += wt * v[y].y; } else { acc.z += wt * v[y].z; acc.w += wt * v[y].w; }
        }
      }
    }
    o_s[warp][lane] = acc;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (t4 == 0) { m_s[warp][n + 8 * j] = m[j]; l_s[warp][n + 8 * j] = l[j]; }
    if (SPLIT) __syncthreads();
    else __syncwarp();
    // 16 rows x 8 columns; of a whole CTA or of this warp's own sums
    for (int e = SPLIT ? threadIdx.x : lane; e < ROWS * 8; e += SPLIT ? 256 : 32) {
      const int row = e >> 3, c = e & 7, r = tile * ROWS + row, w0 = SPLIT ? 0 : warp;
      if (row >= n_rows) continue;
      float mm = -CUDART_INF_F, ll = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < EACH; ++w) mm = fmaxf(mm, m_s[w0 + w][row]);
      const float ref = mm == -CUDART_INF_F ? 0.f : mm;
#pragma unroll
      for (int w = 0; w < EACH; ++w) {
        const float wt = ex2(m_s[w0 + w][row] - ref);
        ll += wt * l_s[w0 + w][row];
        sum += wt * reinterpret_cast<const float*>(&o_s[w0 + w][(row & 7) * 4 + (c >> 1)])[2 * (row >> 3) + (c & 1)];
      }
      a.out[b * a.o_sb + (r / G) * a.o_st + (long long)(hk * G + r % G) * HD + column<C::VW>(i, c)] = __float2bfloat16_rn(ll == 0.f ? 0.f : sum / ll);
    }
    __syncwarp();
  }
}

// Units that a share may be longer for the sake of whole pieces: of 128 to 256 keys, and of 64 of the other kernel.  KV heads of 128 in 8
// bits, 4 heads a group, 8 sequences: single tokens over 12000 keys 57.7 us cut equally, 60.4 in pieces 5 longer; 64 drafts over 4000
// keys 99.2 us and, in pieces 9 longer, 92.6.
constexpr int FEW = 4, WIDE_FEW = 12;
// Units that the longest share of a cluster's item may have beyond an equal one, with the cache filled: what the second kernel and cut items
// cost.  8 KV heads of 128 in 8 bits, 4 heads a group, with clusters and with the second kernel: one token of one sequence over 1000
// keys 9.0 and 10.6 us, 8000 keys (3.0 units) 16.2 and 16.0; 16 sequences over 2000 keys (1.5) 23.0 and 26.9, 8000 keys (5.7) 62.7 and
// 60.9; 64 drafts of 4 sequences over 4000 keys (4.2) 52.8 and 58.2, 8000 keys (8.4) 88.5 and 80.9; 32 of one over 4000 keys
// (4.4) 26.6 and 25.6.
constexpr double LONGER = 3, WIDE_LONGER = 4.3;

static int clusters(const MeshKvCache* c, bool w, int ranks) {
  const bool q8 = c->bits == 8;
  if (w) return wide_clusters(c->head_dim, q8, ranks);
#define MESH_CLUSTERS(HD, Q8) clusters_at_once<Cfg<HD, Q8>::WARPS * 32, Cfg<HD, Q8>::SMEM>(attention_kernel<HD, Q8>, ranks)
  if (q8) return c->head_dim == 64 ? MESH_CLUSTERS(64, true) : c->head_dim == 128 ? MESH_CLUSTERS(128, true) : MESH_CLUSTERS(256, true);
  return c->head_dim == 64 ? MESH_CLUSTERS(64, false) : c->head_dim == 128 ? MESH_CLUSTERS(128, false) : MESH_CLUSTERS(256, false);
#undef MESH_CLUSTERS
}

static int unit_of(const MeshKvCache* c, bool w) {
  const bool q8 = c->bits == 8;
  if (w) return WIDE_UNIT;
  return c->head_dim == 64 ? (q8 ? Cfg<64, true>::UNIT : Cfg<64, false>::UNIT)
       : c->head_dim == 128 ? (q8 ? Cfg<128, true>::UNIT : Cfg<128, false>::UNIT) : (q8 ? Cfg<256, true>::UNIT : Cfg<256, false>::UNIT);
}
static int tiles_of(const MeshKvCache* c, const MeshDraftAttention* a, bool w) {
  const int rows = w ? WIDE_ROWS : ROWS;
  return (a->T * (a->q_heads / c->kv_heads) + rows - 1) / rows;
}
// Units of keys that the longest sequence may have.
static long long longest_of(const MeshKvCache* c, const MeshDraftAttention* a, bool w) {
  long long keys = c->max_seq;
  if (a->window > 0 && (long long)a->window + a->T < keys) keys = (long long)a->window + a->T;
  return (keys + unit_of(c, w) - 1) / unit_of(c, w);
}
// CTAs of a cluster that has an item; 0: the keys are cut into shares of all.
static int ranks_of(const MeshKvCache* c, const MeshDraftAttention* a, bool w) {
  const long long items = (long long)c->B * c->kv_heads * tiles_of(c, a, w), longest = longest_of(c, a, w), most = sm_count();
  if (a->splits > 0 || items > most) return 0;
  for (int ranks = MOST_RANKS; ranks >= 1; --ranks) {
    if (ranks > longest || ranks * items > most || (ranks > 1 && clusters(c, w, ranks) < items)) continue;
    return longest * (1.0 / ranks - 1.0 * items / most) <= (w ? WIDE_LONGER : LONGER) ? ranks : 0;
  }
  return 0;
}

// The kernel for many rows, with tiles of 128, from three tiles of 16 on: it has a longer start and end, and this one fetches the
// keys once per tile.  Eight sequences in caches half to wholly filled, 8 KV heads of 128 in 8 bits, 4 heads a group, this kernel and the
// other one: 8 drafts in caches of 2000 keys 21.8 and 29.7 us, of 6000 55.8 and 60.2, of 16000 100 and 119; 12 drafts in full ones of 500 keys 24.7
// and 17.0, of 12000 136 and 121.  With bf16 rows two full tiles are where they meet: 8 drafts in caches of 2000 keys 21.3 and 26.5 us, of 6000
// 55.3 and 53.7, of 12000 93.8 and 83.8 (heads of 256: 18.8 and 21.8, 39.5 and 38.5, 57.2 and 55.5); 5 drafts, of which some sequences have one
// tile, in caches of 12000 keys of 128 65.8 and 82.4.  The host knows how long a cache is, not how full: the kernel that wins in all
// shorter contexts has them too.
// But where clusters have all tiles of 16 at once and a CTA only a few units, the shorter start counts: 16 drafts of 4 sequences over
// 500 keys 10.8 and 15.7 us, over 1000 (6 units) 14.6 and 16.7, over 2000 (11) 21.4 and 21.0 (bf16: 14.2 and 14.3, 21.2 and 18.0).
constexpr int UNITS = 6;
static bool wide(const MeshKvCache* c, const MeshDraftAttention* a) {
  if (a->T * (a->q_heads / c->kv_heads) <= 2 * ROWS) return false;
  return longest_of(c, a, false) > UNITS * ranks_of(c, a, false);
}

static void cut(const MeshKvCache* c, const MeshDraftAttention* a, Args& p) {
  const bool w = wide(c, a);
  p.rows = w ? WIDE_ROWS : ROWS;
  p.unit = unit_of(c, w);
  p.tiles = tiles_of(c, a, w);
  // CTAs: one per SM, or per unit of work where the longest sequences have fewer
  const long long units = (long long)c->B * c->kv_heads * p.tiles * longest_of(c, a, w);
  const long long most = a->splits > 0 ? a->splits : sm_count();
  p.shares = (int)(units < most ? units : most);
  p.few = a->splits > 0 ? 0 : w ? WIDE_FEW : FEW;
  p.cluster = ranks_of(c, a, w);
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

template <int HD, bool Q8>
static int run(const Args& p, void* stream) {
  using C = Cfg<HD, Q8>;
  static_assert(C::STAGES >= 2 && C::SMEM <= 224 * 1024 && ROWS * C::OUT_PITCH * 2 <= C::SMEM, "ring of a warp");
  static std::atomic<unsigned long long> configured{0};   // a bit per device
  int dev = 0;
  MESH_CUDA_OK(cudaGetDevice(&dev));
  if (!(configured.load() >> (dev & 63) & 1)) {
    MESH_CUDA_OK(cudaFuncSetAttribute(attention_kernel<HD, Q8>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    configured.fetch_or(1ull << (dev & 63));
  }
  MESH_CUDA_OK(launch(attention_kernel<HD, Q8>, dim3(grid_of(p)), C::WARPS * 32, C::SMEM, stream, p));
  if (p.part) {
    const unsigned items = (unsigned)(p.B * p.kv_heads * p.tiles);
    if (p.shares > 2ll * items) MESH_CUDA_OK(launch(join_kernel<HD, Q8, true>, dim3(items, HD / 8), 256, 0, stream, p));
    else MESH_CUDA_OK(launch(join_kernel<HD, Q8, false>, dim3(items), 256, 0, stream, p));
  }
  return 0;
}

}  // namespace draft
}  // namespace mesh

extern "C" long long mesh_draft_attention_scratch(const MeshKvCache* c, const MeshDraftAttention* a) {
  using namespace mesh::draft;
  if (check(c, a)) return -1;
  Args p;
  cut(c, a, p);
  return p.shares <= 1 || p.cluster ? 0 : 2ll * p.shares * p.rows * (c->head_dim + 2);
}

extern "C" int mesh_draft_attention(const MeshKvCache* c, const MeshDraftAttention* a, void* stream) {
  using namespace mesh;
  using namespace mesh::draft;
  if (int rc = check(c, a)) return rc;
  if (c->B == 0 || a->T == 0) return 0;
  if (((uintptr_t)a->q % 2) || ((uintptr_t)a->out % 4) || a->o_sb % 2 || a->o_st % 2)
    return set_error(-2, "draft_attention: rows of the output must start on a multiple of 4 bytes");
  Args p;
  memset(&p, 0, sizeof(p));
  p.q = (const __nv_bfloat16*)a->q; p.out = (__nv_bfloat16*)a->out;
  p.q_sb = a->q_sb; p.q_st = a->q_st; p.o_sb = a->o_sb; p.o_st = a->o_st;
  p.k = (const uint8_t*)c->k; p.v = (const uint8_t*)c->v; p.k_scale = c->k_scale; p.v_scale = c->v_scale;
  p.pos = a->pos; p.counts = a->counts; p.visible = a->visible;
  p.B = c->B; p.T = a->T; p.q_heads = a->q_heads; p.kv_heads = c->kv_heads; p.max_seq = c->max_seq; p.window = a->window;
  p.status = (Status*)a->status;
  cut(c, a, p);
  if ((long long)c->B * c->kv_heads * p.tiles * ((c->max_seq + p.unit - 1) / p.unit + 1) > 0x7fffffff || p.shares > 0x3fffffff)
    return set_error(-2, "draft_attention: too many rows and keys for one call");
  p.scale_log2 = a->scale * 1.4426950408889634f;
  if (p.shares > 1 && !p.cluster) {
    if (!a->scratch || (uintptr_t)a->scratch % 16) return set_error(-2, "draft_attention: scratch memory must be given and start on a multiple of 16 bytes");
    p.part = (float4*)a->scratch;
    p.part_ml = (float2*)(a->scratch + 2ll * p.shares * p.rows * c->head_dim);
  }
  if (wide(c, a)) return run_wide(p, c->head_dim, c->bits == 8, stream);
  switch (c->head_dim * 2 + (c->bits == 8)) {
    case 128: return run<64, false>(p, stream);
    case 129: return run<64, true>(p, stream);
    case 256: return run<128, false>(p, stream);
    case 257: return run<128, true>(p, stream);
    case 512: return run<256, false>(p, stream);
    default: return run<256, true>(p, stream);
  }
}
