// What the two kernels for the attention of drafts have in common: their arguments, what a sequence's rows see, and how the work is
// cut into shares.
#pragma once
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

struct Args {
  const __nv_bfloat16* q; __nv_bfloat16* out; long long q_sb, q_st, o_sb, o_st;
  const uint8_t* k; const uint8_t* v; const float* k_scale; const float* v_scale;
  const int* pos; const int* counts; const long long* visible;
  int B, T, q_heads, kv_heads, max_seq, window;
  int rows, unit, tiles;              // query rows of a tile, keys of a unit of work, most tiles of a (sequence, KV head)
  float scale_log2;                   // scale * log2(e): exponentials are powers of two
  float4* part; float2* part_ml;      // two slots per CTA: the output as its threads hold it, and {m, l} of the rows
  int shares;                         // CTAs of the attention kernel
  int few;                            // see cut_work; 0: equal shares in any case
  int cluster;                        // CTAs of an item, a cluster (see item_of_cluster); 0: shares of all keys, and a kernel that joins them
  Status* status;
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
  s.pos = min(max(a.pos[b], 0), a.max_seq);
  s.count = a.counts ? min(a.counts[b], a.T) : a.T;
  s.hi = min(s.pos + max(s.count, 0), a.max_seq);
  s.lo = a.window > 0 ? max(0, s.pos - a.window + 1) : 0;          // the root's; its descendants see less
  return s;
}

// How the work is cut.  Sequence b has `tiles` tiles of query rows per KV head and `units` units of keys; its items follow one
// another, KV head by KV head, tile by tile.  All units together are fewer than 2^31 (checked before the launch).
struct Load {
  Seq s; int tiles, units, work;
};
__device__ __forceinline__ int whole_pieces(int units, int piece) { return piece > 1 ? (units + piece - 1) / piece * piece : units; }
// piece: see cut_work; the units of an item are counted up to a multiple of it.
__device__ __forceinline__ Load load_of(const Args& a, int b, int piece) {
  Load l;
  l.s = sequence(a, b);
  const int rows = max(l.s.count, 0) * (a.q_heads / a.kv_heads);
  l.tiles = (rows + a.rows - 1) / a.rows;
  l.units = whole_pieces(max(1, (l.s.hi - l.s.lo + a.unit - 1) / a.unit), piece);      // rows that see nothing are written too
  l.work = l.tiles * l.units * a.kv_heads;
  return l;
}
// The shares are `per` units each, the first `more` of one more.  A warp makes the cut: lane i also keeps tiles (all KV heads') and units
// of sequence i, so that what follows need not fetch the lengths again.
struct Cut {
  int total, shares, per, more, piece, tiles, units;
};
__device__ __forceinline__ int share_begin(const Cut& c, int i) { return i * c.per + min(i, c.more); }
__device__ __forceinline__ int share_of(const Cut& c, int w) {
  const int edge = c.more * (c.per + 1);
  return w < edge ? w / (c.per + 1) : c.more + (w - edge) / c.per;
}
// Work of sequence i0 + lane, i0 a multiple of 32.
__device__ __forceinline__ int work_of_lane(const Args& a, const Cut& c, int i0) {
  if (i0 == 0) return c.tiles * whole_pieces(c.units, c.piece);
  const int i = i0 + (threadIdx.x & 31);
  return i < a.B ? load_of(a, i, c.piece).work : 0;
}
__device__ __forceinline__ int sum_of_lanes(int v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Equal shares of all units, whatever items they end in.  A share that ends inside an item costs a partial result, written,
// read and joined, and the next one a new start: some units' time (`few` of them).  So where items cut into equal pieces, each a share, make
// the longest share at most that much longer, they are cut so.  Eight sequences, 8 KV heads of 128 in 8 bits, 4 heads a group: 8 drafts
// over 500 keys 15.0 us instead of 22.3, over 4000 keys 40.6 instead of 48.7; 64 drafts over 1500 keys 48.7 instead of 60.
__device__ __forceinline__ Cut cut_work(const Args& a) {
  const int lane = threadIdx.x & 31;
  Cut c;
  int all = 0, items = 0, longest = 1;
  c.tiles = c.units = 0;
  for (int i = lane; i < a.B; i += 32) {
    const Load l = load_of(a, i, 1);
    if (i < 32) { c.tiles = l.tiles * a.kv_heads; c.units = l.units; }
    all += l.work;
    items += l.tiles * a.kv_heads;
    if (l.tiles) longest = max(longest, l.units);
  }
  all = sum_of_lanes(all);
  items = sum_of_lanes(items);
  c.total = all;
  c.shares = max(1, min(a.shares, all));
  c.per = all / c.shares;
  c.more = all - c.per * c.shares;
  c.piece = 1;
  if (a.few == 0 || all <= a.shares || items > a.shares) return c;       // a unit each: cut at every item's end already
  longest = (int)__reduce_max_sync(0xffffffffu, (unsigned)longest);
  const int pieces = a.shares / items, piece = (longest + pieces - 1) / pieces;      // at most `pieces` of any item
  if (piece - c.per > a.few) return c;
  c.piece = piece;
  all = 0;
  for (int i0 = 0; i0 < a.B; i0 += 32) all += work_of_lane(a, c, i0);
  c.total = sum_of_lanes(all);
  c.shares = c.total / piece;
  c.per = piece;
  c.more = 0;
  return c;
}
// The sequence that unit w of the work belongs to, and the work before it.  w < total.
__device__ __forceinline__ int sequence_of(const Args& a, const Cut& c, int w, int& before) {
  const int lane = threadIdx.x & 31;
  before = 0;
  for (int i0 = 0; i0 < a.B; i0 += 32) {
    const int mine = work_of_lane(a, c, i0);
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, before + upto > w);
    if (past) {
      const int l = __ffs(past) - 1;
      before += __shfl_sync(0xffffffffu, upto - mine, l);
      return i0 + l;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return a.B;
}

// The stretches of a CTA's share, each within one item.  `begin` by warp 0, then a barrier; `next` by any thread that keeps a Walk.
struct Stretch {
  Seq s; int b, hk, tile, n_rows;     // n_rows: query rows of the tile that exist
  int k_lo, k_hi;                     // slots
  bool whole;                         // all of the item: its result is final
  int slot;                           // where it goes otherwise
};
struct Walk {
  int at, stop;                       // units, relative to the first of sequence b
  int b, piece; bool first;
  int ranks;                          // clusters: CTAs that have keys of the item
};
// Where contexts are short a second kernel would cost a third of the time: then an item is a cluster's, cut evenly among its CTAs, which
// join their results through distributed shared memory.  It may be no item, if its sequence has fewer tiles.
struct Item {
  int b, hk, tile;
};
__device__ __forceinline__ Item item_of_cluster(const Args& a) {
  const int item = blockIdx.x / a.cluster;
  return {item / a.tiles / a.kv_heads, item / a.tiles % a.kv_heads, item % a.tiles};
}
__device__ __forceinline__ void begin_walk(const Args& a, Walk* w) {
  if (a.cluster) {
    const Item x = item_of_cluster(a);
    const Load l = load_of(a, x.b, 1);
    const int rank = blockIdx.x % a.cluster, per = (l.units + a.cluster - 1) / a.cluster, first = (x.hk * l.tiles + x.tile) * l.units;
    if ((threadIdx.x & 31) == 0) {
      const bool there = x.tile < l.tiles;
      *w = {there ? first + min(rank * per, l.units) : 0, there ? first + min((rank + 1) * per, l.units) : 0, x.b, 1, true, there ? (l.units + per - 1) / per : 0};
    }
    return;
  }
  const Cut c = cut_work(a);
  if ((threadIdx.x & 31) == 0) *w = {0, 0, 0, c.piece, true, 0};
  if ((int)blockIdx.x < min(c.shares, c.total)) {
    const int w0 = share_begin(c, blockIdx.x), w1 = share_begin(c, blockIdx.x + 1);
    int before;
    const int b = sequence_of(a, c, w0, before);
    if ((threadIdx.x & 31) == 0) { w->at = w0 - before; w->stop = w1 - before; w->b = b; }
  }
}
__device__ __forceinline__ bool next(const Args& a, Walk& w, Stretch& x) {
  if (w.at >= w.stop) return false;
  Load load = load_of(a, w.b, w.piece);
  while (w.at >= load.work) {
    w.at -= load.work;
    w.stop -= load.work;
    load = load_of(a, ++w.b, w.piece);
  }
  const int item = w.at / load.units, u0 = w.at - item * load.units, u1 = min(load.units, u0 + w.stop - w.at);
  x.s = load.s;
  x.b = w.b;
  x.hk = item / load.tiles;
  x.tile = item % load.tiles;
  x.n_rows = min(load.s.count * (a.q_heads / a.kv_heads) - x.tile * a.rows, a.rows);
  x.k_lo = min(load.s.lo + u0 * a.unit, load.s.hi);
  x.k_hi = min(load.s.lo + u1 * a.unit, load.s.hi);
  x.whole = u1 - u0 == load.units;
  x.slot = 2 * blockIdx.x + (w.first ? 0 : 1);
  w.at += u1 - u0;
  w.first = false;
  return true;
}

// The shares that an item was cut into, by warp 0: c[0] .. c[1], and whether it is not the first stretch of the first of them
// (equal shares: not cut, or there is no such item).
__device__ __forceinline__ void shares_of_item(const Args& a, int b, int hk, int tile, int (&c)[3]) {
  const Cut cut = cut_work(a);
  int before = 0;
  for (int i0 = 0; i0 <= b; i0 += 32) {
    const int mine = work_of_lane(a, cut, i0);
    if (i0 + (int)(threadIdx.x & 31) < b) before += mine;
  }
  before = sum_of_lanes(before);
  int tiles = __shfl_sync(0xffffffffu, cut.tiles, b & 31) / a.kv_heads;
  int units = whole_pieces(__shfl_sync(0xffffffffu, cut.units, b & 31), cut.piece);
  if (b >= 32) {
    const Load load = load_of(a, b, cut.piece);
    tiles = load.tiles;
    units = load.units;
  }
  if ((threadIdx.x & 31) == 0) {
    c[0] = c[1] = c[2] = 0;
    if (tile < tiles) {
      const int w = before + (hk * tiles + tile) * units;
      c[0] = share_of(cut, w);
      c[1] = share_of(cut, w + units - 1);
      c[2] = share_begin(cut, c[0]) >= w ? 0 : 1;
    }
  }
}

// Four floats, or two, of another CTA's shared memory.
__device__ __forceinline__ float4 cluster_load4(uint32_t at, int cta) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(mapa_u32(at, cta)) : "memory");
  return v;
}
__device__ __forceinline__ float2 cluster_load2(uint32_t at, int cta) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(mapa_u32(at, cta)) : "memory");
  return v;
}
constexpr int MOST_RANKS = 8;         // CTAs of a cluster

template <class... P>
static cudaError_t launch(void (*kern)(P...), dim3 grid, int threads, int smem, void* stream, const Args& a) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = a.cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, a);
}

// Clusters of `ranks` CTAs that the current device runs at the same time, a CTA taking an SM: it depends on how the SMs lie together, which
// differs from device to device (sixteen of eight fit into 148 SMs, but not always into their groups).  0 if it cannot be told.
template <int THREADS, int SMEM, class... P>
static int clusters_at_once(void (*kern)(P...), int ranks) {
  static std::atomic<int> known[64][MOST_RANKS + 1];                   // one more than it; kernels of the same sizes have the same
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  std::atomic<int>& k = known[dev & 63][ranks];
  if (k.load()) return k.load() - 1;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(ranks * 64);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  k.store(n + 1);
  return n;
}

static inline unsigned grid_of(const Args& a) { return a.cluster ? (unsigned)(a.B * a.kv_heads * a.tiles * a.cluster) : (unsigned)a.shares; }

// The kernel for many query rows (draft_attention_wide.cu): rows of a tile, keys of a unit, and the call.
constexpr int WIDE_ROWS = 128, WIDE_UNIT = 64;
int run_wide(const Args& p, int head_dim, bool q8, void* stream);
int wide_clusters(int head_dim, bool q8, int ranks);

}  // namespace draft
}  // namespace mesh
