// Page bounds, and the choice of pages a one-token decode reads.
//
// page_bounds: elementwise minimum and maximum of a full page's keys, per layer and KV head.
// A page of one head is contiguous (32 KB at 128 x 128 x 16 bits). As many CTAs as the SMs hold
// walk an equal share of the (layer, page, head) list each, through a ring of kBoundsStages
// stages that bulk copies fill, so that the next blocks are on their way while one is looked
// through (16-bit types as packed pairs: half the instructions of widening them); lanes of one
// column meet by shuffles, warps in shared memory. NaN keys give NaN bounds. Bound: HBM reads
// of the keys: 256 pages x 8 heads x 4 layers (273 MB) take 49.5 us, 5.5 TB/s; a CTA per page
// (its start and the last wave) took 54, a CTA per block without the ring 61.
//
// select_pages: score(page) = max over the KV group's query heads of
//   sum_d q_d * (q_d >= 0 ? max_d : min_d),
// the most a key of the page can score; the take - 1 best full pages (ties: the lowest page)
// and the page being written, in ascending order. A cluster of 1 to 8 CTAs per (request, KV
// head) shares the pages out; their scores meet in the first CTA's shared memory.
//
// Which page is read hangs on scores next to each other, so the choice must not depend on the
// order of summation: a score is its exact sum rounded once to fp32 (products of 16-bit values
// are exact in fp32, fp32 ones keep their rounding error by an FMA; the sums carry their
// rounding errors along, Knuth's two-sum; lanes meet in 64 bits). For 16-bit types only the
// pages whose place is in doubt are summed that way: all are scored first on the tensor
// cores (the dot product of [q > 0, q < 0] with [max, min], 8 pages and 4 heads per mma, each
// bound read once), with the sum of the terms' magnitudes beside it, which bounds the error;
// pages further than that from the threshold are in or out for certain. 64 requests x 256 pages
// x 8 KV heads x 4 heads take 25 us; with maxima and minima as operands of their own (four
// mma instead of two per 16 dims) and a second search for the pages in doubt 34, exact sums of
// every page 62, conversions to 64 bits 80; the bounds' bytes need 10. Bound: the latency of a
// CTA's passes (scores 13 us, search and lists 7).
// A product outside the range of fp32 makes its page's score infinite or NaN.
//
// Bound: HBM reads of the bounds on large batches, the chain of barriers on small ones.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "chunk_schedule.cuh"

namespace hyt {

namespace {

constexpr int kBoundsThreads = 256;
constexpr int kSelectThreads = 128;

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T>
__device__ __forceinline__ void unpack16(const uint4& v, float (&f)[16 / sizeof(T)]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T* e = reinterpret_cast<const T*>(&w[i]);
      f[2 * i] = Elem<T>::to_float(e[0]);
      f[2 * i + 1] = Elem<T>::to_float(e[1]);
    }
  }
}

// Minimum and maximum of 32-bit words of one or two values, NaN if either is.
template <typename T>
struct MinMax;
template <>
struct MinMax<float> {
  static __device__ __forceinline__ uint32_t lo(uint32_t a, uint32_t b) {
    return __float_as_uint(min_nan(__uint_as_float(a), __uint_as_float(b)));
  }
  static __device__ __forceinline__ uint32_t hi(uint32_t a, uint32_t b) {
    return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
  }
};
template <>
struct MinMax<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t lo(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ uint32_t hi(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
};
template <>
struct MinMax<__half> {
  static __device__ __forceinline__ uint32_t lo(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ uint32_t hi(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
};

constexpr int kBoundsStages = 3;
constexpr int kBoundsBlock = 32 * 1024;  // most bytes of a stage

// A place in the list of blocks: a part (stage_rows rows) of a head of a page entry of a layer.
struct BoundsCursor {
  int part, head, entry, layer;
  __device__ __forceinline__ BoundsCursor(const BoundsParams& p, int64_t item) {
    part = 0;
    head = int(item % p.num_kv_heads);
    const int64_t rest = item / p.num_kv_heads;
    entry = int(rest % p.count);
    layer = int(rest / p.count);
  }
  __device__ __forceinline__ void next(const BoundsParams& p, int parts) {
    if (++part < parts) return;
    part = 0;
    if (++head < p.num_kv_heads) return;
    head = 0;
    if (++entry < p.count) return;
    entry = 0;
    ++layer;
  }
};

// CTA c of G takes items (layer, page entry, KV head) [c, c + 1) * items / G.
template <typename T>
__global__ void __launch_bounds__(kBoundsThreads) page_bounds_kernel(const BoundsParams p, int64_t items, int stage_rows) {
  constexpr int kPer = 16 / int(sizeof(T));
  constexpr int kWarps = kBoundsThreads / 32;
  extern __shared__ __align__(128) uint8_t ring[];  // [kBoundsStages][stage_rows * D], then per warp and column
  __shared__ uint64_t full[kBoundsStages];
  __shared__ int32_t page_s[kBoundsStages];  // page of the stage's block, -1: skipped
  __shared__ int abort_s;
  const int D = p.head_dim, chunks = D / kPer;  // 16-byte columns of a row (<= 64)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rows = 1 << p.page_shift, parts = (rows + stage_rows - 1) / stage_rows;
  const int stage_bytes = stage_rows * D * int(sizeof(T));
  const int64_t item0 = items * blockIdx.x / gridDim.x;
  const int64_t blocks = (items * (blockIdx.x + 1) / gridDim.x - item0) * parts;
  // [2][lo, hi][kWarps][chunks]: the warps' results of a head and of the one after
  uint4* results = reinterpret_cast<uint4*>(ring + kBoundsStages * stage_bytes);
  if (tid == 0) {
    abort_s = 0;
    for (int s = 0; s < kBoundsStages; ++s) mbar_init(&full[s], 1);
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  BoundsCursor ahead(p, item0), at = ahead;
  int64_t loaded = 0;  // blocks, of thread 0
  auto load = [&](int st) {  // thread 0: the next block into stage st
    int32_t page = p.pages[ahead.entry];
    if (page < -1 || page >= p.num_pages) {
      flag_error(p.error_word, HYT_DEVERR_PAGE_RANGE);
      page = -1;
    }
    page_s[st] = page;
    if (page >= 0) {
      const uint32_t bytes = uint32_t(min(stage_rows, rows - ahead.part * stage_rows) * D * int(sizeof(T)));
      const int64_t plane = int64_t(p.first_layer + ahead.layer) * p.num_kv_heads + ahead.head;
      mbar_arrive_expect_tx(&full[st], bytes);
      bulk_load(ring + st * stage_bytes,
                static_cast<const T*>(p.k_pool) +
                    (plane * p.capacity + (int64_t(page) << p.page_shift) + ahead.part * stage_rows) * D,
                bytes, &full[st]);
    } else {
      mbar_arrive(&full[st]);
    }
    ahead.next(p, parts);
    ++loaded;
  };
  if (tid == 0)
    for (int i = 0; i < kBoundsStages && i < blocks; ++i) load(i);
  __syncthreads();

  // columns that divide a warp's lanes: 32 / chunks rows side by side per warp; else a warp takes
  // whole rows, ceil(chunks / 32) columns per lane
  const bool side_by_side = chunks <= 32 && 32 % chunks == 0;
  const int per_warp = side_by_side ? 32 / chunks : 1, groups = kWarps * per_warp;
  const int first = side_by_side ? warp * per_warp + lane / chunks : warp;
  const int columns = side_by_side ? 1 : (chunks + 31) / 32;  // at most 2
  uint4 lo[2], hi[2];
  bool any = false;
  int st = 0, which = 0;
  uint32_t phase = 0u;
  for (int64_t i = 0; i < blocks; ++i, at.next(p, parts)) {
    const int here = min(stage_rows, rows - at.part * stage_rows);
    if (at.part == 0) any = false;
    mbar_wait(&full[st], phase, p.error_word, &abort_s);
    const int32_t page = page_s[st];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = side_by_side ? lane % chunks : lane + 32 * k;
      if (k >= columns || c >= chunks || page < 0) continue;
      const uint4* column = reinterpret_cast<const uint4*>(ring + st * stage_bytes) + c;
      bool begun = any;
#pragma unroll 4
      for (int r = first; r < here; r += groups) {
        const uint4 v = column[r * chunks];
        if (!begun) lo[k] = hi[k] = v;
        begun = true;
        lo[k].x = MinMax<T>::lo(lo[k].x, v.x), hi[k].x = MinMax<T>::hi(hi[k].x, v.x);
        lo[k].y = MinMax<T>::lo(lo[k].y, v.y), hi[k].y = MinMax<T>::hi(hi[k].y, v.y);
        lo[k].z = MinMax<T>::lo(lo[k].z, v.z), hi[k].z = MinMax<T>::hi(hi[k].z, v.z);
        lo[k].w = MinMax<T>::lo(lo[k].w, v.w), hi[k].w = MinMax<T>::hi(hi[k].w, v.w);
      }
    }
    any = any || first < here;
    const bool ends = at.part == parts - 1 && page >= 0;
    uint4* lo_s = results + which * 2 * kWarps * chunks;
    uint4* hi_s = lo_s + kWarps * chunks;
    bool mine = any;
    if (!ends) {
    } else if (side_by_side) {  // rows that exist come first: a lane without one takes its partner's
      for (int off = chunks; off < 32; off <<= 1) {
        const uint4 a = make_uint4(__shfl_xor_sync(0xffffffffu, lo[0].x, off), __shfl_xor_sync(0xffffffffu, lo[0].y, off),
                                   __shfl_xor_sync(0xffffffffu, lo[0].z, off), __shfl_xor_sync(0xffffffffu, lo[0].w, off));
        const uint4 b = make_uint4(__shfl_xor_sync(0xffffffffu, hi[0].x, off), __shfl_xor_sync(0xffffffffu, hi[0].y, off),
                                   __shfl_xor_sync(0xffffffffu, hi[0].z, off), __shfl_xor_sync(0xffffffffu, hi[0].w, off));
        const bool theirs = __shfl_xor_sync(0xffffffffu, mine ? 1 : 0, off) != 0;
        if (theirs && mine) {
          lo[0] = make_uint4(MinMax<T>::lo(lo[0].x, a.x), MinMax<T>::lo(lo[0].y, a.y), MinMax<T>::lo(lo[0].z, a.z), MinMax<T>::lo(lo[0].w, a.w));
          hi[0] = make_uint4(MinMax<T>::hi(hi[0].x, b.x), MinMax<T>::hi(hi[0].y, b.y), MinMax<T>::hi(hi[0].z, b.z), MinMax<T>::hi(hi[0].w, b.w));
        } else if (theirs) {
          lo[0] = a, hi[0] = b;
        }
        mine |= theirs;
      }
      if (lane < chunks) lo_s[warp * chunks + lane] = lo[0], hi_s[warp * chunks + lane] = hi[0];
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (lane + 32 * k < chunks) lo_s[warp * chunks + lane + 32 * k] = lo[k], hi_s[warp * chunks + lane + 32 * k] = hi[k];
    }
    // the stage has been read and the head's results are there; those of the head before last,
    // whose place the next head's take, went out before this barrier
    __syncthreads();
    if (tid == 0 && i + kBoundsStages < blocks) {
      if (*const_cast<volatile int*>(&abort_s) == 0) load(st);
      else page_s[st] = -1;  // a wait gave up: its stage may still be written, the rest is skipped
    }
    if (++st == kBoundsStages) st = 0, phase ^= 1u;
    if (!ends) continue;
    which ^= 1;
    const int used = min(kWarps, (rows + per_warp - 1) / per_warp);  // warps that had a row (of a full first part)
    const int words = chunks * 4;
    uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<T*>(p.k_bounds) +
                                                ((int64_t(p.first_layer + at.layer) * p.num_kv_heads + at.head) * p.num_pages + page) * 2 * D);
    for (int i = tid; i < 2 * words; i += kBoundsThreads) {
      const bool is_hi = i >= words;
      const int w = is_hi ? i - words : i;
      const uint32_t* from = reinterpret_cast<const uint32_t*>(is_hi ? hi_s : lo_s);
      uint32_t x = from[w];
      for (int k = 1; k < used; ++k) x = is_hi ? MinMax<T>::hi(x, from[k * words + w]) : MinMax<T>::lo(x, from[k * words + w]);
      out[i] = x;
    }
  }
  // every block was waited for above; if a wait gave up, see that no copy is in flight at the exit
  if (tid == 0 && abort_s)
    for (int64_t i = loaded > kBoundsStages ? loaded - kBoundsStages : 0; i < loaded; ++i)
      mbar_drain(&full[i % kBoundsStages], uint32_t(i / kBoundsStages) & 1u);
}

// Order-preserving unsigned key of a score; NaN ranks above everything.
__device__ __forceinline__ uint32_t score_key(float x) {
  if (isnan(x)) return 0xFFFFFFFFu;
  if (x == 0.f) x = 0.f;  // -0 ties with +0
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// A sum of fp32 terms with its rounding errors, two at a time.
struct PairSum {
  uint64_t s = 0, e = 0;  // packed pairs of +0
  __device__ __forceinline__ void add(uint64_t p) {
    const uint64_t minus = f2_pack(-1.f, -1.f);
    const uint64_t t = f2_add(s, p), bb = f2_fma(s, minus, t);   // t = s + p rounded; bb = t - s
    const uint64_t back = f2_fma(bb, minus, t);                  // t - bb
    e = f2_add(e, f2_add(f2_fma(back, minus, s), f2_fma(bb, minus, p)));
    s = t;
  }
  __device__ __forceinline__ double total() const {
    float s0, s1, e0, e1;
    f2_unpack(s, s0, s1);
    f2_unpack(e, e0, e1);
    // a sum that overflowed or met a NaN or infinity has no error term worth having
    return isfinite(s0) && isfinite(s1) ? (double(s0) + double(s1)) + (double(e0) + double(e1)) : double(s0) + double(s1);
  }
};

constexpr int kLanes = 16;  // lanes that sum one page exactly

// Key of one head's exact score of a page, on all 16 lanes of the half-warp (both halves call
// together). lo: the page's bounds.
template <typename T>
__device__ __forceinline__ uint32_t exact_key(int head_dim, const T* qh, const T* lo, int l16) {
  constexpr int kPer = 16 / int(sizeof(T));
  PairSum acc;
  for (int c = l16; c < head_dim / kPer; c += kLanes) {
    float fl[kPer], fh[kPer];
    unpack16<T>(__ldg(reinterpret_cast<const uint4*>(lo) + c), fl);
    unpack16<T>(__ldg(reinterpret_cast<const uint4*>(lo + head_dim) + c), fh);
#pragma unroll
    for (int e = 0; e < kPer; e += 2) {
      const float qa = Elem<T>::to_float(qh[c * kPer + e]), qb = Elem<T>::to_float(qh[c * kPer + e + 1]);
      const uint64_t q2 = f2_pack(qa, qb), x2 = f2_pack(qa >= 0.f ? fh[e] : fl[e], qb >= 0.f ? fh[e + 1] : fl[e + 1]);
      const uint64_t prod = f2_mul(q2, x2);
      acc.add(prod);
      if constexpr (sizeof(T) == 4) acc.e = f2_add(acc.e, f2_fma(q2, x2, f2_mul(prod, f2_pack(-1.f, -1.f))));
    }
  }
  double total = acc.total();
#pragma unroll
  for (int off = kLanes / 2; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
  return score_key(float(total));
}

// The tensor cores' fp32 accumulation of 16 products and the running sum may drop bits below
// 2^-23 of the largest of them; 2 steps of 17 terms per 32 dims for the maxima and 2 for the
// minima keep the error of a score under 2^-20 of the sum of the terms' magnitudes per dim,
// with a factor of 3 to spare.
__device__ __forceinline__ float score_slack(int head_dim, float magnitude) {
  return magnitude * float((head_dim + 31) / 32 * 32) * 9.5367432e-7f;
}

// kSteps: 16-byte chunks of a bounds row per lane of a quad (head_dim <= 32 kSteps).
template <typename T, int kSteps>
__global__ void __launch_bounds__(kSelectThreads) select_pages_kernel(const SelectParams p) {
  constexpr bool kTensor = sizeof(T) == 2;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  constexpr int kWarps = kSelectThreads / 32;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  // [last] keys, page ids and list entries (the first CTA's are used), then the bounds' ring
  uint32_t* keys = reinterpret_cast<uint32_t*>(smem_raw);
  int32_t* ids = reinterpret_cast<int32_t*>(keys) + p.ranked;
  int32_t* doubtful = ids + p.ranked;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int unit = int(blockIdx.x) / ranks;
  const int b = unit / p.num_kv_heads, g = unit - b * p.num_kv_heads;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int D = p.head_dim, group = p.num_q_heads / p.num_kv_heads;
  __shared__ int counts[2][3][kWarps], warp_count[kWarps];
  __shared__ int s_doubtful;
  __shared__ int s_magnitude;  // largest sum of magnitudes of a score, as the bits of a float
  launch_dependents();  // the attention kernel may start up; it waits for this grid's results

  const int64_t out_row = (int64_t(b) * p.num_kv_heads + g) * p.take;
  const int32_t* table = p.page_table + int64_t(b) * p.page_table_stride;
  if (kTensor && warp == 0 && lane < 2 * group && lane / 2 < group)  // q is needed right after the bounds
    asm volatile("prefetch.global.L1 [%0];" ::"l"(static_cast<const T*>(p.q) + int64_t(b) * p.q_sb +
                                                  (int64_t(g) * group + lane / 2) * p.q_sh + (lane & 1) * min(64, D - 1)));
  const int len = p.cache_lens[b];
  const int last = len >= 0 ? len >> p.page_shift : p.table_width;  // the page being written
  if (last >= p.table_width || last > kSelectMaxPages) {
    if (rank != 0) return;
    if (tid == 0 && g == 0) flag_error(p.error_word, HYT_DEVERR_TABLE_RANGE);
    for (int i = tid; i < p.take; i += kSelectThreads) p.selected[out_row + i] = p.pages[out_row + i] = -1;
    if (g == 0 && tid == 0) p.lens[b] = 0;
    return;
  }
  const int count = min(last + 1, p.take);
  if (g == 0 && rank == 0 && tid == 0)
    p.lens[b] = ((count - 1) << p.page_shift) + (len & ((1 << p.page_shift) - 1));
  if (last < p.take) {  // every page is read
    if (rank != 0) return;
    for (int i = tid; i < p.take; i += kSelectThreads) {
      p.selected[out_row + i] = i < count ? i : -1;
      p.pages[out_row + i] = i < count ? table[i] : -1;
    }
    return;
  }

  // ---- scores of the full pages 0 .. last - 1: this CTA's share
  const T* bounds = static_cast<const T*>(p.k_bounds) + (int64_t(p.layer) * p.num_kv_heads + g) * p.num_pages * 2 * D;
  const T* q0 = static_cast<const T*>(p.q) + int64_t(b) * p.q_sb + int64_t(g) * group * p.q_sh;
  auto page_at = [&](int i) {  // physical page, -1 past the end or refused
    if (i >= last) return -1;
    const int32_t page = table[i];
    if (page >= 0 && page < p.num_pages) return int(page);
    flag_error(p.error_word, HYT_DEVERR_PAGE_RANGE);
    return -1;
  };
  if (tid == 0) s_magnitude = 0, s_doubtful = 0;
  // the first CTA has started and cleared its magnitude: its shared memory may be written
  if (ranks > 1) cluster.sync();
  else __syncthreads();
  uint32_t* to = cluster.map_shared_rank(keys, 0);
  int32_t* to_id = cluster.map_shared_rank(ids, 0);
  if constexpr (kTensor) {
    // 8 pages per warp and turn: lane (n = lane / 4, j = lane % 4) reads 16-byte chunks j + 4 t
    // of page n's two rows. A operand: row n the maxima, row n + 8 the minima of page n; B
    // operand: column n the positive (n < 4) or negative values of head n % 4 of four, read the
    // same way: the order of the dims differs from memory's, alike on both sides. Of the
    // product, maxima x positive and minima x negative make the scores
    const int n = lane >> 2, j = lane & 3, chunks = D / 8;
    const int first = (rank * kWarps + warp) * 8, stride = ranks * kWarps * 8;
    float magnitude = 0.f;
    // the bounds of the next kRing - 1 turns are on their way to shared memory, every lane's
    // 16-byte pieces to its own places (nobody else reads them)
    constexpr int kRing = kSteps <= 4 ? 3 : 2;
    uint4* ring = reinterpret_cast<uint4*>(smem_raw + (p.ranked * 12 + 15) / 16 * 16) + tid;
    int ahead = first, slot = 0;
    auto fetch = [&]() {
      const int page = page_at(ahead + n);
      const uint4* lo = reinterpret_cast<const uint4*>(bounds + int64_t(max(page, 0)) * 2 * D);
#pragma unroll
      for (int t = 0; t < kSteps; ++t) {
        const int c = j + 4 * t;
        const bool there = c < chunks && page >= 0;
        cp_async16(&ring[(slot * 2 * kSteps + 2 * t) * kSelectThreads], there ? lo + c : lo, there ? 16 : 0);
        cp_async16(&ring[(slot * 2 * kSteps + 2 * t + 1) * kSelectThreads], there ? lo + chunks + c : lo, there ? 16 : 0);
      }
      cp_async_commit();
      ahead += stride;
      slot = slot + 1 == kRing ? 0 : slot + 1;
      return page;
    };
    uint32_t qw[kSteps][4];
    auto load_q = [&](int h0) {
      const T* qh = q0 + int64_t(min(h0 + (n & 3), group - 1)) * p.q_sh;
#pragma unroll
      for (int t = 0; t < kSteps; ++t) {
        const int c = j + 4 * t;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (c < chunks) {
          if (p.q_vec) {
            v = __ldg(reinterpret_cast<const uint4*>(qh) + c);
          } else {
            const uint16_t* e = reinterpret_cast<const uint16_t*>(qh + c * 8);
            v.x = e[0] | (uint32_t(e[1]) << 16);
            v.y = e[2] | (uint32_t(e[3]) << 16);
            v.z = e[4] | (uint32_t(e[5]) << 16);
            v.w = e[6] | (uint32_t(e[7]) << 16);
          }
        }
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t negative = ((w[k] & 0x80008000u) >> 15) * 0xFFFFu;  // ones where q < 0
          qw[t][k] = w[k] & (n < 4 ? ~negative : negative);
        }
      }
    };
    int ids_ahead[kRing];  // pages of this lane's n in the turns to come
#pragma unroll
    for (int k = 0; k < kRing - 1; ++k) ids_ahead[k] = fetch();
    if (group <= 4) load_q(0);
    int at = 0;
    for (int i0 = first; i0 < last; i0 += stride) {
      const int page = ids_ahead[0];
      ids_ahead[kRing - 1] = fetch();
#pragma unroll
      for (int k = 0; k < kRing - 1; ++k) ids_ahead[k] = ids_ahead[k + 1];
      cp_async_wait<kRing - 1>();
      const uint4* here = &ring[at * 2 * kSteps * kSelectThreads];
      at = at + 1 == kRing ? 0 : at + 1;
      float top = -INFINITY;  // best over the heads (lanes j = 0, 1)
      bool nan = false;
      for (int h0 = 0; h0 < group; h0 += 4) {
        if (group > 4) load_q(h0);
        float s[4] = {0.f, 0.f, 0.f, 0.f}, m[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < kSteps; ++t) {
          const uint4 l4 = here[2 * t * kSelectThreads], h4 = here[(2 * t + 1) * kSelectThreads];
          const uint32_t lw[4] = {l4.x, l4.y, l4.z, l4.w}, hw[4] = {h4.x, h4.y, h4.z, h4.w};
          constexpr uint32_t kAbs = 0x7FFF7FFFu;
#pragma unroll
          for (int w = 0; w < 4; w += 2) {
            const uint32_t x[4] = {hw[w], lw[w], hw[w + 1], lw[w + 1]};
            const uint32_t x_abs[4] = {x[0] & kAbs, x[1] & kAbs, x[2] & kAbs, x[3] & kAbs};
            mma_16816<kHalf>(s, x, qw[t][w], qw[t][w + 1]);
            mma_16816<kHalf>(m, x_abs, qw[t][w] & kAbs, qw[t][w + 1] & kAbs);
          }
        }
        // lanes j = 0, 1: maxima x heads h0 + 2 j, + 1; j = 2, 3: minima x the same heads
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float score = s[e] + __shfl_xor_sync(0xffffffffu, s[2 + e], 2);
          const float size = m[e] + __shfl_xor_sync(0xffffffffu, m[2 + e], 2);
          if (j < 2 && h0 + 2 * j + e < group) {
            nan |= isnan(score);
            top = fmaxf(top, score);
            if (i0 + n < last) magnitude = max_nan(magnitude, size);
          }
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      nan |= __shfl_xor_sync(0xffffffffu, nan ? 1 : 0, 1) != 0;
      if (j == 0 && i0 + n < last) {
        to[i0 + n] = page < 0 ? 0u : (nan ? 0xFFFFFFFFu : score_key(top));
        to_id[i0 + n] = page;
      }
    }
    cp_async_wait<0>();
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) magnitude = max_nan(magnitude, __shfl_xor_sync(0xffffffffu, magnitude, off));
    // bits of floats >= 0 are ordered like the floats, NaN above all
    if (lane == 0) atomicMax(cluster.map_shared_rank(&s_magnitude, 0), __float_as_int(magnitude) & 0x7FFFFFFF);
  } else {
    const int l16 = lane % kLanes;
    constexpr int kPages = kWarps * (32 / kLanes);  // pages a CTA scores at a time
    for (int i0 = rank * kPages; i0 < last; i0 += ranks * kPages) {
      const int i = i0 + warp * (32 / kLanes) + lane / kLanes;
      const int page = page_at(i);
      uint32_t key = 0u;
      for (int h = 0; h < group; ++h)
        key = max(key, exact_key<T>(D, q0 + int64_t(h) * p.q_sh, bounds + int64_t(max(page, 0)) * 2 * D, l16));
      if (i < last && l16 == 0) {
        to[i] = page < 0 ? 0u : key;
        to_id[i] = page;
      }
    }
  }
  if (ranks > 1) {
    cluster.sync();
    if (rank != 0) return;
  } else {
    __syncthreads();
  }

  // counts over the CTA of what each thread counted for three questions; one barrier
  int step = 0;
  auto count3 = [&](int a, int b3, int c, int (&all)[3]) {
    int mine[3];
    if (last <= 8 * kSelectThreads) {  // a warp's counts fit 10 bits each: one reduction
      const uint32_t sum = __reduce_add_sync(0xffffffffu, uint32_t(a) | uint32_t(b3) << 10 | uint32_t(c) << 20);
      mine[0] = sum & 1023u, mine[1] = (sum >> 10) & 1023u, mine[2] = sum >> 20;
    } else {
      mine[0] = __reduce_add_sync(0xffffffffu, a);
      mine[1] = __reduce_add_sync(0xffffffffu, b3);
      mine[2] = __reduce_add_sync(0xffffffffu, c);
    }
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (lane == k) counts[step & 1][k][warp] = mine[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      all[k] = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) all[k] += counts[step & 1][k][w];
    }
    ++step;
  };
  const int want = p.take - 1;  // 0 .. last
  // The largest value that at least `want` keys reach (want >= 1), two bits at a time from the
  // highest in which the keys differ: they are scores of one query, so a histogram of their
  // leading bits would pile up in one bin. `exactly`: ended early, exactly `want` keys reach it.
  bool exactly = false, settled = false;
  auto threshold_of = [&]() {
    uint32_t ones = 0xFFFFFFFFu, any = 0u;
    for (int i = tid; i < last; i += kSelectThreads) ones &= keys[i], any |= keys[i];
    ones = __reduce_and_sync(0xffffffffu, ones);
    any = __reduce_or_sync(0xffffffffu, any);
    if (lane == 0) counts[step & 1][0][warp] = int(ones), counts[step & 1][1][warp] = int(any);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) ones &= uint32_t(counts[step & 1][0][w]), any |= uint32_t(counts[step & 1][1][w]);
    ++step;
    exactly = false;
    if (ones == any) return ones;  // all keys are the same
    int bit = (31 - __clz(ones ^ any)) | 1;  // the upper bit of the pair that holds the highest difference
    uint32_t t = bit == 31 ? 0u : ones & ~((2u << bit) - 1u);
    for (; bit >= 0 && !exactly; bit -= 2) {
      const uint32_t unit = 1u << (bit - 1);
      int c[3] = {0, 0, 0}, all[3];
      for (int i = tid; i < last; i += kSelectThreads) {
        const uint32_t key = keys[i];
#pragma unroll
        for (int k = 0; k < 3; ++k) c[k] += key >= t + unit * uint32_t(k + 1) ? 1 : 0;
      }
      count3(c[0], c[1], c[2], all);
#pragma unroll
      for (int k = 2; k >= 0; --k) {
        if (all[k] >= want) {
          t += unit * uint32_t(k + 1);
          exactly = all[k] == want;
          break;
        }
      }
    }
    return t;
  };
  if (kTensor && want > 0) {
    // scores within the error of the want-th best are in doubt: those are summed exactly. Those
    // above count as the best there is, those below as the worst
    uint32_t t = threshold_of();
    if (exactly) {  // the smallest key that reaches t, instead of t itself
      uint32_t least = 0xFFFFFFFFu;
      for (int i = tid; i < last; i += kSelectThreads)
        if (keys[i] >= t) least = min(least, keys[i]);
      least = __reduce_min_sync(0xffffffffu, least);
      if (lane == 0) warp_count[warp] = int(least);
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWarps; ++w) least = min(least, uint32_t(warp_count[w]));
      t = least;
    }
    const float score = __uint_as_float((t & 0x80000000u) ? (t & 0x7FFFFFFFu) : ~t);
    const float slack = 2.f * score_slack(D, __int_as_float(s_magnitude));
    const uint32_t above0 = score_key(score + slack), below0 = score_key(score - slack);
    int c[3] = {0, 0, 0}, all[3];
    for (int i = tid; i < last; i += kSelectThreads) {
      const uint32_t key = keys[i];
      c[0] += key == 0xFFFFFFFFu ? 1 : 0;
      c[1] += key > above0 ? 1 : 0;
      c[2] += key >= below0 ? 1 : 0;
    }
    count3(c[0], c[1], c[2], all);
    // a NaN key may hide a score of any size (zero times an infinite bound of the other side)
    const bool known = isfinite(score) && isfinite(slack) && all[0] == 0;
    const uint32_t above = known ? above0 : 0xFFFFFFFFu, below = known ? below0 : 0u;
    settled = known && all[2] == want;  // everything in doubt is in
    for (int i = tid; i < last; i += kSelectThreads) {
      const uint32_t key = keys[i];
      // refused pages (key 0) stay below everything, NaN keys are summed again
      const bool doubt = key != 0u && ((key >= below && key <= above) || key == 0xFFFFFFFFu);
      if (doubt && !settled) doubtful[atomicAdd(&s_doubtful, 1)] = i;
      keys[i] = doubt ? (settled ? 0xFFFFFFFFu : 0u) : (key > above ? 0xFFFFFFFFu : 0u);
    }
    __syncthreads();
    const int tasks = s_doubtful * group;  // (page, head), a half-warp each; in any order
    for (int task0 = 0; task0 < tasks; task0 += kWarps * 2) {
      const int task = min(task0 + warp * 2 + lane / kLanes, tasks - 1), which = task / group;
      const int i = doubtful[which], h = task - which * group;
      const uint32_t key = exact_key<T>(D, q0 + int64_t(h) * p.q_sh, bounds + int64_t(ids[i]) * 2 * D, lane % kLanes);
      if (lane % kLanes == 0) atomicMax(&keys[i], key);
    }
    __syncthreads();
    // a few in doubt: a warp ranks them (a search over all keys takes 9,000 cycles). Those for which
    // there is room are in
    if (known && !settled && s_doubtful <= 32) {
      if (warp == 0) {
        const int left = s_doubtful, i = lane < left ? doubtful[lane] : last;
        const uint32_t key = lane < left ? keys[i] : 0u;
        int better = 0;
        for (int o = 0; o < left; ++o) {
          const uint32_t other = __shfl_sync(0xffffffffu, key, o);
          const int other_i = __shfl_sync(0xffffffffu, i, o);
          better += other > key || (other == key && other_i < i) ? 1 : 0;
        }
        __syncwarp();
        if (lane < left) keys[i] = better < want - all[1] ? 0xFFFFFFFFu : 0u;
      }
      settled = true;
      __syncthreads();
    }
  }
  uint32_t threshold = 0xFFFFFFFFu;  // keys above it are in, and the first `need` of those equal to it
  int need = 0;
  if (settled) {
    threshold = 0xFFFFFFFEu;  // the keys that are in are all ones by now, the others 0
  } else if (want > 0) {
    threshold = threshold_of();
    if (exactly) {
      --threshold;  // exactly `want` keys are above threshold - 1 (threshold >= 1)
    } else {
      int c = 0, all[3];
      for (int i = tid; i < last; i += kSelectThreads) c += keys[i] > threshold ? 1 : 0;
      count3(c, 0, 0, all);
      need = want - all[0];
    }
  }

  // ---- emit in ascending order: warp w takes pages [w * share, (w + 1) * share)
  const int share = (last + kWarps * 32 - 1) / (kWarps * 32) * 32;
  const int first = min(warp * share, last), end = min(first + share, last);
  int equal = 0;
  for (int i = first + lane; i < first + share; i += 32)
    equal += __popc(__ballot_sync(0xffffffffu, i < end && keys[i] == threshold));
  if (lane == 0) warp_count[warp] = equal;
  __syncthreads();
  int equal_before = 0;  // equal keys before this warp's
  for (int w = 0; w < warp; ++w) equal_before += warp_count[w];
  __syncthreads();
  int mine = 0, r = equal_before;
  for (int i = first + lane; i < first + share; i += 32) {
    const bool eq = i < end && keys[i] == threshold, gt = i < end && keys[i] > threshold;
    const uint32_t eqs = __ballot_sync(0xffffffffu, eq);
    const bool in = gt || (eq && r + __popc(eqs & ((1u << lane) - 1)) < need);
    mine += __popc(__ballot_sync(0xffffffffu, in));
    r += __popc(eqs);
  }
  if (lane == 0) warp_count[warp] = mine;
  __syncthreads();
  int at = 0;
  for (int w = 0; w < warp; ++w) at += warp_count[w];
  r = equal_before;
  for (int i = first + lane; i < first + share; i += 32) {
    const bool eq = i < end && keys[i] == threshold, gt = i < end && keys[i] > threshold;
    const uint32_t eqs = __ballot_sync(0xffffffffu, eq);
    const bool in = gt || (eq && r + __popc(eqs & ((1u << lane) - 1)) < need);
    const uint32_t ins = __ballot_sync(0xffffffffu, in);
    if (in) {
      const int slot = at + __popc(ins & ((1u << lane) - 1));
      p.selected[out_row + slot] = i;
      p.pages[out_row + slot] = ids[i];
    }
    at += __popc(ins);
    r += __popc(eqs);
  }
  if (tid == 0) {
    p.selected[out_row + p.take - 1] = last;
    p.pages[out_row + p.take - 1] = table[last];
  }
}

}  // namespace

cudaError_t run_page_bounds(const BoundsParams& p, int dtype, cudaStream_t stream) {
  if (p.count == 0 || p.layers == 0) return cudaSuccess;
  const int row_bytes = p.head_dim * (dtype == HYT_DTYPE_F32 ? 4 : 2), rows = 1 << p.page_shift;
  const int block = row_bytes >= 512 ? kBoundsBlock * 3 / 4 : kBoundsBlock;  // so that an SM holds two CTAs
  const int stage_rows = rows * int64_t(row_bytes) <= block ? rows : block / row_bytes;
  const int smem = kBoundsStages * stage_rows * row_bytes + 4 * (kBoundsThreads / 32) * row_bytes;
  // as many CTAs as fit the SMs at once, an equal share of the items each
  const int64_t items = int64_t(p.num_kv_heads) * p.count * p.layers;
  const int64_t slots = 148 * std::min<int64_t>(8, (220 << 10) / (smem + 1024));
  const unsigned grid = unsigned(std::min(items, slots));
  auto launch = [&](auto kernel) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    kernel<<<grid, kBoundsThreads, smem, stream>>>(p, items, stage_rows);
    return cudaGetLastError();
  };
  switch (dtype) {
    case HYT_DTYPE_BF16: return launch(page_bounds_kernel<__nv_bfloat16>);
    case HYT_DTYPE_F16: return launch(page_bounds_kernel<__half>);
    default: return launch(page_bounds_kernel<float>);
  }
}

cudaError_t run_select_pages(const SelectParams& params, int dtype, cudaStream_t stream) {
  SelectParams p = params;
  const int units = p.batch * p.num_kv_heads;
  const int ranked = p.table_width < kSelectMaxPages ? p.table_width : kSelectMaxPages;
  p.ranked = ranked;
  // CTAs per unit: enough to give every SM two, none with less than 32 pages
  int ranks = 1;
  while (ranks < 8 && units * ranks < 2 * 148 && ranked >= 64 * ranks) ranks *= 2;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = unsigned(ranks);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(unsigned(units * ranks));
  config.blockDim = dim3(kSelectThreads);
  size_t ring = 0;  // 3 (head_dim above 128: 2) turns of two bounds pieces per step and thread
  if (dtype != HYT_DTYPE_F32) ring = size_t(kSelectThreads) * 2 * 16 * (p.head_dim <= 128 ? 3 * 4 : 2 * 8);
  config.dynamicSmemBytes = (size_t(ranked) * 12 + 15) / 16 * 16 + ring;
  config.stream = stream;
  config.attrs = &attr;
  config.numAttrs = 1;
  auto launch = [&](auto kernel) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(config.dynamicSmemBytes));
    return e != cudaSuccess ? e : cudaLaunchKernelEx(&config, kernel, p);
  };
  switch (dtype) {
    case HYT_DTYPE_BF16:
      return p.head_dim <= 128 ? launch(select_pages_kernel<__nv_bfloat16, 4>) : launch(select_pages_kernel<__nv_bfloat16, 8>);
    case HYT_DTYPE_F16:
      return p.head_dim <= 128 ? launch(select_pages_kernel<__half, 4>) : launch(select_pages_kernel<__half, 8>);
    default: return launch(select_pages_kernel<float, 1>);
  }
}

}  // namespace hyt
