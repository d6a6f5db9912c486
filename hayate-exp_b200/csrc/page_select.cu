// Page bounds, and the choice of pages a one-token decode reads.
//
// page_bounds: elementwise minimum and maximum of a full page's keys, per layer and KV head.
// One pass over the page: a thread keeps one 16-byte column of every n-th row, the row groups
// meet in shared memory. NaN keys give NaN bounds. Bound: HBM reads of the keys.
//
// select_pages: score(page) = max over the KV group's query heads of
//   sum_d q_d * (q_d >= 0 ? max_d : min_d),
// the most a key of the page can score; the take - 1 best full pages (ties: the lowest page)
// and the page being written, in ascending order. Which page is read hangs on scores next
// to each other, so a score must not depend on the order of summation: products of 16-bit
// values are exact in fp32 (fp32 ones keep their rounding error by an FMA), the sums carry
// their rounding errors along (Knuth's two-sum, on packed pairs), lanes meet in 64 bits, and
// the result is rounded once. That costs 5.5 instructions a term; converting to 64 bits term
// by term took 80 us on 64 requests x 256 pages x 8 KV heads (4 heads a group), this 20.
// A cluster of 1 to 8 CTAs per (request, KV head) shares the pages out, 16 lanes per page and
// the bounds read once; the keys (order-preserving 32-bit scores) meet in the first CTA's
// shared memory, which finds the (take - 1)-th largest 8 bits at a time.
#include <cooperative_groups.h>

#include <type_traits>

#include "chunk_schedule.cuh"

namespace hyt {

namespace {

constexpr int kBoundsThreads = 256;
constexpr int kSelectThreads = 256;

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

// Grid: (KV head, page entry, layer).
template <typename T>
__global__ void __launch_bounds__(kBoundsThreads) page_bounds_kernel(const BoundsParams p) {
  constexpr int kPer = 16 / int(sizeof(T));
  __shared__ float lo_s[kBoundsThreads * kPer], hi_s[kBoundsThreads * kPer];
  const int32_t page = p.pages[blockIdx.y];
  if (page == -1) return;
  if (page < 0 || page >= p.num_pages) {
    if (threadIdx.x == 0) flag_error(p.error_word, HYT_DEVERR_PAGE_RANGE);
    return;
  }
  const int D = p.head_dim, chunks = D / kPer;       // 16-byte columns of a row (<= 64)
  const int groups = kBoundsThreads / chunks;        // rows read side by side
  const int c = threadIdx.x % chunks, rg = threadIdx.x / chunks;
  const int64_t plane = int64_t(p.first_layer + blockIdx.z) * p.num_kv_heads + blockIdx.x;
  const int rows = 1 << p.page_shift;
  const T* keys = static_cast<const T*>(p.k_pool) + (plane * p.capacity + (int64_t(page) << p.page_shift)) * D + c * kPer;
  float lo[kPer], hi[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) lo[e] = INFINITY, hi[e] = -INFINITY;
  if (rg < groups) {
    constexpr int kAhead = 8;
    for (int r0 = rg; r0 < rows; r0 += groups * kAhead) {
      uint4 v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (r0 + u * groups < rows) v[u] = __ldg(reinterpret_cast<const uint4*>(keys + int64_t(r0 + u * groups) * D));
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (r0 + u * groups >= rows) break;
        float f[kPer];
        unpack16<T>(v[u], f);
#pragma unroll
        for (int e = 0; e < kPer; ++e) lo[e] = min_nan(lo[e], f[e]), hi[e] = max_nan(hi[e], f[e]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) {  // [e][thread]: no bank conflicts
    lo_s[e * kBoundsThreads + threadIdx.x] = lo[e];
    hi_s[e * kBoundsThreads + threadIdx.x] = hi[e];
  }
  __syncthreads();
  T* out = static_cast<T*>(p.k_bounds) + (plane * p.num_pages + page) * 2 * D;
  for (int d = threadIdx.x; d < 2 * D; d += kBoundsThreads) {
    const bool is_hi = d >= D;
    const int dd = is_hi ? d - D : d, cc = dd / kPer, e = dd - cc * kPer;
    const float* from = (is_hi ? hi_s : lo_s) + e * kBoundsThreads;
    float x = from[cc];
    for (int g = 1; g < min(groups, rows); ++g)
      x = is_hi ? max_nan(x, from[g * chunks + cc]) : min_nan(x, from[g * chunks + cc]);
    out[d] = Elem<T>::from_float(x);  // exact: x is one of the keys' values
  }
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

// kHeads: query heads scored per pass over a page's bounds.
template <typename T, int kHeads>
__global__ void __launch_bounds__(kSelectThreads) select_pages_kernel(const SelectParams p) {
  constexpr int kPer = 16 / int(sizeof(T));
  constexpr int kWarps = kSelectThreads / 32;
  constexpr int kLanes = 16;  // per page
  extern __shared__ __align__(16) uint32_t keys[];  // [last], the first CTA's are used
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int unit = int(blockIdx.x) / ranks;
  const int b = unit / p.num_kv_heads, g = unit - b * p.num_kv_heads;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int D = p.head_dim, group = p.num_q_heads / p.num_kv_heads;
  __shared__ int hist[256];
  __shared__ int warp_count[kWarps];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  launch_dependents();  // the attention kernel may start up; it waits for this grid's results

  const int64_t out_row = (int64_t(b) * p.num_kv_heads + g) * p.take;
  const int32_t* table = p.page_table + int64_t(b) * p.page_table_stride;
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

  // ---- scores of the full pages 0 .. last - 1: this CTA's share, 16 lanes per page
  {
    if (ranks > 1) cluster.sync();  // the first CTA has started: its shared memory may be written
    uint32_t* to = cluster.map_shared_rank(keys, 0);
    const T* bounds = static_cast<const T*>(p.k_bounds) +
                      (int64_t(p.layer) * p.num_kv_heads + g) * p.num_pages * 2 * D;
    const T* q0 = static_cast<const T*>(p.q) + int64_t(b) * p.q_sb + int64_t(g) * group * p.q_sh;
    const int sub = lane / kLanes, l16 = lane % kLanes, chunks = D / kPer;
    constexpr int kPages = kWarps * (32 / kLanes);  // pages a CTA scores at a time
    for (int i0 = rank * kPages; i0 < last; i0 += ranks * kPages) {
      const int i = i0 + warp * (32 / kLanes) + sub;
      int32_t page = -1;
      if (i < last) {
        page = table[i];
        if (page < 0 || page >= p.num_pages) {
          if (l16 == 0) flag_error(p.error_word, HYT_DEVERR_PAGE_RANGE);
          page = -1;
        }
      }
      const T* lo = bounds + int64_t(max(page, 0)) * 2 * D;
      float best = -INFINITY;
      bool nan = false;
      for (int h0 = 0; h0 < group; h0 += kHeads) {
        PairSum acc[kHeads];
        for (int c = l16; c < chunks; c += kLanes) {
          const uint4 lraw = __ldg(reinterpret_cast<const uint4*>(lo) + c);
          const uint4 hraw = __ldg(reinterpret_cast<const uint4*>(lo + D) + c);
          const uint32_t lw[4] = {lraw.x, lraw.y, lraw.z, lraw.w}, hw[4] = {hraw.x, hraw.y, hraw.z, hraw.w};
#pragma unroll
          for (int h = 0; h < kHeads; ++h) {
            if (h0 + h >= group) break;
            const T* qh = q0 + int64_t(h0 + h) * p.q_sh + c * kPer;
            if constexpr (sizeof(T) == 2) {
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                const float qa = Elem<T>::to_float(qh[2 * w]), qb = Elem<T>::to_float(qh[2 * w + 1]);
                const uint32_t m = (qa >= 0.f ? 0x0000FFFFu : 0u) | (qb >= 0.f ? 0xFFFF0000u : 0u);
                const uint32_t x = (hw[w] & m) | (lw[w] & ~m);
                const T* xe = reinterpret_cast<const T*>(&x);
                acc[h].add(f2_mul(f2_pack(qa, qb), f2_pack(Elem<T>::to_float(xe[0]), Elem<T>::to_float(xe[1]))));
              }
            } else {
#pragma unroll
              for (int w = 0; w < 4; w += 2) {
                const float qa = qh[w], qb = qh[w + 1];
                const uint64_t q2 = f2_pack(qa, qb);
                const uint64_t x2 = f2_pack(__uint_as_float(qa >= 0.f ? hw[w] : lw[w]),
                                            __uint_as_float(qb >= 0.f ? hw[w + 1] : lw[w + 1]));
                const uint64_t prod = f2_mul(q2, x2);
                acc[h].add(prod);
                acc[h].e = f2_add(acc[h].e, f2_fma(q2, x2, f2_mul(prod, f2_pack(-1.f, -1.f))));
              }
            }
          }
        }
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
          double total = acc[h].total();
#pragma unroll
          for (int off = kLanes / 2; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
          if (h0 + h < group) {
            const float x = float(total);
            nan |= isnan(x);
            best = fmaxf(best, x);
          }
        }
      }
      if (i < last && l16 == 0) to[i] = page < 0 ? 0u : (nan ? 0xFFFFFFFFu : score_key(best));
    }
  }
  cluster.sync();
  if (rank != 0) return;

  // ---- the (take - 1)-th largest key, 8 bits at a time
  int need = p.take - 1;  // of the keys that match the prefix so far, this many are wanted
  uint32_t prefix = 0, mask = 0;
  for (int shift = 24; shift >= 0 && need > 0; shift -= 8) {
    for (int i = tid; i < 256; i += kSelectThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < last; i += kSelectThreads)
      if ((keys[i] & mask) == prefix) atomicAdd(&hist[(keys[i] >> shift) & 255], 1);
    __syncthreads();
    if (warp == 0) {  // lane l: bins 255 - 8 l .. 248 - 8 l, from the top
      int bin[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        bin[j] = hist[255 - lane * 8 - j];
        sum += bin[j];
      }
      int scan = sum;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, scan, off);
        if (lane >= off) scan += v;
      }
      int above = scan - sum;
      if (above < need && need <= scan) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (above < need && need <= above + bin[j]) {
            s_prefix = prefix | (uint32_t(255 - lane * 8 - j) << shift);
            s_need = need - above;
          }
          above += bin[j];
        }
      }
    }
    __syncthreads();
    prefix = s_prefix;
    need = s_need;
    mask |= 255u << shift;
  }
  // pages with key > prefix are in; of those equal to it the first `need`

  // ---- emit in ascending order: warp w takes pages [w * share, (w + 1) * share)
  const int share = (last + kWarps * 32 - 1) / (kWarps * 32) * 32;
  const int first = min(warp * share, last), end = min(first + share, last);
  int equal = 0;
  for (int i = first + lane; i < first + share; i += 32)
    equal += __popc(__ballot_sync(0xffffffffu, i < end && keys[i] == prefix));
  if (lane == 0) warp_count[warp] = equal;
  __syncthreads();
  int equal_before = 0;  // equal keys before this warp's
  for (int w = 0; w < warp; ++w) equal_before += warp_count[w];
  __syncthreads();
  const bool any = p.take > 1;
  int mine = 0, r = equal_before;
  for (int i = first + lane; i < first + share; i += 32) {
    const bool eq = any && i < end && keys[i] == prefix, gt = any && i < end && keys[i] > prefix;
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
    const bool eq = any && i < end && keys[i] == prefix, gt = any && i < end && keys[i] > prefix;
    const uint32_t eqs = __ballot_sync(0xffffffffu, eq);
    const bool in = gt || (eq && r + __popc(eqs & ((1u << lane) - 1)) < need);
    const uint32_t ins = __ballot_sync(0xffffffffu, in);
    if (in) {
      const int slot = at + __popc(ins & ((1u << lane) - 1));
      p.selected[out_row + slot] = i;
      p.pages[out_row + slot] = table[i];
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
  const dim3 grid(unsigned(p.num_kv_heads), unsigned(p.count), unsigned(p.layers));
  switch (dtype) {
    case HYT_DTYPE_BF16: page_bounds_kernel<__nv_bfloat16><<<grid, kBoundsThreads, 0, stream>>>(p); break;
    case HYT_DTYPE_F16: page_bounds_kernel<__half><<<grid, kBoundsThreads, 0, stream>>>(p); break;
    default: page_bounds_kernel<float><<<grid, kBoundsThreads, 0, stream>>>(p); break;
  }
  return cudaGetLastError();
}

cudaError_t run_select_pages(const SelectParams& p, int dtype, cudaStream_t stream) {
  const int group = p.num_q_heads / p.num_kv_heads, units = p.batch * p.num_kv_heads;
  const int ranked = p.table_width < kSelectMaxPages ? p.table_width : kSelectMaxPages;
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
  config.dynamicSmemBytes = size_t(ranked) * 4;
  config.stream = stream;
  config.attrs = &attr;
  config.numAttrs = 1;
  auto launch = [&](auto kernel) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(config.dynamicSmemBytes));
    return e != cudaSuccess ? e : cudaLaunchKernelEx(&config, kernel, p);
  };
  auto heads = [&](auto type) {
    using T = decltype(type);
    if (group == 1) return launch(select_pages_kernel<T, 1>);
    if (group == 2) return launch(select_pages_kernel<T, 2>);
    return launch(select_pages_kernel<T, 4>);
  };
  switch (dtype) {
    case HYT_DTYPE_BF16: return heads(__nv_bfloat16{});
    case HYT_DTYPE_F16: return heads(__half{});
    default: return heads(float{});
  }
}

}  // namespace hyt
