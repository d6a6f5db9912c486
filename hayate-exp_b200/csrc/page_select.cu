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
// to each other, so the sums run in 64 bits (a product of two 16-bit values is exact there)
// and are rounded once to fp32: the choice does not depend on the order of summation.
// One CTA per (request, KV head): 8 lanes per page, 2 rows of bounds per page read once; the
// take - 1 best by a radix selection on order-preserving 32-bit keys in shared memory.
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

constexpr int kHeadsAtOnce = 4;

template <typename T>
__global__ void __launch_bounds__(kSelectThreads) select_pages_kernel(const SelectParams p) {
  constexpr int kPer = 16 / int(sizeof(T));
  constexpr int kWarps = kSelectThreads / 32;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  const int g = blockIdx.x, b = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int D = p.head_dim, group = p.num_q_heads / p.num_kv_heads;
  double* qs = reinterpret_cast<double*>(smem_raw);               // [group][D]
  uint32_t* keys = reinterpret_cast<uint32_t*>(qs + group * D);   // [last]
  __shared__ int hist[256];
  __shared__ int warp_count[kWarps];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;

  const int64_t out_row = (int64_t(b) * p.num_kv_heads + g) * p.take;
  const int32_t* table = p.page_table + int64_t(b) * p.page_table_stride;
  const int len = p.cache_lens[b];
  const int last = len >= 0 ? len >> p.page_shift : p.table_width;  // the page being written
  if (last >= p.table_width || last > kSelectMaxPages) {
    if (tid == 0 && g == 0) flag_error(p.error_word, HYT_DEVERR_TABLE_RANGE);
    for (int i = tid; i < p.take; i += kSelectThreads) p.selected[out_row + i] = p.pages[out_row + i] = -1;
    if (g == 0 && tid == 0) p.lens[b] = 0;
    return;
  }
  const int count = min(last + 1, p.take);
  if (g == 0 && tid == 0) p.lens[b] = ((count - 1) << p.page_shift) + (len & ((1 << p.page_shift) - 1));
  if (last < p.take) {  // every page is read
    for (int i = tid; i < p.take; i += kSelectThreads) {
      p.selected[out_row + i] = i < count ? i : -1;
      p.pages[out_row + i] = i < count ? table[i] : -1;
    }
    return;
  }

  const T* q = static_cast<const T*>(p.q) + int64_t(b) * p.q_sb + int64_t(g) * group * p.q_sh;
  for (int i = tid; i < group * D; i += kSelectThreads)
    qs[i] = double(Elem<T>::to_float(q[int64_t(i / D) * p.q_sh + i % D]));
  __syncthreads();

  // ---- scores of the full pages 0 .. last - 1, 8 lanes per page
  const T* bounds = static_cast<const T*>(p.k_bounds) +
                    (int64_t(p.layer) * p.num_kv_heads + g) * p.num_pages * 2 * D;
  const int sub = lane >> 3, l8 = lane & 7, chunks = D / kPer;
  for (int i0 = warp * 4; i0 < last; i0 += kWarps * 4) {
    const int i = i0 + sub;
    int32_t page = -1;
    if (i < last) {
      page = table[i];
      if (page < 0 || page >= p.num_pages) {
        if (l8 == 0) flag_error(p.error_word, HYT_DEVERR_PAGE_RANGE);
        page = -1;
      }
    }
    const T* lo = bounds + int64_t(max(page, 0)) * 2 * D;
    float best = -INFINITY;
    bool nan = false;
    for (int h0 = 0; h0 < group; h0 += kHeadsAtOnce) {
      double acc[kHeadsAtOnce] = {0., 0., 0., 0.};
      for (int c = l8; c < chunks; c += 8) {
        float fl[kPer], fh[kPer];
        unpack16<T>(__ldg(reinterpret_cast<const uint4*>(lo) + c), fl);
        unpack16<T>(__ldg(reinterpret_cast<const uint4*>(lo + D) + c), fh);
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const double dl = fl[e], dh = fh[e];
#pragma unroll
          for (int h = 0; h < kHeadsAtOnce; ++h) {
            if (h0 + h >= group) break;
            const double qv = qs[(h0 + h) * D + c * kPer + e];
            acc[h] = fma(qv, qv >= 0. ? dh : dl, acc[h]);
          }
        }
      }
#pragma unroll
      for (int h = 0; h < kHeadsAtOnce; ++h) {
#pragma unroll
        for (int off = 4; off > 0; off >>= 1) acc[h] += __shfl_xor_sync(0xffffffffu, acc[h], off);
        if (h0 + h < group) {
          const float x = float(acc[h]);
          nan |= isnan(x);
          best = fmaxf(best, x);
        }
      }
    }
    if (i < last && l8 == 0) keys[i] = page < 0 ? 0u : (nan ? 0xFFFFFFFFu : score_key(best));
  }
  __syncthreads();

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
  int rank = 0;  // equal keys before this warp's
  for (int w = 0; w < warp; ++w) rank += warp_count[w];
  __syncthreads();
  const bool any = p.take > 1;
  int mine = 0, r = rank;
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
  r = rank;
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
  const int group = p.num_q_heads / p.num_kv_heads;
  const int ranked = p.table_width < kSelectMaxPages ? p.table_width : kSelectMaxPages;
  const int smem = group * p.head_dim * 8 + ranked * 4;
  const dim3 grid(unsigned(p.num_kv_heads), unsigned(p.batch));
  auto launch = [&](auto kernel) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    kernel<<<grid, kSelectThreads, smem, stream>>>(p);
    return cudaGetLastError();
  };
  switch (dtype) {
    case HYT_DTYPE_BF16: return launch(select_pages_kernel<__nv_bfloat16>);
    case HYT_DTYPE_F16: return launch(select_pages_kernel<__half>);
    default: return launch(select_pages_kernel<float>);
  }
}

}  // namespace hyt
