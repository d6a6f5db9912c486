// Pages and rows moved inside the KV pools, every layer in one launch.
//
// copy_pages: page src[m] -> page dst[m] of every (layer, KV head) plane of K and V: forks
// that get their own copy of the page being written, and copy-on-write. A page of a plane is
// one contiguous block (32 KB at 128 tokens x 128 bf16), so the copy is a plain stream:
// 16-byte loads, kUnroll in flight per thread, then the stores. Bound: HBM, one read and one
// write of every byte: 64 pages x 36 layers x 8 heads (2.42 GB) take 384 us, 6.3 TB/s.
//
// compact_rows: request b's row base[b] + src[i] -> base[b] + i, src strictly increasing (so
// src[i] >= i): the accepted path of a drafted tree moves up behind the context, in place.
// A CTA serves one request: it looks its rows' pool offsets up once, kThreads rows at a time,
// and every thread owns one 16-byte column of one plane and takes the rows in order, kRowsAhead
// loads before their stores: row i + kRowsAhead is read after rows < i + kRowsAhead were written,
// and src[i + kRowsAhead] >= i + kRowsAhead, so nothing is read after it was overwritten, and no
// two threads touch the same bytes. Bound: HBM, 256-byte pieces (a row of one head), one read
// and one write of each: 64 paths of 6 to 12 rows x 36 layers x 8 heads (171 MB) take 32 us, 5.3
// TB/s (offsets looked up by every thread for itself: 39 us).
#include "chunk_schedule.cuh"

namespace hyt {

namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 8;

template <int kBytes>
struct Vec;
template <>
struct Vec<16> { using type = uint4; };
template <>
struct Vec<8> { using type = uint2; };
template <>
struct Vec<4> { using type = uint32_t; };
template <>
struct Vec<2> { using type = uint16_t; };

template <int kVec>
__global__ void __launch_bounds__(kThreads) copy_pages_kernel(const MoveParams p, int planes_per_cta) {
  using V = typename Vec<kVec>::type;
  const int m = blockIdx.y;
  const int32_t src = p.src[m], dst = p.dst[m];
  // refuse ids outside the pool, and entries whose target another entry reads (the result
  // would depend on the order); of two entries with one target the last one counts
  const bool outside = src < 0 || src >= p.num_pages || dst < 0 || dst >= p.num_pages;
  int read = 0, skip = src == dst;
  for (int i = threadIdx.x; i < p.count; i += kThreads) {
    if (i != m && p.src[i] == dst && p.dst[i] != dst) read = 1;
    if (i > m && p.dst[i] == dst) skip = 1;
  }
  read = __syncthreads_or(read);
  skip = __syncthreads_or(skip);
  if (outside || read) {
    if (threadIdx.x == 0) flag_error(p.error_word, outside ? HYT_DEVERR_PAGE_RANGE : HYT_DEVERR_MOVE_ORDER);
    return;
  }
  if (skip) return;
  const int64_t page_bytes = p.row_bytes << p.page_shift, plane_bytes = p.row_bytes * p.capacity;
  const int n = int(page_bytes / kVec);
  const int first = int(blockIdx.x) * planes_per_cta, last = min(first + planes_per_cta, 2 * p.planes);
  for (int plane = first; plane < last; ++plane) {
    uint8_t* pool = plane < p.planes ? p.k_pool + plane * plane_bytes : p.v_pool + (plane - p.planes) * plane_bytes;
    const V* from = reinterpret_cast<const V*>(pool + src * page_bytes);
    V* to = reinterpret_cast<V*>(pool + dst * page_bytes);
    for (int i0 = threadIdx.x; i0 < n; i0 += kThreads * kUnroll) {
      V v[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (i0 + u * kThreads < n) v[u] = from[i0 + u * kThreads];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (i0 + u * kThreads < n) to[i0 + u * kThreads] = v[u];
    }
  }
}

template <int kVec>
__global__ void __launch_bounds__(kThreads) compact_rows_kernel(const MoveParams p) {
  using V = typename Vec<kVec>::type;
  // 36 layers, us with 4 / 12 / 16 rows ahead: 64 paths of 2 to 4 rows 9 / 13 / 18, of 6 to 12 31 / 32 / 37,
  // 16 of 32 29 / 30 / 29; 300 rows of 4 requests 89 / 67 / 63, 1,000 of one 229 / 145 / 136
  constexpr int kRowsAhead = 12;
  __shared__ int64_t from_s[kThreads], to_s[kThreads];  // byte offsets in a plane, -1: nothing to do
  const int b = blockIdx.y;
  const int begin = p.start[b], end = p.start[b + 1];
  if (begin < 0 || end < begin || end > p.count) {
    if (blockIdx.x == 0 && threadIdx.x == 0) flag_error(p.error_word, HYT_DEVERR_PACKED_RANGE);
    return;
  }
  const int chunks = int(p.row_bytes / kVec);
  const int64_t column = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t plane = column / chunks;
  const bool mine = plane < 2 * int64_t(p.planes);
  const int64_t plane_bytes = p.row_bytes * p.capacity;
  uint8_t* pool = !mine ? nullptr
                        : (plane < p.planes ? p.k_pool + plane * plane_bytes : p.v_pool + (plane - p.planes) * plane_bytes) +
                              (column - plane * chunks) * kVec;
  const int64_t base = p.base[b];
  const int32_t* table = p.page_table + int64_t(b) * p.page_table_stride;
  int why = 0;
  auto row = [&](int64_t pos) -> int64_t {  // byte offset of a position's row in a plane, or -1
    const int64_t lp = pos >> p.page_shift;
    if (pos < 0 || lp >= p.table_width) {
      why |= HYT_DEVERR_TABLE_RANGE;
      return -1;
    }
    const int32_t page = table[lp];
    if (page < 0 || page >= p.num_pages) {
      why |= HYT_DEVERR_PAGE_RANGE;
      return -1;
    }
    return ((int64_t(page) << p.page_shift) + (pos & ((1 << p.page_shift) - 1))) * p.row_bytes;
  };
  for (int group = begin; group < end; group += kThreads) {
    const int here = min(end - group, kThreads);
    __syncthreads();  // the offsets of the group before have been used
    if (int(threadIdx.x) < here) {
      const int i = group + int(threadIdx.x), at = i - begin;
      const int s = p.src[i], prev = i > begin ? p.src[i - 1] : -1;
      int64_t from = -1, to = -1;
      if (s < at || s <= prev) why |= HYT_DEVERR_MOVE_ORDER;
      else if (s != at) from = row(base + s), to = row(base + at);
      from_s[threadIdx.x] = from < 0 || to < 0 ? -1 : from;
      to_s[threadIdx.x] = to;
    }
    __syncthreads();
    if (!mine) continue;
    for (int i0 = 0; i0 < here; i0 += kRowsAhead) {
      V v[kRowsAhead];
#pragma unroll
      for (int u = 0; u < kRowsAhead; ++u)
        if (i0 + u < here && from_s[i0 + u] >= 0) v[u] = *reinterpret_cast<const V*>(pool + from_s[i0 + u]);
#pragma unroll
      for (int u = 0; u < kRowsAhead; ++u)
        if (i0 + u < here && from_s[i0 + u] >= 0) *reinterpret_cast<V*>(pool + to_s[i0 + u]) = v[u];
    }
  }
  if (why && blockIdx.x == 0) flag_error(p.error_word, why);
}

// Widest vector that rows, planes and both pools are aligned to.
int move_vec(const MoveParams& p) {
  for (int v : {16, 8, 4})
    if (p.row_bytes % v == 0 && reinterpret_cast<uintptr_t>(p.k_pool) % v == 0 &&
        reinterpret_cast<uintptr_t>(p.v_pool) % v == 0)
      return v;
  return 2;
}

}  // namespace

cudaError_t run_copy_pages(const MoveParams& p, cudaStream_t stream) {
  if (p.count == 0) return cudaSuccess;
  const int planes = 2 * p.planes;
  // enough CTAs to fill the GPU several times over, then more planes per CTA: each CTA reads
  // the entry list once
  const int64_t blocks = int64_t(planes) * p.count;
  const int per = int(blocks / (148 * 32) < 1 ? 1 : (blocks / (148 * 32) > 16 ? 16 : blocks / (148 * 32)));
  const dim3 grid(unsigned((planes + per - 1) / per), unsigned(p.count));
  switch (move_vec(p)) {
    case 16: copy_pages_kernel<16><<<grid, kThreads, 0, stream>>>(p, per); break;
    case 8: copy_pages_kernel<8><<<grid, kThreads, 0, stream>>>(p, per); break;
    case 4: copy_pages_kernel<4><<<grid, kThreads, 0, stream>>>(p, per); break;
    default: copy_pages_kernel<2><<<grid, kThreads, 0, stream>>>(p, per); break;
  }
  return cudaGetLastError();
}

cudaError_t run_compact_rows(const MoveParams& p, cudaStream_t stream) {
  const int vec = move_vec(p);
  const int64_t columns = 2 * int64_t(p.planes) * (p.row_bytes / vec);
  const dim3 grid(unsigned((columns + kThreads - 1) / kThreads), unsigned(p.batch));
  switch (vec) {
    case 16: compact_rows_kernel<16><<<grid, kThreads, 0, stream>>>(p); break;
    case 8: compact_rows_kernel<8><<<grid, kThreads, 0, stream>>>(p); break;
    case 4: compact_rows_kernel<4><<<grid, kThreads, 0, stream>>>(p); break;
    default: compact_rows_kernel<2><<<grid, kThreads, 0, stream>>>(p); break;
  }
  return cudaGetLastError();
}

}  // namespace hyt
