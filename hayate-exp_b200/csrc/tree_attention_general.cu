// Chunk attention on CUDA cores (fp32 pools, head sizes the tensor-core kernel does not
// take), and the merge of split units that both kernels share.
//
//   out[row] = sum_j softmax_j(scale * q[row] . k_j) v_j
//
// over the cached keys and the step's own nodes that the row's mask shows
// (chunk_visible64); a row that sees nothing is zeros. Serves trees of drafted tokens and
// one-token decode over chosen pages (a page-table row per KV head).
//
// Up to 8 rows per unit (chunk_attention_rows_kernel): the keys' bytes weigh more than the
// products, so K and V go straight from global memory to registers (see there).
//
// More rows: a CTA holds a block of 16 or 64 query rows (all heads of a KV group next to each other, so
// a key is read once for the whole group) in shared memory as fp32 and streams the unit's keys
// in 64-key tiles: S = Q K^T from registers (thread (ty, tx): rows ty * kRows / 16 .., keys
// tx + 16 j), online softmax in base 2 with 16-lane shuffles, P through shared memory (over
// K's tile, which S has finished with), O += P V in registers (dims tx * 4 + 64 c). All
// arithmetic is fp32; 16-bit inputs are widened once, on the way into shared memory.
//
// Masked values never reach a sum: a masked score is -inf by selection, V rows past the
// request's end are stored as zeros if they are not finite, and so are non-finite V values
// of drafted nodes, which are added at the end to the rows that see them (0 * inf would
// be NaN in every row).
//
// Bound at 64 rows: fp32 FMA and the shared-memory reads that feed it (25 of 75 TFLOP/s).
#include <type_traits>

#include "chunk_schedule.cuh"

namespace hyt {

namespace {

constexpr int kThreads = 256;
constexpr int kKeys = 64;

template <typename T>
__device__ __forceinline__ void widen16(const uint4& v, float (&f)[16 / sizeof(T)]) {
  if constexpr (sizeof(T) == 4) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  } else {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T* e = reinterpret_cast<const T*>(&w[i]);
      f[2 * i] = Elem<T>::to_float(e[0]);
      f[2 * i + 1] = Elem<T>::to_float(e[1]);
    }
  }
}

// kRows: query rows per unit; kChunks: 64-dim column chunks of O (ceil(head_dim / 64)).
template <typename T, int kRows, int kChunks>
__global__ void __launch_bounds__(kThreads) chunk_attention_general_kernel(const ChunkParams P) {
  constexpr int kR = kRows / 16;       // rows per thread
  constexpr int kD = kChunks * 64;     // padded head size
  constexpr int kLd = kD + 4;          // shared row length: consecutive rows 4 banks apart
  constexpr int kLdP = kKeys + 4;
  constexpr int kPer = 16 / int(sizeof(T));
  const AttentionParams& p = P.a;
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const int D = p.head_dim;

  extern __shared__ __align__(16) float smem[];
  float* qs = smem;                // [kRows][kLd]
  float* ks = qs + kRows * kLd;    // [kKeys][kLd], then P [kRows][kLdP]
  float* vs = ks + kKeys * kLd;    // [kKeys][kLd]
  float* ps = ks;
  __shared__ int64_t sums[kThreads / 32];
  __shared__ ChunkStart start;
  __shared__ int nonfinite;        // a drafted node's V is not finite

  chunk_find_start<kThreads>(P, blockIdx.x, P.ctas, sums, &start);
  launch_dependents();  // the merge kernel may start up; it waits for this grid's results
  ChunkWalk walk(P, start, blockIdx.x);
  ChunkSegment seg;
  const float scale_log2 = p.scale * kLog2e;
  const int page_mask = (1 << p.page_shift) - 1;

  bool more = walk.next(P, seg);
  if (tid == 0) chunk_write_join(P, start, blockIdx.x, more ? &seg : nullptr);
  for (; more; more = walk.next(P, seg)) {
    const int rows_left = seg.queries * P.group - seg.row0;  // valid rows of this unit (may exceed kRows)
    const int32_t* table = chunk_table(P, seg.b, seg.g);
    const int64_t plane = (int64_t(p.layer) * p.num_kv_heads + seg.g) * p.capacity;
    const T* kp = static_cast<const T*>(p.k_pool) + plane * D;
    const T* vp = static_cast<const T*>(p.v_pool) + plane * D;

    const ChunkRows unit(seg.t0, seg.hl0);
    __syncthreads();  // the previous segment's shared tiles are done with
    if (tid == 0) nonfinite = 0;
    for (int i = tid; i < kRows * kD; i += kThreads) {
      const int r = i / kD, d = i - r * kD;
      float v = 0.f;
      if (r < rows_left && d < D) {
        int t, hl;
        unit.at(P, r, t, hl);
        v = Elem<T>::to_float(static_cast<const T*>(p.q)[seg.q_base + t * p.q_st + hl * p.q_sh + d]);
      }
      qs[r * kLd + d] = v;
    }

    float o[kR][kChunks][4], m_run[kR], l_run[kR];
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      m_run[i] = -INFINITY;
      l_run[i] = 0.f;
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][c][e] = 0.f;
    }

    for (int tile = seg.k_lo; tile < seg.k_hi; ++tile) {
      const int k0 = tile * kKeys;
      // a tile never crosses a page: pages are powers of two of at least 64 tokens
      const int lp = k0 >> p.page_shift;
      int32_t page = -1;
      if (!seg.refused) {
        page = table[lp];
        if (page < 0 || page >= p.num_pages) {
          if (tid == 0) flag_error(p.error_word, HYT_DEVERR_PAGE_RANGE);
          page = -1;
        }
      }
      const int kv_here = page < 0 ? 0 : min(seg.kv - k0, kKeys);  // keys of the tile that exist
      __syncthreads();  // Q stored (first tile); P and V of the previous tile read
      {
        constexpr int kChunk16 = kD / kPer;  // 16-byte chunks of a padded row
        constexpr int kEach = kKeys * kChunk16 / kThreads;
        constexpr int kBatch = kEach % 4 == 0 ? 4 : (kEach % 3 == 0 ? 3 : 2);  // pairs of loads that go out together
        static_assert(kEach * kThreads == kKeys * kChunk16 && kEach % kBatch == 0, "whole batches of the tile's chunks");
        const int64_t slot0 = (int64_t(max(page, 0)) << p.page_shift) + (k0 & page_mask);
        const bool check = k0 + kKeys > seg.len;
#pragma unroll 1
        for (int i0 = 0; i0 < kEach; i0 += kBatch) {
          uint4 kraw[kBatch], vraw[kBatch];
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            const int i = tid + (i0 + u) * kThreads, r = i / kChunk16, d = (i - r * kChunk16) * kPer;
            kraw[u] = vraw[u] = make_uint4(0u, 0u, 0u, 0u);
            if (r < kv_here && d < D) {
              kraw[u] = __ldg(reinterpret_cast<const uint4*>(kp + (slot0 + r) * D + d));
              vraw[u] = __ldg(reinterpret_cast<const uint4*>(vp + (slot0 + r) * D + d));
            }
          }
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            const int i = tid + (i0 + u) * kThreads, r = i / kChunk16, d = (i - r * kChunk16) * kPer;
            float kf[kPer], vf[kPer];
            widen16<T>(kraw[u], kf);
            widen16<T>(vraw[u], vf);
            if (check && k0 + r >= seg.len) {
#pragma unroll
              for (int e = 0; e < kPer; ++e)
                if (!isfinite(vf[e])) {
                  vf[e] = 0.f;
                  nonfinite = 1;
                }
            }
#pragma unroll
            for (int e = 0; e < kPer; e += 4) {
              *reinterpret_cast<float4*>(ks + r * kLd + d + e) = make_float4(kf[e], kf[e + 1], kf[e + 2], kf[e + 3]);
              *reinterpret_cast<float4*>(vs + r * kLd + d + e) = make_float4(vf[e], vf[e + 1], vf[e + 2], vf[e + 3]);
            }
          }
        }
      }
      __syncthreads();

      // ---- S: rows ty * kR + i, keys tx + 16 j
      float s[kR][4];
#pragma unroll
      for (int i = 0; i < kR; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 4
      for (int d = 0; d < kD; d += 4) {
        float4 kf[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) kf[j] = *reinterpret_cast<const float4*>(ks + (tx + 16 * j) * kLd + d);
#pragma unroll
        for (int i = 0; i < kR; ++i) {
          const float4 qf = *reinterpret_cast<const float4*>(qs + (ty * kR + i) * kLd + d);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            s[i][j] = fmaf(qf.w, kf[j].w, fmaf(qf.z, kf[j].z, fmaf(qf.y, kf[j].y, fmaf(qf.x, kf[j].x, s[i][j]))));
        }
      }

      // ---- mask, online softmax (base 2); a row's 64 keys sit on 16 lanes
      float pr[kR][4];
#pragma unroll
      for (int i = 0; i < kR; ++i) {
        const int row = ty * kR + i;
        uint64_t seen = ~0ull;
        if (page < 0 || row >= rows_left)
          seen = 0ull;
        else if (k0 + kKeys > seg.len) {
          int t, hl;
          unit.at(P, row, t, hl);
          seen = chunk_visible64(P, seg, t, k0 - seg.len);
        }
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[i][j] = (seen >> (tx + 16 * j)) & 1 ? s[i][j] * scale_log2 : -INFINITY;
          mx = fmaxf(mx, s[i][j]);
        }
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        const float m_new = fmaxf(m_run[i], mx);
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = ex2(m_run[i] - m_use);  // 0 before anything was seen
        m_run[i] = m_new;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          pr[i][j] = ex2(s[i][j] - m_use);
          sum += pr[i][j];
        }
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        l_run[i] = l_run[i] * alpha + sum;
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][c][e] *= alpha;
      }
      __syncthreads();  // K read by everyone: P takes its place
#pragma unroll
      for (int i = 0; i < kR; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) ps[(ty * kR + i) * kLdP + tx + 16 * j] = pr[i][j];
      __syncwarp();  // a row's P is written and read by the same half-warp

      // ---- O += P V: dims tx * 4 + 64 c
#pragma unroll 2
      for (int k = 0; k < kKeys; k += 4) {
        float4 pf[kR];
#pragma unroll
        for (int i = 0; i < kR; ++i) pf[i] = *reinterpret_cast<const float4*>(ps + (ty * kR + i) * kLdP + k);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            const float4 vf = *reinterpret_cast<const float4*>(vs + (k + kk) * kLd + c * 64 + tx * 4);
#pragma unroll
            for (int i = 0; i < kR; ++i) {
              const float w = kk == 0 ? pf[i].x : (kk == 1 ? pf[i].y : (kk == 2 ? pf[i].z : pf[i].w));
              o[i][c][0] = fmaf(w, vf.x, o[i][c][0]);
              o[i][c][1] = fmaf(w, vf.y, o[i][c][1]);
              o[i][c][2] = fmaf(w, vf.z, o[i][c][2]);
              o[i][c][3] = fmaf(w, vf.w, o[i][c][3]);
            }
          }
        }
      }
    }

    __syncthreads();
    const bool fix = nonfinite != 0;
    const int64_t slot = int64_t(blockIdx.x) * 2 + (seg.first ? 0 : 1);
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      const int row = ty * kR + i;
      if (row >= rows_left) continue;
      int t, hl;
      unit.at(P, row, t, hl);
      if (fix && !seg.refused) {  // non-finite V of the nodes this row sees, left out above
        const int lo = max(seg.k_lo * kKeys, seg.len), hi = min(seg.k_hi * kKeys, seg.kv);
        for (int pos = lo; pos < hi; ++pos) {
          if (!(chunk_visible64(P, seg, t, pos - seg.len) & 1)) continue;
          const int32_t page = table[pos >> p.page_shift];
          if (page < 0 || page >= p.num_pages) continue;
          const T* vrow = vp + ((int64_t(page) << p.page_shift) + (pos & page_mask)) * D;
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int d = c * 64 + tx * 4 + e;
              if (d >= D) continue;
              const float v = Elem<T>::to_float(vrow[d]);
              if (!isfinite(v)) o[i][c][e] += v;
            }
        }
      }
      if (seg.whole) {
        const float inv = l_run[i] == 0.f ? 0.f : 1.f / l_run[i];
        T* out = static_cast<T*>(p.out) + seg.o_base + t * p.o_st + hl * p.o_sh;
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int d = c * 64 + tx * 4 + e;
            if (d < D) out[d] = Elem<T>::from_float(o[i][c][e] * inv);
          }
      } else {
        float4* wo = chunk_partial_o(P, slot);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const int d = c * 64 + tx * 4;
          if (d < D)
            wo[int64_t(d / 4) * P.unit_rows + row] = make_float4(o[i][c][0], o[i][c][1], o[i][c][2], o[i][c][3]);
        }
        if (tx == 0) chunk_partial_ml(P, slot)[row] = make_float2(m_run[i], l_run[i]);
      }
    }
  }
}

// Units of up to kRows <= 8 rows: a decode step over chosen pages, small trees. Per 64-key tile
// a key belongs to 4 lanes, each with every 4th 16-byte chunk of the key in registers (Q from
// shared memory, the lanes' sums meet by shuffles); one warp per row then takes the tile's
// softmax through shared memory; for O += P V warp w has keys 8 w .., a lane 16 bytes of
// the dims, and the warps' O meet at the end. K and V are read from global memory once,
// straight into registers, a tile's K and half of its V in flight together. A masked key's P is
// an exact 0 and its V is not multiplied, so values that are not finite stay where they are
// seen. Bound: HBM reads of K and V. On 16 requests x 25K
// fp32 tokens, 30 pages, 4 rows: 151 us, 3.5 TB/s; staging K and V in shared memory for 16-row
// blocks took 366 us, 1.4 TB/s.
// kWide: keys of more than 32 16-byte chunks (fp32 heads above 128).
template <typename T, int kRows, bool kWide>
__global__ void __launch_bounds__(kThreads, kRows * (kWide ? 2 : 1) * int(16 / sizeof(T)) <= 32 ? 2 : 1)
    chunk_attention_rows_kernel(const ChunkParams P) {
  constexpr int kPer = 16 / int(sizeof(T));
  constexpr int kKChunks = kWide ? 16 : 8;  // 16-byte chunks of a key per lane
  constexpr int kVChunks = kWide ? 2 : 1;   // of a V row per lane
  constexpr int kWarps = kThreads / 32, kVKeys = kKeys / kWarps, kVBatch = 4;
  const AttentionParams& p = P.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int D = p.head_dim, chunks = D / kPer;

  extern __shared__ __align__(16) float smem[];
  float* qs = smem;                                  // [kRows][D]
  float* ps = qs + kRows * D;                        // [2][kRows][kKeys]
  float* red = ps + 2 * kRows * kKeys;               // [kWarps][kRows][D], at a segment's end
  __shared__ float alpha_s[2][kRows], m_s[kRows], l_s[kRows];
  __shared__ int64_t sums[kWarps];
  __shared__ ChunkStart start;

  chunk_find_start<kThreads>(P, blockIdx.x, P.ctas, sums, &start);
  launch_dependents();  // the merge kernel may start up; it waits for this grid's results
  ChunkWalk walk(P, start, blockIdx.x);
  ChunkSegment seg;
  const float scale_log2 = p.scale * kLog2e;
  const int page_mask = (1 << p.page_shift) - 1;
  const int key = tid >> 2, j4 = tid & 3;  // S: this lane's key of the tile and chunks j4 + 4 t

  bool more = walk.next(P, seg);
  if (tid == 0) chunk_write_join(P, start, blockIdx.x, more ? &seg : nullptr);
  for (; more; more = walk.next(P, seg)) {
    const int rows = min(seg.queries * P.group - seg.row0, kRows);
    const ChunkRows unit(seg.t0, seg.hl0);
    const int32_t* table = chunk_table(P, seg.b, seg.g);
    const int64_t plane = (int64_t(p.layer) * p.num_kv_heads + seg.g) * p.capacity;
    const T* kp = static_cast<const T*>(p.k_pool) + plane * D;
    const T* vp = static_cast<const T*>(p.v_pool) + plane * D;
    __syncthreads();  // the previous segment's shared values are done with
    for (int i = tid; i < kRows * D; i += kThreads) {
      const int r = i / D, d = i - r * D;
      float v = 0.f;
      if (r < rows) {
        int t, hl;
        unit.at(P, r, t, hl);
        v = Elem<T>::to_float(static_cast<const T*>(p.q)[seg.q_base + t * p.q_st + hl * p.q_sh + d]);
      }
      qs[i] = v;
    }
    if (tid < kRows) m_s[tid] = -INFINITY, l_s[tid] = 0.f;
    __syncthreads();
    float o[kRows][kVChunks][kPer];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int c = 0; c < kVChunks; ++c)
#pragma unroll
        for (int e = 0; e < kPer; ++e) o[r][c][e] = 0.f;

    for (int tile = seg.k_lo; tile < seg.k_hi; ++tile) {
      const int k0 = tile * kKeys, buf = tile & 1;
      int32_t page = -1;
      if (!seg.refused) {
        page = table[k0 >> p.page_shift];
        if (page < 0 || page >= p.num_pages) {
          if (tid == 0) flag_error(p.error_word, HYT_DEVERR_PAGE_RANGE);
          page = -1;
        }
      }
      const int kv_here = page < 0 ? 0 : min(seg.kv - k0, kKeys);  // keys of the tile that exist
      const int64_t slot0 = (int64_t(max(page, 0)) << p.page_shift) + (k0 & page_mask);
      uint4 kraw[kKChunks];
#pragma unroll
      for (int t = 0; t < kKChunks; ++t) {
        const int c = j4 + 4 * t;
        kraw[t] = make_uint4(0u, 0u, 0u, 0u);
        if (c < chunks && key < kv_here)
          kraw[t] = __ldg(reinterpret_cast<const uint4*>(kp + (slot0 + key) * D) + c);
      }
      uint4 vraw[kVBatch][kVChunks];
      auto load_v = [&](int first) {  // keys first .. of this warp
#pragma unroll
        for (int u = 0; u < kVBatch; ++u)
#pragma unroll
          for (int c = 0; c < kVChunks; ++c) {
            const int k = warp * kVKeys + first + u, ch = lane + 32 * c;
            vraw[u][c] = make_uint4(0u, 0u, 0u, 0u);
            if (ch < chunks && k < kv_here) vraw[u][c] = __ldg(reinterpret_cast<const uint4*>(vp + (slot0 + k) * D) + ch);
          }
      };
      load_v(0);

      // ---- S of this lane's key, all rows
      float s[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) s[r] = 0.f;
#pragma unroll
      for (int t = 0; t < kKChunks; ++t) {
        const int c = j4 + 4 * t;
        if (4 * t >= chunks) continue;  // the same for every lane
        float kf[kPer];
        widen16<T>(kraw[t], kf);
        const int d = min(c, chunks - 1) * kPer;  // lanes past the row's end multiply by zeros
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
#pragma unroll
          for (int e = 0; e < kPer; e += 4) {
            const float4 qf = *reinterpret_cast<const float4*>(qs + r * D + d + e);
            s[r] = fmaf(qf.x, kf[e], fmaf(qf.y, kf[e + 1], fmaf(qf.z, kf[e + 2], fmaf(qf.w, kf[e + 3], s[r]))));
          }
        }
      }
      const bool masked = page < 0 || k0 + kKeys > seg.len;
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        s[r] += __shfl_xor_sync(0xffffffffu, s[r], 1);
        s[r] += __shfl_xor_sync(0xffffffffu, s[r], 2);
        if (j4 == (r & 3)) {
          bool seen = r < rows && page >= 0;
          if (masked && seen && k0 + key >= seg.len) {
            int t, hl;
            unit.at(P, r, t, hl);
            seen = chunk_visible64(P, seg, t, k0 + key - seg.len) & 1;
          }
          ps[(buf * kRows + r) * kKeys + key] = seen ? s[r] * scale_log2 : -INFINITY;
        }
      }
      __syncthreads();
      // ---- softmax of the tile, a warp per row
      for (int r = warp; r < kRows; r += kWarps) {
        float* row = ps + (buf * kRows + r) * kKeys;
        const float x0 = row[lane], x1 = row[lane + 32];
        float mx = fmaxf(x0, x1);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        const float m_old = m_s[r], m_new = fmaxf(m_old, mx), m_use = m_new == -INFINITY ? 0.f : m_new;
        const float p0 = ex2(x0 - m_use), p1 = ex2(x1 - m_use);
        float sum = p0 + p1;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        row[lane] = p0;
        row[lane + 32] = p1;
        if (lane == 0) {
          const float alpha = ex2(m_old - m_use);  // 0 before anything was seen
          alpha_s[buf][r] = alpha;
          l_s[r] = l_s[r] * alpha + sum;
          m_s[r] = m_new;
        }
      }
      __syncthreads();
      // ---- O += P V
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const float alpha = alpha_s[buf][r];
#pragma unroll
        for (int c = 0; c < kVChunks; ++c)
#pragma unroll
          for (int e = 0; e < kPer; ++e) o[r][c][e] *= alpha;
      }
#pragma unroll
      for (int first = 0; first < kVKeys; first += kVBatch) {
        float vf[kVBatch][kVChunks][kPer];
#pragma unroll
        for (int u = 0; u < kVBatch; ++u)
#pragma unroll
          for (int c = 0; c < kVChunks; ++c) widen16<T>(vraw[u][c], vf[u][c]);
        if (first + kVBatch < kVKeys) load_v(first + kVBatch);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float4 w4 = *reinterpret_cast<const float4*>(ps + (buf * kRows + r) * kKeys + warp * kVKeys + first);
          const float w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
          for (int u = 0; u < kVBatch; ++u) {
            if (masked && w[u] == 0.f) continue;  // warp-uniform
#pragma unroll
            for (int c = 0; c < kVChunks; ++c)
#pragma unroll
              for (int e = 0; e < kPer; ++e) o[r][c][e] = fmaf(w[u], vf[u][c][e], o[r][c][e]);
          }
        }
      }
    }

    // ---- the warps' O meet in shared memory
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int c = 0; c < kVChunks; ++c) {
        const int ch = lane + 32 * c;
        if (ch < chunks)
#pragma unroll
          for (int e = 0; e < kPer; e += 4)
            *reinterpret_cast<float4*>(red + (warp * kRows + r) * D + ch * kPer + e) =
                make_float4(o[r][c][e], o[r][c][e + 1], o[r][c][e + 2], o[r][c][e + 3]);
      }
    __syncthreads();
    const int64_t slot = int64_t(blockIdx.x) * 2 + (seg.first ? 0 : 1);
    for (int i = tid; i < rows * (D / 4); i += kThreads) {
      const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(red + (w * kRows + r) * D + d);
        sum = make_float4(sum.x + x.x, sum.y + x.y, sum.z + x.z, sum.w + x.w);
      }
      if (seg.whole) {
        const float l = l_s[r], inv = l == 0.f ? 0.f : 1.f / l;
        int t, hl;
        unit.at(P, r, t, hl);
        T* out = static_cast<T*>(p.out) + seg.o_base + t * p.o_st + hl * p.o_sh + d;
        out[0] = Elem<T>::from_float(sum.x * inv);
        out[1] = Elem<T>::from_float(sum.y * inv);
        out[2] = Elem<T>::from_float(sum.z * inv);
        out[3] = Elem<T>::from_float(sum.w * inv);
      } else {
        chunk_partial_o(P, slot)[int64_t(d / 4) * P.unit_rows + r] = sum;
        if (d == 0) chunk_partial_ml(P, slot)[r] = make_float2(m_s[r], l_s[r]);
      }
    }
  }
}

template <typename T, int kRows, bool kWide>
cudaError_t launch_rows(const ChunkParams& p, cudaStream_t stream) {
  auto kernel = chunk_attention_rows_kernel<T, kRows, kWide>;
  const int smem = (kRows * p.a.head_dim + 2 * kRows * kKeys + kThreads / 32 * kRows * p.a.head_dim) * 4;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  if (p.after_selection) return launch_after(kernel, dim3(p.ctas), kThreads, smem, stream, p);
  kernel<<<p.ctas, kThreads, smem, stream>>>(p);
  return cudaGetLastError();
}

// ------------------------------------------------------------------ merge
constexpr int kMergeThreads = 256;

// CTA (c - 1, y): rows 32 y .. of the unit that CTA c's join record names. Warp w, lane r: row r,
// dims 4 (w + 8 k): the partials are stored with consecutive rows next to each other, so every
// load is 512 contiguous bytes; the joined rows go through shared memory so that the stores
// are contiguous too (storing from the accumulators, 2 bytes of 32 rows at a time, cost
// 30 us on 8 requests x 256 nodes). kAhead parts' loads at a time. Fixed order, no atomics.
// Launched while the attention kernel runs; waits for its results before it reads anything.
constexpr int kMergeRows = 32;

// kGroups: ceil(head_dim / 32)
template <typename T, int kGroups>
__global__ void __launch_bounds__(kMergeThreads) chunk_merge_kernel(const ChunkParams P) {
  __shared__ T rows_s[kMergeRows][kGroups * 32 + 2];
  const AttentionParams& p = P.a;
  const int c = int(blockIdx.x) + 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = int(blockIdx.y) * kMergeRows + lane;
  wait_for_primary();
  const int4 j0 = __ldcg(reinterpret_cast<const int4*>(P.ws_join + c));
  const int4 j1 = __ldcg(reinterpret_cast<const int4*>(P.ws_join + c) + 1);
  const int b = j0.x, g = j0.y, row0 = j0.z, rows = j0.w, slot0 = j1.x, parts = j1.y, start = j1.z;
  const int here = min(rows - int(blockIdx.y) * kMergeRows, kMergeRows);  // rows of this CTA
  if (here <= 0) return;
  const int dims4 = p.head_dim / 4;
  constexpr int kAhead = kGroups <= 4 ? 4 : 2;
  float m = -INFINITY, l = 0.f;
  float4 o[kGroups];
#pragma unroll
  for (int k = 0; k < kGroups; ++k) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < parts; i0 += kAhead) {
    float2 ml[kAhead];
    float4 v[kAhead][kGroups];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t slot = i0 + u == 0 ? slot0 : int64_t(c - 1 + i0 + u) * 2;
      ml[u] = make_float2(-INFINITY, 0.f);
      if (i0 + u < parts && lane < here) {
        ml[u] = __ldcg(&chunk_partial_ml(P, slot)[row]);
#pragma unroll
        for (int k = 0; k < kGroups; ++k)
          if (warp + 8 * k < dims4) v[u][k] = __ldcg(&chunk_partial_o(P, slot)[int64_t(warp + 8 * k) * P.unit_rows + row]);
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (ml[u].y == 0.f) continue;  // nothing seen in this part
      const float m_new = fmaxf(m, ml[u].x), m_use = m_new == -INFINITY ? 0.f : m_new;
      const float f = ex2(ml[u].x - m_use), keep = m == -INFINITY ? 0.f : ex2(m - m_use);
      l = fmaf(ml[u].y, f, l * keep);
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        o[k].x = fmaf(v[u][k].x, f, o[k].x * keep);
        o[k].y = fmaf(v[u][k].y, f, o[k].y * keep);
        o[k].z = fmaf(v[u][k].z, f, o[k].z * keep);
        o[k].w = fmaf(v[u][k].w, f, o[k].w * keep);
      }
      m = m_new;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int k = 0; k < kGroups; ++k) {
    const int d = (warp + 8 * k) * 4;
    if (d >= p.head_dim) break;
    rows_s[lane][d] = Elem<T>::from_float(o[k].x * inv);
    rows_s[lane][d + 1] = Elem<T>::from_float(o[k].y * inv);
    rows_s[lane][d + 2] = Elem<T>::from_float(o[k].z * inv);
    rows_s[lane][d + 3] = Elem<T>::from_float(o[k].w * inv);
  }
  __syncthreads();
  const ChunkRows unit(row0 / P.group, row0 % P.group);
  const int64_t o_base = (p.q_start != nullptr ? int64_t(start) * p.o_st : int64_t(b) * p.o_sb) + int64_t(g) * P.group * p.o_sh;
  for (int r = warp; r < here; r += kMergeThreads / 32) {
    int t, hl;
    unit.at(P, int(blockIdx.y) * kMergeRows + r, t, hl);
    T* out = static_cast<T*>(p.out) + o_base + t * p.o_st + hl * p.o_sh;
#pragma unroll
    for (int d = lane; d < kGroups * 32; d += 32)
      if (d < p.head_dim) out[d] = rows_s[r][d];
  }
}

template <typename T>
cudaError_t launch_merge(const ChunkParams& p, cudaStream_t stream) {
  const dim3 grid(unsigned(p.ctas - 1), unsigned((p.unit_rows + kMergeRows - 1) / kMergeRows));
  if (p.a.head_dim <= 64) return launch_after(chunk_merge_kernel<T, 2>, grid, kMergeThreads, 0, stream, p);
  if (p.a.head_dim <= 128) return launch_after(chunk_merge_kernel<T, 4>, grid, kMergeThreads, 0, stream, p);
  return launch_after(chunk_merge_kernel<T, 8>, grid, kMergeThreads, 0, stream, p);
}

template <typename T, int kRows, int kChunks>
constexpr int general_smem() {
  return (kRows + 2 * kKeys) * (kChunks * 64 + 4) * 4;
}

template <typename T, int kRows, int kChunks>
cudaError_t launch_general(const ChunkParams& p, cudaStream_t stream) {
  static_assert(kRows * (kKeys + 4) <= kKeys * (kChunks * 64 + 4), "P must fit in K's tile");
  auto kernel = chunk_attention_general_kernel<T, kRows, kChunks>;
  constexpr int smem = general_smem<T, kRows, kChunks>();
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  if (p.after_selection) return launch_after(kernel, dim3(p.ctas), kThreads, smem, stream, p);
  kernel<<<p.ctas, kThreads, smem, stream>>>(p);
  return cudaGetLastError();
}

template <typename T, int kRows>
cudaError_t launch_general_dim(const ChunkParams& p, cudaStream_t stream) {
  switch ((p.a.head_dim + 63) / 64) {
    case 1: return launch_general<T, kRows, 1>(p, stream);
    case 2: return launch_general<T, kRows, 2>(p, stream);
    case 3: return launch_general<T, kRows, 3>(p, stream);
    default: return launch_general<T, kRows, 4>(p, stream);
  }
}

template <typename T>
cudaError_t launch_general_rows(const ChunkParams& p, cudaStream_t stream) {
  if constexpr (sizeof(T) == 4) {
    if (p.a.head_dim > 128) {
      switch (p.unit_rows) {
        case 4: return launch_rows<T, 4, true>(p, stream);
        case 8: return launch_rows<T, 8, true>(p, stream);
        case 16: return launch_general_dim<T, 16>(p, stream);
        default: return launch_general_dim<T, 64>(p, stream);
      }
    }
  }
  switch (p.unit_rows) {
    case 4: return launch_rows<T, 4, false>(p, stream);
    case 8: return launch_rows<T, 8, false>(p, stream);
    case 16: return launch_general_dim<T, 16>(p, stream);
    default: return launch_general_dim<T, 64>(p, stream);
  }
}

}  // namespace

// Rows per unit by the rows of the largest request: 4 or 8 go to the kernel that reads K and V
// straight into registers (151 us against 366 for 4 rows on 16 x 25K fp32 tokens, 30 pages read),
// 16 to the staged one (188 us against 251 for the other on 16 x 2K tokens x 16 rows, whose
// accumulators leave it one CTA per SM), more to blocks of 64.
ChunkShape chunk_shape_general(int64_t max_rows, int dtype, int head_dim, int num_sms) {
  (void)dtype;
  if (max_rows <= 8) {  // two CTAs per SM fit whatever the head size
    return {max_rows <= 4 ? 4 : 8, kKeys, 2, num_sms * 2};
  }
  // resident CTAs per SM by shared memory (228 KB per SM, 1 KB reserved per CTA)
  const int rows = max_rows <= 16 ? 16 : 64;
  const int smem = (rows + 2 * kKeys) * ((head_dim + 63) / 64 * 64 + 4) * 4 + 1024;
  return {rows, kKeys, 1, num_sms * (smem * 3 <= 228 * 1024 ? 3 : (smem * 2 <= 228 * 1024 ? 2 : 1))};
}

cudaError_t run_chunk_attention_general(const ChunkParams& p, int dtype, cudaStream_t stream) {
  switch (dtype) {
    case HYT_DTYPE_BF16: return launch_general_rows<__nv_bfloat16>(p, stream);
    case HYT_DTYPE_F16: return launch_general_rows<__half>(p, stream);
    default: return launch_general_rows<float>(p, stream);
  }
}

cudaError_t run_chunk_merge(const ChunkParams& p, int dtype, cudaStream_t stream) {
  if (p.ctas < 2) return cudaSuccess;
  switch (dtype) {
    case HYT_DTYPE_BF16: return launch_merge<__nv_bfloat16>(p, stream);
    case HYT_DTYPE_F16: return launch_merge<__half>(p, stream);
    default: return launch_merge<float>(p, stream);
  }
}

}  // namespace hyt
