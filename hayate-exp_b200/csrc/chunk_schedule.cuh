// How the chunk-attention kernels (tree_attention*.cu) share out their work.
//
// A unit is (request b, KV head g, block of `unit_rows` query rows); rows of a request are
// numbered t * group + hl (query t, local head hl). A unit streams the request's keys in
// tiles of `tile_keys`, and starting and ending it costs about as much as `unit_cost` tiles.
// All units, request after request, form one line of W positions: unit_cost for a unit's
// ends, then its tiles. CTA c of G takes W / G of them, the first W % G CTAs one more: every CTA
// works about as long whatever the lengths, and W needs no host copy of the lengths, so a
// captured launch follows them. A CTA's stretch falls into segments, one per unit it has
// tiles of. A segment that covers its unit writes the rows; another writes a partial
// (unnormalised O, running max, sum) to one of the CTA's two slots (slot 0: its first segment,
// slot 1: its last; those between are whole), and the merge kernel joins a unit's partials
// in order, as the join record of the CTA with the unit's second part says.
#pragma once

#include "common.cuh"
#include "kernels.cuh"

namespace hyt {

struct ChunkRequest {
  int len, queries;      // cached tokens, queries of this step
  int start;             // row of the first query on a packed batch's token axis
  int row_blocks, tiles; // units per KV head, key tiles per unit
  bool refused;          // lengths the page table cannot hold: nothing is visible
};

// Lengths of request b. One whose rows leave the token axis gets no work (its rows are not
// known to be its own); one whose length is negative or needs more pages than its table
// row holds gets one tile in which nothing is visible, so its rows become zeros.
__device__ __forceinline__ ChunkRequest chunk_request(const ChunkParams& P, int b, int& why) {
  const AttentionParams& p = P.a;
  ChunkRequest r{0, 0, 0, 0, 0, false};
  const bool packed = p.q_start != nullptr;
  const int len = p.cache_lens[b];  // the loads go out together
  const int s = packed ? p.q_start[b] : 0;
  const int n = packed ? p.q_len[b] : p.query_len;
  if (packed && (n < 0 || n > p.query_len || s < 0 || int64_t(s) + n > p.total_tokens)) {
    why |= HYT_DEVERR_PACKED_RANGE;
    return r;
  }
  if (n == 0) return r;
  r.len = len;
  r.queries = n;
  r.start = s;
  r.row_blocks = int((int64_t(n) * P.group + P.unit_rows - 1) >> P.unit_shift);
  const int64_t kv = int64_t(len) + n;
  if (len < 0 || kv > (int64_t(P.table_width) << p.page_shift) || kv > INT32_MAX - 256) {
    why |= HYT_DEVERR_TABLE_RANGE;
    r.refused = true;
    r.tiles = 1;
    return r;
  }
  r.tiles = int((kv + P.tile_keys - 1) >> P.tile_shift);
  return r;
}

// Line positions of a request.
__device__ __forceinline__ int64_t chunk_work(const ChunkParams& P, const ChunkRequest& r) {
  return r.tiles == 0 ? 0 : int64_t(P.a.num_kv_heads) * r.row_blocks * (r.tiles + P.unit_cost);
}

struct ChunkStart {
  int64_t total;  // W
  int64_t base;   // W / CTAs, and the remainder: the first `rem` CTAs take one more
  int64_t off;    // first position of the CTA within request b's
  int rem;
  int b;

  __device__ __forceinline__ int64_t begin(int c) const { return base * c + min(c, rem); }
};

// a / b for a >= 0, b > 0; nearly always within 32 bits, where it is several times cheaper
__device__ __forceinline__ int64_t chunk_div(int64_t a, int b) {
  return a <= 0xFFFFFFFFll ? int64_t(uint32_t(a) / uint32_t(b)) : a / b;
}

// Where CTA c of `ctas` starts. Called by all kThreads threads; `sums` holds kThreads / 32
// shared entries. Ends with a barrier.
template <int kThreads>
__device__ __forceinline__ void chunk_find_start(const ChunkParams& P, int c, int ctas, int64_t* sums,
                                                 ChunkStart* start) {
  constexpr int kWarps = kThreads / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  wait_for_primary();  // page selection writes the lengths and pages of a decode over chosen pages
  const int per = (P.a.batch + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, P.a.batch), b1 = min(b0 + per, P.a.batch);
  int why = 0;
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += chunk_work(P, chunk_request(P, b, why));
  if (why && c == 0) flag_error(P.a.error_word, why);
  int64_t scan = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, scan, off);
    if (lane >= off) scan += v;
  }
  if (lane == 31) sums[warp] = scan;
  if (tid == 0) start->b = 0, start->off = 0;
  __syncthreads();
  int64_t before = scan - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sums[w];
    total += sums[w];
  }
  const int64_t base = chunk_div(total, ctas);
  const int rem = int(total - base * ctas);
  const int64_t begin = base * c + min(c, rem);
  if (tid == 0) {
    start->total = total;
    start->base = base;
    start->rem = rem;
  }
  if (begin >= before && begin < before + mine) {  // one thread, if total > 0 and begin < total
    int64_t off = begin - before;
    int b = b0;
    for (; b < b1 - 1; ++b) {
      const int64_t w = chunk_work(P, chunk_request(P, b, why));
      if (off < w) break;
      off -= w;
    }
    start->b = b;
    start->off = off;
  }
  __syncthreads();
}

// The same for one full warp on its own (no barrier); the result on every lane, with request
// start.b in `r`.
__device__ __forceinline__ ChunkStart chunk_find_start_warp(const ChunkParams& P, int c, int ctas, ChunkRequest& r) {
  const int lane = threadIdx.x & 31;
  wait_for_primary();
  int64_t before_all = 0, mine = 0;
  int why = 0;
  r = ChunkRequest{0, 0, 0, 0, 0, false};
  if (lane < P.a.batch) {  // the first 32 requests are looked at once
    r = chunk_request(P, lane, why);
    mine = chunk_work(P, r);
  }
  int64_t total = mine;
  for (int b0 = 32; b0 < P.a.batch; b0 += 32)
    if (b0 + lane < P.a.batch) total += chunk_work(P, chunk_request(P, b0 + lane, why));
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, off);
    why |= __shfl_xor_sync(0xffffffffu, why, off);
  }
  if (why && c == 0 && lane == 0) flag_error(P.a.error_word, why);
  ChunkStart start;
  start.total = total;
  start.base = chunk_div(total, ctas);
  start.rem = int(total - start.base * ctas);
  start.off = 0;
  start.b = 0;
  const int64_t begin = start.begin(c);
  for (int b0 = 0; b0 < P.a.batch && begin < total; b0 += 32) {  // the request that holds `begin`
    if (b0 > 0) {
      mine = 0;
      if (b0 + lane < P.a.batch) {
        r = chunk_request(P, b0 + lane, why);
        mine = chunk_work(P, r);
      }
    }
    int64_t scan = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, scan, off);
      if (lane >= off) scan += v;
    }
    const int64_t before = before_all + scan - mine;
    const uint32_t holds = __ballot_sync(0xffffffffu, begin >= before && begin < before + mine);
    if (holds) {
      const int from = __ffs(holds) - 1;
      start.b = b0 + from;
      start.off = begin - __shfl_sync(0xffffffffu, before, from);
      r.len = __shfl_sync(0xffffffffu, r.len, from);
      r.queries = __shfl_sync(0xffffffffu, r.queries, from);
      r.start = __shfl_sync(0xffffffffu, r.start, from);
      r.row_blocks = __shfl_sync(0xffffffffu, r.row_blocks, from);
      r.tiles = __shfl_sync(0xffffffffu, r.tiles, from);
      r.refused = __shfl_sync(0xffffffffu, r.refused ? 1 : 0, from) != 0;
      break;
    }
    before_all += __shfl_sync(0xffffffffu, scan, 31);
  }
  return start;
}

struct ChunkSegment {
  int b, g, row0;        // request, KV head, first row of the unit
  int len, queries, kv;  // cached tokens, queries, their sum
  int k_lo, k_hi;        // key tiles [k_lo, k_hi) of the unit
  int t0, hl0;           // query and local head of row0
  int64_t q_base, o_base, mask_row;  // query 0 of head group g in q and out (elements), in the mask (rows)
  bool whole, first, refused;
};

// Walks a CTA's segments; every role of the CTA walks the same ones.
struct ChunkWalk {
  int64_t left, off;  // positions left to the CTA; first of them within request b's
  int64_t work;
  int b;
  bool started;
  ChunkRequest r;

  __device__ __forceinline__ ChunkWalk(const ChunkParams& P, const ChunkStart& s, int c) {
    left = s.begin(c + 1) - s.begin(c);
    off = s.off;
    b = s.b;
    started = false;
    work = 0;
    if (left > 0) load(P);
  }
  // with request s.b at hand
  __device__ __forceinline__ ChunkWalk(const ChunkParams& P, const ChunkStart& s, int c, const ChunkRequest& first) {
    left = s.begin(c + 1) - s.begin(c);
    off = s.off;
    b = s.b;
    started = false;
    r = first;
    work = chunk_work(P, r);
  }
  __device__ __forceinline__ void load(const ChunkParams& P) {
    int why = 0;
    r = chunk_request(P, b, why);
    work = chunk_work(P, r);
  }
  __device__ __forceinline__ bool next(const ChunkParams& P, ChunkSegment& s) {
    while (left > 0) {
      while (off >= work) {  // the next request that has work (left > 0: there is one)
        off -= work;
        ++b;
        load(P);
      }
      const int span = r.tiles + P.unit_cost;
      const int64_t unit = chunk_div(off, span);
      const int o = int(off - unit * span), n = int(min(int64_t(span - o), left));
      s.k_lo = max(o - P.unit_cost, 0);
      s.k_hi = o + n - P.unit_cost;
      off += n;
      left -= n;
      if (s.k_hi <= s.k_lo) continue;  // the stretch ends before the unit's first tile
      s.b = b;
      s.g = int(chunk_div(unit, r.row_blocks));
      s.row0 = int(unit - int64_t(s.g) * r.row_blocks) * P.unit_rows;
      s.len = r.len;
      s.queries = r.queries;
      s.kv = r.refused ? 0 : r.len + r.queries;
      s.whole = s.k_lo == 0 && s.k_hi == r.tiles;
      s.refused = r.refused;
      s.first = !started;
      started = true;
      s.t0 = s.row0 / P.group;
      s.hl0 = s.row0 - s.t0 * P.group;
      const bool packed = P.a.q_start != nullptr;
      s.q_base = (packed ? int64_t(r.start) * P.a.q_st : int64_t(b) * P.a.q_sb) + int64_t(s.g) * P.group * P.a.q_sh;
      s.o_base = (packed ? int64_t(r.start) * P.a.o_st : int64_t(b) * P.a.o_sb) + int64_t(s.g) * P.group * P.a.o_sh;
      s.mask_row = packed ? r.start : int64_t(b) * P.a.query_len;
      return true;
    }
    return false;
  }
};

// CTA c's join record, written by one thread with the CTA's first segment (null: it has none):
// if that segment is its unit's second part, what the merge kernel joins; else no rows.
__device__ __forceinline__ void chunk_write_join(const ChunkParams& P, const ChunkStart& start, int c,
                                                 const ChunkSegment* seg) {
  ChunkJoin j{0, 0, 0, 0, 0, 0, 0, 0};
  if (seg != nullptr && seg->k_lo > 0) {
    const int64_t begin = start.begin(c), unit_begin = begin - seg->k_lo - P.unit_cost;
    const int64_t before = start.begin(c - 1);
    if (before <= unit_begin + P.unit_cost) {  // CTA c - 1 holds the unit's first tile
      const int64_t kv = seg->refused ? 1 : int64_t(seg->len) + seg->queries;
      const int64_t unit_end = unit_begin + P.unit_cost + ((kv + P.tile_keys - 1) >> P.tile_shift);
      j.b = seg->b;
      j.g = seg->g;
      j.row0 = seg->row0;
      j.rows = min(seg->queries * P.group - seg->row0, P.unit_rows);
      j.start = int(P.a.q_start != nullptr ? seg->mask_row : 0);
      j.slot0 = (c - 1) * 2 + (before >= unit_begin ? 0 : 1);
      j.parts = 2;
      while (c - 1 + j.parts < P.ctas && start.begin(c - 1 + j.parts) < unit_end) ++j.parts;
    }
  }
  P.ws_join[c] = j;
}

// Row `r` of a unit whose first row is row0: query t and local head hl. row0 / group is the
// same for every row of the unit; r is small, so its division is a 16-bit multiplication
// (group_magic = ceil(2^20 / group), exact for (group - 1) + r < 1024 and group < 1024).
struct ChunkRows {
  int t0, hl0;  // query and local head of row0
  __device__ __forceinline__ ChunkRows(int t, int hl) : t0(t), hl0(hl) {}
  __device__ __forceinline__ void at(const ChunkParams& P, int r, int& t, int& hl) const {
    const int x = hl0 + r;
    const int dt = P.group < 512 ? int((uint32_t(x) * P.group_magic) >> 20) : x / P.group;
    t = t0 + dt;
    hl = x - dt * P.group;
  }
};

// Page table row that request b's KV head g walks.
__device__ __forceinline__ const int32_t* chunk_table(const ChunkParams& P, int b, int g) {
  return P.a.page_table + int64_t(b) * P.a.page_table_stride + int64_t(g) * P.table_head_stride;
}

// Which of the 64 chunk-local nodes node0 .. node0 + 63 query t of the segment's request sees, as
// bits (negative nodes are cached tokens: seen by all; nodes from `queries` on exist for
// nobody). Without a mask the chunk is causal.
__device__ __forceinline__ uint64_t chunk_visible64(const ChunkParams& P, const ChunkSegment& seg, int t, int node0) {
  const int queries = seg.queries;
  if (node0 >= queries || node0 <= -64) return node0 <= -64 ? ~0ull : 0ull;
  const int first = max(node0, 0);
  uint64_t bits = 0;
  if (P.mask == nullptr) {
    const int n = t + 1 - first;  // nodes first .. t
    bits = n <= 0 ? 0ull : (n >= 64 ? ~0ull : (1ull << n) - 1);
  } else {
    const uint32_t* words = reinterpret_cast<const uint32_t*>(P.mask) + (seg.mask_row + t) * P.mask_words;
    const int w = first >> 5, sh = first & 31;
    const uint32_t w0 = w < P.mask_words ? words[w] : 0u;
    const uint32_t w1 = w + 1 < P.mask_words ? words[w + 1] : 0u;
    const uint32_t w2 = w + 2 < P.mask_words ? words[w + 2] : 0u;
    bits = uint64_t(__funnelshift_r(w0, w1, sh)) | (uint64_t(__funnelshift_r(w1, w2, sh)) << 32);
  }
  const int n = queries - first;  // >= 1
  if (n < 64) bits &= (1ull << n) - 1;
  if (node0 < 0) bits = (bits << -node0) | ((1ull << -node0) - 1);  // -63 .. -1
  return bits;
}

// Where a partial of slot `slot` lives: O as [dims / 4][unit_rows] float4 (consecutive rows
// next to each other), (max in log2 units, sum) per row.
__device__ __forceinline__ float4* chunk_partial_o(const ChunkParams& P, int64_t slot) {
  return reinterpret_cast<float4*>(P.ws_o) + slot * (int64_t(P.a.head_dim / 4) * P.unit_rows);
}
__device__ __forceinline__ float2* chunk_partial_ml(const ChunkParams& P, int64_t slot) {
  return reinterpret_cast<float2*>(P.ws_ml) + slot * P.unit_rows;
}

}  // namespace hyt
