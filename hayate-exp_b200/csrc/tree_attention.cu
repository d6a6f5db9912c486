// Chunk attention on tcgen05 tensor cores: trees of drafted tokens, and one-token decode over
// chosen pages, for bf16 / f16 and head sizes 64 .. 128.
//
//   out[row] = sum_j softmax_j(scale * q[row] . k_j) v_j
//
// over the cached keys and the step's own nodes that the row's mask shows. The rows of a
// unit are all heads of one KV group times the request's queries (row t * group + hl), so a
// key is read once for the whole group and a tree of 32 nodes with 4 heads fills the 128
// lanes of an MMA. Work is shared out by chunk_schedule.cuh: 148 CTAs, one per SM, each an
// equal stretch of 128-key tiles.
//
// Two streams x = 0, 1 of S / P / O keep the tensor cores and the softmax warps busy at the
// same time:
//   one row block per unit (kDual false, at most 128 rows): stream x takes the tiles i with
//     i % 2 == x, both with the same Q, and the two online softmaxes are joined at the end;
//   two row blocks (kDual true): stream x is row block x, both see every tile, so a K/V tile
//     brought into shared memory serves 256 rows.
// 640 threads: warps 0-7 softmax of stream 0, 8-15 of stream 1 (in a stream, warps w and
// w + 4 own rows 32 (w % 4) .. and half of the 128 key columns each), warp 16 the TMA
// producer, which also walks the CTA's segments and hands them to the others through a
// shared ring, warp 17 the MMA issuer, warps 18-19 look through V past the cached tokens and,
// once the last S of a segment is done, bring the next one's Q: by TMA (boxes of 32 rows: a
// group's heads x 32 / group tokens), or row by row where q's layout has no such map or the
// group does not divide 32 (64 KB took 9,000 to 12,000 cycles that way, 1,000 by TMA). Per tile, S = Q K^T (shared x shared), P goes back over
// S's columns as 16-bit pairs, O += P V (TMEM x shared). Issue order PV(s), QK(s + 2).
// TMEM (512 columns): S_0/P_0 [0,128), S_1/P_1 [128,256), O_0 [256,384), O_1 [384,512).
// Shared memory: Q 32 KB per row block, 2 K stages, 3 (one row block) or 2 V stages of 32 KB.
// Head sizes below 128 are padded with zeros by TMA's out-of-range fill and the Q stores;
// up to 64, the second 64-dim half is neither loaded nor multiplied.
//
// Masking: scores by selection. V rows of the tiles that reach past the cached tokens are
// looked through (by the Q warps, beside the softmax) before they are multiplied: values that
// are not finite become zeros, and those of drafted nodes are added at the end to the rows
// that see them (0 * inf would be NaN in every row). A tile whose page was refused is not
// multiplied. A visible score that is NaN or +inf makes its row NaN.
//
// P is rounded to the storage type (the MMA's operand type); scores, running maximum and
// sum, and O are fp32. The running maximum may lag by up to 2^8 (O / l is exact all the same).
//
// Bound by HBM up to 128 rows a unit: 64 requests x 16 nodes over 1K to 8K tokens, 32 / 8 heads of
// 128, take 205 us for 1.23 GB with the merge (6.0 TB/s). Above, by the chain of a stream's
// softmax and its 16 MMAs, 3,250 to 3,400 cycles per 256 x 128 tile of which the MMAs are 2,048:
// 4 x 33..64 nodes over 32K tokens 143 us (0.70 PFLOP/s of visible pairs), 8 x 256 nodes over 2K to
// 4K 128 us (0.77). Two row blocks per unit instead of one: a K/V tile is read half as often (the
// first kernel, with one, took 199 us on the latter). A unit's ends cost about 4 tiles: the first
// tile runs on cold instructions, and O goes out as 128 KB of partials.
#include <type_traits>

#include "chunk_schedule.cuh"

namespace hyt {

namespace {

constexpr int kRows = 128;
constexpr int kKeys = 128;
constexpr int kSoftmaxThreads = 512;
constexpr int kProducerWarp = 16, kMmaWarp = 17;
constexpr int kSoftmaxBar = 9;  // named barrier of all softmax warps (1 .. 8: row-quarter pairs)
constexpr int kQWarp = 18, kQThreads = 64;
constexpr int kThreads = 640;  // 5 warps of 96 registers per sub-partition
constexpr int kSegments = 8;   // ring of segments: the producer is at most 5 ahead (V stages + 2)
constexpr int kTileBytes = kRows * 128 * 2;
constexpr int kChunkBytes = kTileBytes / 2;  // [128 rows x 64 elements]
constexpr int kKStages = 2;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kOCol = 256;
constexpr float kRescaleThreshold = 8.0f;  // log2 units
constexpr float kUnseen = 2.0f;  // rescale factor, else at most 1, of a row that saw nothing yet (O and sum are 0)

// measured on 64 requests x 16 nodes, 8 x 256 nodes and 64 requests over 16 chosen pages: 3 tiles take 207, 127
// and 123 us, 4 take 205, 129 and 123, 6 take 206, 130 and 123; one user (8 units of 8 tiles) 13.5, 13.5 and 13.8
constexpr int kUnitCost = 4;

struct Shared {
  uint64_t q_full, q_empty;
  uint64_t v_check, v_ok;  // V of a tile past the cached tokens: to be looked through; done
  uint64_t seg_full[kSegments];
  uint64_t k_full[kKStages], k_empty[kKStages], v_full[3], v_empty[3];
  uint64_t s_full[2], p_full[2];
  uint64_t o_done, drain;
  uint32_t tmem_base;
  int32_t abort;       // a bounded wait gave up: later waits return at once
  int32_t fix[2];      // a drafted node's V is not finite, per segment parity
  int32_t refused[8];  // per tile (ring): page refused, nothing of the tile is visible
  ChunkSegment seg[kSegments];  // segment i in entry i % kSegments; no tiles: the end
  float m[2][kRows];         // running maxima of the streams (joined at the end)
  float sum[2][2][kRows];    // [stream][column half][row]
  float max[2][2][2][kRows]; // [stream][parity][column half][row]
};

template <bool kDual>
struct Layout {
  static constexpr int kVStages = kDual ? 2 : 3;
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + (kDual ? 2 : 1) * kTileBytes;
  static constexpr int kV = kK + kKStages * kTileBytes;
  static constexpr int kShared = kV + kVStages * kTileBytes;
  static constexpr int kBytes = kShared + int(sizeof(Shared)) + 1024;
};

// Byte offset of 16-byte chunk `chunk` of row `r` in a [128 x 128] tile stored as two
// 128B-swizzled [128 x 64] chunks.
__device__ __forceinline__ uint32_t sw128_offset(int r, int chunk) {
  return uint32_t((chunk >> 3) * kChunkBytes + r * 128 + (((chunk & 7) ^ (r & 7)) << 4));
}

// P = 2^(s * scale_log2 - m) of 64 scores, written to TMEM as packed 16-bit pairs; returns
// their sum. 7 of 8 exponentials on MUFU, 1 of 8 on the FMA pipe, where a NaN would get lost: a score
// there that is NaN or +inf makes m, and with it the row, NaN (elsewhere s - m is NaN already).
template <typename T>
__device__ __forceinline__ float exp_tile(const float (&s)[64], uint64_t scale2, float m, uint32_t p_addr) {
  float top = 0.f;
#pragma unroll
  for (int c = 7; c < 64; c += 16) top = fmax3_nan(top, s[c], s[c + 8]);
  m = fmaf(top, 0.f, m);
  const uint64_t neg_m2 = f2_pack(-m, -m);
  uint64_t sum2a = f2_pack(0.f, 0.f), sum2b = sum2a;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t packed[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int k = c * 32 + 2 * i;
      const uint64_t x2 = f2_fma(f2_pack(s[k], s[k + 1]), scale2, neg_m2);
      float a, b;
      f2_unpack(x2, a, b);
      const float pa = ex2(a);
      const float pb = (i & 3) == 3 ? ex2_poly(b) : ex2(b);
      if (i & 1) sum2b = f2_add(sum2b, f2_pack(pa, pb));
      else sum2a = f2_add(sum2a, f2_pack(pa, pb));
      packed[i] = Elem<T>::pack2(pa, pb);
    }
    tmem_st16(p_addr + c * 16, packed);
  }
  float sa0, sa1, sb0, sb1;
  f2_unpack(sum2a, sa0, sa1);
  f2_unpack(sum2b, sb0, sb1);
  return (sa0 + sb0) + (sa1 + sb1);
}

template <int kStages>
struct Ring {
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++stage == kStages) stage = 0, phase ^= 1u;
  }
};

struct TreeKernelParams {
  ChunkParams c;
  int32_t q_vec, o_vec;  // q / out rows start on 16-byte boundaries
  int32_t q_tma;         // q_map holds q as (dim, head, token), boxes of 64 dims x a group's heads x 32 / group tokens
};

// The rare paths are kept out of line: the code between two segments is fetched cold (the
// softmax loop has pushed it out of the instruction cache), so its size is time.

__device__ __noinline__ void store_unaligned16(void* at, uint4 w) {
  uint16_t* e = static_cast<uint16_t*>(at);
  e[0] = uint16_t(w.x), e[1] = uint16_t(w.x >> 16), e[2] = uint16_t(w.y), e[3] = uint16_t(w.y >> 16);
  e[4] = uint16_t(w.z), e[5] = uint16_t(w.z >> 16), e[6] = uint16_t(w.w), e[7] = uint16_t(w.w >> 16);
}

// One half of a 4 x 4 exchange of pieces: lanes that differ in bit kBit swap w[v] (v with the bit) of
// the lane without it for w[v - kBit] of the lane with it.
template <int kBit>
__device__ __forceinline__ void swap_pieces(uint4 (&w)[4], int lane) {
  const bool upper = (lane & kBit) != 0;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    if (!(v & kBit)) continue;
    uint32_t* lo = reinterpret_cast<uint32_t*>(&w[v - kBit]);
    uint32_t* hi = reinterpret_cast<uint32_t*>(&w[v]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t got = __shfl_xor_sync(0xffffffffu, upper ? lo[e] : hi[e], kBit);
      if (upper) lo[e] = got;
      else hi[e] = got;
    }
  }
}

// acc + 0 * x for a pair of values: +-0 where both are finite so far
template <typename T>
__device__ __forceinline__ uint32_t times_zero(uint32_t x, uint32_t acc) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value)
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0u), "r"(acc));
  else
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0u), "r"(acc));
  return r;
}

// Zeros for the values that are not finite in 16-byte chunk `chunk` of rows first, first + step ..
// of a tile; whether one is in a row below `rows`.
template <typename T>
__device__ __noinline__ bool zero_not_finite(uint8_t* tile, int first, int step, int chunk, int rows) {
  constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  bool found = false;
  for (int r = first; r < kKeys; r += step) {
    uint32_t* at = reinterpret_cast<uint32_t*>(tile + sw128_offset(r, chunk));
    for (int e = 0; e < 4; ++e) {
      const uint32_t was = at[e];
      uint32_t w = was;
      if ((w & kExp) == kExp) w &= 0xFFFF0000u;
      if ((w & (kExp << 16)) == (kExp << 16)) w &= 0x0000FFFFu;
      if (w == was) continue;
      at[e] = w;
      found |= r < rows;
    }
  }
  return found;
}

// The CTA's n-th tile: nothing of it is visible, its stages hold something else.
__device__ __forceinline__ bool tile_refused(const Shared* sh, int n) {
  return *reinterpret_cast<const volatile int32_t*>(&sh->refused[n & 7]) != 0;
}
// First tile of the segment that reaches past the cached tokens: from there on V is checked.
__device__ __forceinline__ int first_checked(const ChunkSegment& seg) {
  return seg.refused ? seg.k_hi : max(seg.k_lo, seg.len / kKeys);
}

// Adds V of the nodes query t sees that were left out because they are not finite to columns
// [col, col + n) of its row, as just written: to `out`, or to its partial.
template <typename T>
__device__ __noinline__ void add_not_finite(const ChunkParams& P, const ChunkSegment& seg, int t, int col, int n,
                                            T* out, float* partial) {
  const AttentionParams& p = P.a;
  const int lo = max(seg.k_lo * kKeys, seg.len), hi = min(seg.k_hi * kKeys, seg.kv);
  const int32_t* table = chunk_table(P, seg.b, seg.g);
  for (int pos = lo; pos < hi; ++pos) {
    if (!(chunk_visible64(P, seg, t, pos - seg.len) & 1)) continue;
    const int32_t page = table[pos >> p.page_shift];
    if (page < 0 || page >= p.num_pages) continue;
    const int64_t vrow = (int64_t(p.layer) * p.num_kv_heads + seg.g) * p.capacity +
                         (int64_t(page) << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
    const T* v = static_cast<const T*>(p.v_pool) + vrow * p.head_dim + col;
    for (int e = 0; e < n; ++e) {
      const float x = Elem<T>::to_float(v[e]);
      if (isfinite(x)) continue;
      if (seg.whole) {
        out[e] = Elem<T>::from_float(Elem<T>::to_float(out[e]) + x);
      } else {
        float* at = partial + int64_t((col + e) / 4) * P.unit_rows * 4 + (e & 3);
        *at += x;
      }
    }
  }
}

// kChunks: 64-dim halves of a head (1: head_dim 64, 2: up to 128).
template <typename T, bool kDual, int kChunks>
__global__ void __maxnreg__(96)
    tree_attention_kernel(const __grid_constant__ CUtensorMap k_map,
                          const __grid_constant__ CUtensorMap v_map,
                          const __grid_constant__ CUtensorMap q_map,
                          const __grid_constant__ TreeKernelParams kp) {
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  using L = Layout<kDual>;
  constexpr int kVStages = L::kVStages;
  constexpr uint32_t kLoadBytes = kChunks * kChunkBytes;
  const ChunkParams& P = kp.c;
  const AttentionParams& p = P.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Shared* sh = reinterpret_cast<Shared*>(smem + L::kShared);
  int32_t* err = p.error_word;
  volatile int* abort = &sh->abort;

  if (threadIdx.x == kMmaWarp * 32) {
    sh->abort = 0;
    sh->fix[0] = sh->fix[1] = 0;
    mbar_init(&sh->q_full, kp.q_tma ? 1 : kQThreads);
    mbar_init(&sh->q_empty, 1);
    mbar_init(&sh->v_check, 1);
    mbar_init(&sh->v_ok, kQThreads);
    for (int s = 0; s < kSegments; ++s) mbar_init(&sh->seg_full[s], 1);
    for (int s = 0; s < kKStages; ++s) mbar_init(&sh->k_full[s], 1), mbar_init(&sh->k_empty[s], 1);
    for (int s = 0; s < kVStages; ++s) mbar_init(&sh->v_full[s], 1), mbar_init(&sh->v_empty[s], 1);
    for (int x = 0; x < 2; ++x) mbar_init(&sh->s_full[x], 1), mbar_init(&sh->p_full[x], kSoftmaxThreads / 2);
    mbar_init(&sh->o_done, 1);
    mbar_init(&sh->drain, 1);
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  ChunkStart start;  // of the producer warp alone: the others follow its segments
  ChunkRequest first_request;
  if (warp == kProducerWarp) {
    if (lane == 0) {
      tma_prefetch_desc(&k_map);
      tma_prefetch_desc(&v_map);
    }
    start = chunk_find_start_warp(P, blockIdx.x, P.ctas, first_request);
  } else {
    wait_for_primary();
  }
  if (warp == 0) {
    tmem_alloc(&sh->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  const uint32_t smem_base = smem_u32(smem);
  // segment i of the CTA, once the producer has published it; null past the last (or once a
  // wait gave up: then not for all threads alike, so those that meet at barriers or in warp
  // operations vote before they go on)
  auto segment = [&](int i) -> const ChunkSegment* {
    if (!mbar_wait(&sh->seg_full[i % kSegments], (i / kSegments) & 1, err, abort)) return nullptr;
    const ChunkSegment* seg = &sh->seg[i % kSegments];
    return seg->k_hi > seg->k_lo ? seg : nullptr;
  };
  launch_dependents();  // the merge kernel may start up; it waits for this grid's results

  if (warp == kProducerWarp) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      ChunkWalk walk(P, start, blockIdx.x, first_request);
      // an earlier CTA's wait gave up: load nothing, every tile counts as refused
      const bool dead = err != nullptr && (*reinterpret_cast<volatile int32_t*>(err) & HYT_DEVERR_WAIT_TIMEOUT);
      const int page_mask = (1 << p.page_shift) - 1;
      int n = 0, k_loads = 0, v_loads = 0;  // tiles so far, those whose K and V stages were filled
      bool gave_up = false;  // a wait of the CTA ran out: nothing more is published or loaded
      auto pool_row = [&](const int32_t* table, int tile) {
        const int tok = tile * kKeys;
        const int32_t page = table[tok >> p.page_shift];
        return page < 0 || page >= p.num_pages ? -1 : (page << p.page_shift) + (tok & page_mask);
      };
      for (int i = 0; !gave_up; ++i) {
        ChunkSegment seg;
        seg.k_lo = seg.k_hi = 0;
        const bool any = walk.next(P, seg);
        sh->seg[i % kSegments] = seg;
        mbar_arrive(&sh->seg_full[i % kSegments]);
        if (!any) {
          if (i == 0) chunk_write_join(P, start, blockIdx.x, nullptr);
          break;
        }
        const int32_t* table = chunk_table(P, seg.b, seg.g);
        const int plane = p.layer * p.num_kv_heads + seg.g;
        for (int tile = seg.k_lo; tile < seg.k_hi; ++tile, ++n) {
          int row = -1;
          if (!seg.refused && !dead) {
            row = pool_row(table, tile);
            if (row < 0) flag_error(err, HYT_DEVERR_PAGE_RANGE);
          }
          const int ks = n % kKStages, vs = n % kVStages;
          if (n >= kKStages && (!mbar_wait(&sh->k_empty[ks], (n / kKStages - 1) & 1, err, abort) || *abort)) {
            gave_up = true;
            break;
          }
          sh->refused[n & 7] = row < 0;
          if (row >= 0) {
            uint8_t* dst = smem + L::kK + ks * kTileBytes;
            mbar_arrive_expect_tx(&sh->k_full[ks], kLoadBytes);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) tma_load_3d(dst + c * kChunkBytes, &k_map, &sh->k_full[ks], c * 64, row, plane);
          } else {
            mbar_arrive(&sh->k_full[ks]);
          }
          ++k_loads;
          if (n >= kVStages && (!mbar_wait(&sh->v_empty[vs], (n / kVStages - 1) & 1, err, abort) || *abort)) {
            gave_up = true;
            break;
          }
          if (row >= 0) {
            uint8_t* dst = smem + L::kV + vs * kTileBytes;
            mbar_arrive_expect_tx(&sh->v_full[vs], kLoadBytes);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) tma_load_3d(dst + c * kChunkBytes, &v_map, &sh->v_full[vs], c * 64, row, plane);
          } else {
            mbar_arrive(&sh->v_full[vs]);
          }
          ++v_loads;
          if (n == 0) chunk_write_join(P, start, blockIdx.x, &seg);  // beside the first loads
        }
      }
      // nothing in flight when the CTA exits
      for (int i = max(0, k_loads - kKStages); i < k_loads; ++i) mbar_drain(&sh->k_full[i % kKStages], (i / kKStages) & 1);
      for (int i = max(0, v_loads - kVStages); i < v_loads; ++i) mbar_drain(&sh->v_full[i % kVStages], (i / kVStages) & 1);
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------ MMA issuer
    // The whole warp walks and waits; each group of MMAs and its commits is issued by the
    // lane elect.sync picks.
    constexpr uint32_t idesc_qk = umma_idesc_f16(kBf16, 128, 128, false, false);
    constexpr uint32_t idesc_pv = umma_idesc_f16(kBf16, 128, kChunks * 64, false, true);
    const uint64_t q_desc = umma_desc_sw128(smem_base + L::kQ, 16);
    const uint32_t hi = uint32_t(q_desc >> 32);
    const uint32_t q_lo = uint32_t(q_desc);
    const uint32_t k_lo = uint32_t(umma_desc_sw128(smem_base + L::kK, 16));
    const uint32_t v_lo = uint32_t(umma_desc_sw128(smem_base + L::kV, kChunkBytes));
    constexpr uint32_t kStep = kTileBytes >> 4;  // descriptor units from stage to stage
    // run f on the elected lane (checked to be lane 0: every commit covers what came before)
    auto issue = [&](auto&& f) {
      if (elect_one()) {
        if (__activemask() == (1u << lane) && lane == 0) {
          tc_fence_after();
          f();
        } else {
          flag_error(err, HYT_DEVERR_ISSUE_LANE);
        }
      }
      __syncwarp();
    };
    auto qk = [&](int x, int q_block, int stage) {
      const uint32_t a0 = q_lo + q_block * kStep, b0 = k_lo + stage * kStep;
#pragma unroll
      for (int kk = 0; kk < 4 * kChunks; ++kk) {
        const uint32_t off = uint32_t(((kk >> 2) * kChunkBytes + (kk & 3) * 32) >> 4);
        umma_f16_ss_lh(tmem + x * 128, a0 + off, hi, b0 + off, hi, idesc_qk, kk > 0 ? 1u : 0u);
      }
      umma_commit(&sh->s_full[x]);
    };
    auto pv = [&](int x, int stage, bool accumulate) {
      const uint32_t b0 = v_lo + stage * kStep;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)
        umma_f16_ts_lh(tmem + kOCol + x * 128, tmem + x * 128 + kk * 8, b0 + uint32_t((kk * 2048) >> 4), hi, idesc_pv,
                       (kk > 0 || accumulate) ? 1u : 0u);
    };
    Ring<kKStages> kr;  // next K tile to multiply, next V tile
    Ring<kVStages> vr;
    uint32_t p_phase[2] = {0u, 0u}, q_phase = 0u, ok_phase = 0u;
    int n0 = 0;  // tiles before this segment
    // P and V of tile i of the segment (stream x): V in shared memory and, past the cached tokens,
    // looked through by the checkers, who start as soon as it is there
    bool told = false;  // the checkers know of the next tile's V already
    auto wait_pv = [&](const ChunkSegment& seg, int x, int i) {
      mbar_wait(&sh->v_full[vr.stage], vr.phase, err, abort);
      const bool check = seg.k_lo + i >= first_checked(seg) && (!kDual || x == 0);
      if (check && !told && lane == 0) mbar_arrive(&sh->v_check);
      if (!kDual || x == 0) told = false;
      mbar_wait(&sh->p_full[x], p_phase[x], err, abort);
      p_phase[x] ^= 1u;
      if (check) {
        mbar_wait(&sh->v_ok, ok_phase, err, abort);
        ok_phase ^= 1u;
      }
    };
    // after tile i was issued (vr: the next one): if the next one's V, to be checked, is there, say so
    // now, so that the check runs beside the softmax
    auto tell_ahead = [&](const ChunkSegment& seg, int i, int n) {
      if (i + 1 >= n || seg.k_lo + i + 1 < first_checked(seg)) return;
      const bool there = __shfl_sync(0xffffffffu, mbar_try_wait(&sh->v_full[vr.stage], vr.phase) ? 1 : 0, 0) != 0;
      if (there && lane == 0) mbar_arrive(&sh->v_check);
      told = there;
    };
    for (int i = 0;; ++i) {
      const ChunkSegment* found = segment(i);
      if (!__all_sync(0xffffffffu, found != nullptr)) break;
      const ChunkSegment& seg = *found;
      const int n = seg.k_hi - seg.k_lo;
      uint32_t begun = 0u;  // streams whose O holds something of this segment
      mbar_wait(&sh->q_full, q_phase, err, abort);
      q_phase ^= 1u;
      if constexpr (!kDual) {
        for (int s = 0; s < min(n, 2); ++s, kr.next()) {
          mbar_wait(&sh->k_full[kr.stage], kr.phase, err, abort);
          issue([&] {
            qk(s, 0, kr.stage);
            umma_commit(&sh->k_empty[kr.stage]);
            if (s == n - 1) umma_commit(&sh->q_empty);  // no further product reads this Q
          });
        }
        for (int s = 0; s < n; ++s, vr.next(), tell_ahead(seg, s - 1, n)) {
          const int x = s & 1;
          const bool more = s + 2 < n;
          wait_pv(seg, x, s);
          const bool refused = tile_refused(sh, n0 + s);
          issue([&] {
            if (!refused) pv(x, vr.stage, (begun >> x) & 1u);
            umma_commit(&sh->v_empty[vr.stage]);
            if (!more && s == n - 1) umma_commit(&sh->o_done);
          });
          if (more) {
            mbar_wait(&sh->k_full[kr.stage], kr.phase, err, abort);
            issue([&] {
              qk(x, 0, kr.stage);
              umma_commit(&sh->k_empty[kr.stage]);
              if (s + 2 == n - 1) umma_commit(&sh->q_empty);
            });
            kr.next();
          }
          if (!refused) begun |= 1u << x;
        }
      } else {
        mbar_wait(&sh->k_full[kr.stage], kr.phase, err, abort);
        issue([&] {
          qk(0, 0, kr.stage);
          qk(1, 1, kr.stage);
          umma_commit(&sh->k_empty[kr.stage]);
          if (n == 1) umma_commit(&sh->q_empty);  // no further product reads this Q
        });
        kr.next();
        for (int j = 0; j < n; ++j, vr.next(), tell_ahead(seg, j - 1, n)) {
          const bool more = j + 1 < n;
          wait_pv(seg, 0, j);
          const bool refused = tile_refused(sh, n0 + j);
          if (more) mbar_wait(&sh->k_full[kr.stage], kr.phase, err, abort);
          issue([&] {
            if (!refused) pv(0, vr.stage, begun != 0u);
            if (more) qk(0, 0, kr.stage);
          });
          wait_pv(seg, 1, j);
          issue([&] {
            if (!refused) pv(1, vr.stage, begun != 0u);
            umma_commit(&sh->v_empty[vr.stage]);
            if (more) {
              qk(1, 1, kr.stage);
              umma_commit(&sh->k_empty[kr.stage]);
              if (j + 2 == n) umma_commit(&sh->q_empty);
            } else {
              umma_commit(&sh->o_done);
            }
          });
          if (more) kr.next();
          if (!refused) begun = 1u;
        }
      }
      n0 += n;
    }
    issue([&] { umma_commit(&sh->drain); });  // every MMA done before TMEM is released
    mbar_drain(&sh->drain, 0);
  } else if (warp >= kQWarp) {
    // ------------------------------------------------------------ Q loaders, V checkers
    const int tid = int(threadIdx.x) - kQWarp * 32, D = p.head_dim;
    constexpr int kRowChunks = kChunks * 8;            // 16-byte chunks of a padded row
    constexpr int kStepRows = kQThreads / kRowChunks;  // rows the two warps load at a time
    const int c = tid % kRowChunks;
    const int step_t = kStepRows / P.group, step_h = kStepRows - step_t * P.group;
    const int64_t step_off = step_t * p.q_st + step_h * p.q_sh, wrap_off = p.q_st - P.group * p.q_sh;
    // rows of the 32-row quarters that have any (the others' lanes are never looked at). By TMA,
    // rows past the request's are its neighbours' on the token axis: no result comes of them
    auto load_q = [&](const ChunkSegment& seg) {
      const int rows = seg.queries * P.group - seg.row0;
      const int upto = min((kDual ? 2 : 1) * kRows, (rows + 31) & ~31);
      if (kp.q_tma) {
        if (tid != 0) return;
        constexpr int kPartBytes = 32 * 128;  // 32 rows of 64 dims
        int token = int(seg.mask_row) + seg.t0;
        mbar_arrive_expect_tx(&sh->q_full, uint32_t(upto / 32 * kChunks * kPartBytes));
        for (int qr = 0; qr < upto; qr += 32, token += 32 / P.group) {
          uint8_t* dst = smem + L::kQ + (qr >> 7) * kTileBytes + ((qr & (kRows - 1)) >> 5) * kPartBytes;
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
            tma_load_3d(dst + c * kChunkBytes, &q_map, &sh->q_full, c * 64, seg.g * P.group, token);
        }
        return;
      }
      int qr = tid / kRowChunks, t, hl;
      ChunkRows(seg.t0, seg.hl0).at(P, qr, t, hl);
      const T* src = static_cast<const T*>(p.q) + seg.q_base + t * p.q_st + hl * p.q_sh + c * 8;
#pragma unroll 4
      for (; qr < upto; qr += kStepRows) {
        const bool there = qr < rows && c * 8 < D;
        uint8_t* dst = smem + L::kQ + (qr >> 7) * kTileBytes + sw128_offset(qr & (kRows - 1), c);
        if (kp.q_vec) {
          cp_async16(dst, there ? src : static_cast<const T*>(p.q), there ? 16 : 0);  // 0: zeros
        } else {
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (there) {
            const uint16_t* e = reinterpret_cast<const uint16_t*>(src);
            v.x = e[0] | (uint32_t(e[1]) << 16);
            v.y = e[2] | (uint32_t(e[3]) << 16);
            v.z = e[4] | (uint32_t(e[5]) << 16);
            v.w = e[6] | (uint32_t(e[7]) << 16);
          }
          *reinterpret_cast<uint4*>(dst) = v;
        }
        src += step_off;
        hl += step_h;
        if (hl >= P.group) hl -= P.group, src += wrap_off;
      }
    };
    auto q_ready = [&]() {
      if (kp.q_tma) return;
      cp_async_wait_all();
      fence_proxy_async_smem();
      mbar_arrive(&sh->q_full);
    };
    // V of the CTA's n-th tile: values that are not finite become zeros among the rows past the
    // cached tokens. A finite value times zero is zero, another is NaN: one FMA per pair of values
    uint32_t check_phase = 0u;
    auto check_v = [&](const ChunkSegment& seg, int i, int tile, int n) {
      const int stage = n % kVStages;
      mbar_wait(&sh->v_check, check_phase, err, abort);
      check_phase ^= 1u;
      mbar_wait(&sh->v_full[stage], (n / kVStages) & 1, err, abort);  // done; orders TMA's writes before the reads
      const int k0 = tile * kKeys, v0 = max(seg.len - k0, 0) + tid / kRowChunks;
      uint8_t* at0 = smem + L::kV + stage * kTileBytes;
      uint32_t zero[4] = {0u, 0u, 0u, 0u};
#pragma unroll 8
      for (int vr = v0; vr < kKeys; vr += kStepRows) {
        const uint4 v = *reinterpret_cast<const uint4*>(at0 + sw128_offset(vr, c));
        zero[0] = times_zero<T>(v.x, zero[0]), zero[1] = times_zero<T>(v.y, zero[1]);
        zero[2] = times_zero<T>(v.z, zero[2]), zero[3] = times_zero<T>(v.w, zero[3]);
      }
      if (((zero[0] | zero[1]) | (zero[2] | zero[3])) & 0x7FFF7FFFu) {
        if (zero_not_finite<T>(at0, v0, kStepRows, c, seg.kv - k0)) *reinterpret_cast<volatile int32_t*>(&sh->fix[i & 1]) = 1;
      }
      fence_proxy_async_smem();
      mbar_arrive(&sh->v_ok);
    };
    // Per segment: the tiles to check; then, once the segment's last S is done, the next segment's Q
    // (Q before the last tile's check held up that tile's PV by 9,000 cycles)
    if (kp.q_tma && tid == 0) tma_prefetch_desc(&q_map);
    const ChunkSegment* now = segment(0);
    if (now != nullptr) {
      load_q(*now);
      q_ready();
    }
    int loads = now != nullptr ? 1 : 0;
    for (int i = 0, n0 = 0; now != nullptr; ++i) {
      const ChunkSegment seg = *now;
      const int n = seg.k_hi - seg.k_lo;
      const int first = first_checked(seg);
      for (int tile = first; tile < seg.k_hi; ++tile) check_v(seg, i, tile, n0 + tile - seg.k_lo);
      if (!mbar_wait(&sh->q_empty, i & 1, err, abort)) break;  // Q may still be read
      now = segment(i + 1);
      if (now != nullptr) {
        load_q(*now);
        q_ready();
        ++loads;
      }
      n0 += n;
    }
    if (kp.q_tma && tid == 0 && loads > 0) mbar_drain(&sh->q_full, (loads - 1) & 1);  // nothing in flight when the CTA exits
  } else {
    // ------------------------------------------------------------ softmax warps
    const int x = warp >> 3, half = (warp >> 2) & 1, quarter = warp & 3;
    const int r = quarter * 32 + lane;  // row of the block == TMEM lane
    const int block = kDual ? x : 0;    // row block this stream works on
    const uint32_t lane_addr = tmem + (uint32_t(quarter * 32) << 16);
    const int pair_bar = 1 + x * 4 + quarter;
    const float scale_log2 = p.scale * kLog2e;
    const uint64_t scale2 = f2_pack(scale_log2, scale_log2);
    const uint32_t s_addr = lane_addr + x * 128 + half * 64;
    const uint32_t p_addr = lane_addr + x * 128 + half * 32;
    const uint32_t o_addr = lane_addr + kOCol + x * 128 + half * (kChunks * 32);
    const int D = p.head_dim;
    int n0 = 0, segs = 0;
    uint32_t sc = 0;  // S tiles taken so far by this stream

    for (;;) {
      const ChunkSegment* found = segment(segs);
      // All softmax warps go on, or none: they meet at barriers below. O, the sums and `fix` of the
      // segment before have been read by everyone (the entry's next user is one segment on,
      // after another of these barriers)
      if (!named_bar_all(kSoftmaxBar, kSoftmaxThreads, found != nullptr)) break;
      if (threadIdx.x == 0 && segs > 0) sh->fix[(segs - 1) & 1] = 0;
      const ChunkSegment& seg = *found;
      const int n = seg.k_hi - seg.k_lo;
      const int rows_left = seg.queries * P.group - seg.row0;  // may exceed the unit's rows
      const int my_rows = rows_left - block * kRows;
      const bool active = quarter * 32 < my_rows;  // warp-uniform: some of the warp's rows exist
      auto query = [&](int& t, int& hl) {  // of this row
        ChunkRows(seg.t0, seg.hl0).at(P, block * kRows + r, t, hl);
        t = min(t, seg.queries - 1);
      };
      if (half == 0 && active && P.mask != nullptr && (seg.k_hi > seg.len / kKeys)) {  // the row's mask, needed last
        int t, hl;
        query(t, hl);
        asm volatile("prefetch.global.L1 [%0];" ::"l"(P.mask + (seg.mask_row + t) * P.mask_words) : "memory");
      }
      float m_run = -INFINITY, l_run = 0.f;
      // of the CTA's tiles: the segment's end and the first that reaches past the cached tokens
      const int end = n0 + n, tail = n0 + max(seg.len / kKeys - seg.k_lo, 0);
      for (int i = n0 + (kDual ? 0 : x); i < end; i += kDual ? 1 : 2) {
        if constexpr (kDual) sc = uint32_t(i);
        mbar_wait(&sh->s_full[x], sc & 1, err, abort);
        tc_fence_after();
        __syncwarp();
        if (active) {
          float s[64];
          bool none, masked;
          {
            uint32_t raw[2][32];
            tmem_ld32(s_addr, raw[0]);
            tmem_ld32(s_addr + 32, raw[1]);
            none = tile_refused(sh, i);  // beside the loads
            masked = none || i >= tail;
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int e = 0; e < 32; ++e) s[c * 32 + e] = __uint_as_float(raw[c][e]);
          }
          if (masked) {
            int t, hl;
            query(t, hl);
            const uint64_t seen = none || r >= my_rows
                                      ? 0ull
                                      : chunk_visible64(P, seg, t, (seg.k_hi - (end - i)) * kKeys + half * 64 - seg.len);
            const uint32_t seen_lo = uint32_t(seen), seen_hi = uint32_t(seen >> 32);
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              if (!((seen_lo >> c) & 1u)) s[c] = -INFINITY;
              if (!((seen_hi >> c) & 1u)) s[32 + c] = -INFINITY;
            }
          }
          float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
          for (int c = 0; c < 64; c += 4) {
            mx0 = fmax3(mx0, s[c], s[c + 1]);
            mx1 = fmax3(mx1, s[c + 2], s[c + 3]);
          }
          float(*slot)[kRows] = sh->max[x][sc & 1];
          slot[half][r] = fmaxf(mx0, mx1);
          named_bar_sync(pair_bar, 64);
          const float m_tile = fmaxf(slot[0][r], slot[1][r]) * scale_log2;
          const float m_new = fmaxf(m_run, m_tile);
          const bool moves = __any_sync(0xffffffffu, m_new > m_run + kRescaleThreshold);
          float alpha = 1.f;
          if (moves) {
            alpha = m_run == -INFINITY ? kUnseen : ex2(m_run - m_new);
            m_run = m_new;
          }
          const float tile_sum = exp_tile<T>(s, scale2, m_run == -INFINITY ? 0.f : m_run, p_addr);
          l_run = l_run * alpha + tile_sum;
          // If a row saw a tile before, O_x holds products, and is stable: its last PV completed before
          // S_x did. l_run cannot tell: it is the sum over this half's keys, O's dims hold both halves'
          if (moves && __any_sync(0xffffffffu, alpha != kUnseen)) {
            if (alpha == kUnseen) alpha = 0.f;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
              uint32_t o[32];
              tmem_ld32(o_addr + c * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st32(o_addr + c * 32, o);
            }
          }
          tmem_wait_st();
        }
        tc_fence_before();
        mbar_arrive(&sh->p_full[x]);
        if constexpr (!kDual) ++sc;
      }

      // ---- epilogue
      sh->sum[x][half][r] = l_run;
      if (half == 0) sh->m[x][r] = m_run;
      mbar_wait(&sh->o_done, segs & 1, err, abort);
      tc_fence_after();
      named_bar_sync(kSoftmaxBar, kSoftmaxThreads);
      __syncwarp();
      const bool fix = *reinterpret_cast<volatile int32_t*>(&sh->fix[segs & 1]) != 0;
      // one row block: the streams are joined, a quarter of the columns per warp; two: each
      // stream has its own rows, half of the columns per warp
      constexpr int kGroups = kDual ? kChunks : 1;  // 32-column groups per warp
      const int col0 = kDual ? half * (kChunks * 32) : (x * 2 + half) * 32;
      if (active && col0 < kChunks * 64) {
        float f0 = 1.f, f1 = 0.f, m = m_run, l;
        bool use0 = true, use1 = false;
        uint32_t from = lane_addr + kOCol + (kDual ? x * 128 : 0);
        if constexpr (kDual) {
          l = sh->sum[x][0][r] + sh->sum[x][1][r];
          use0 = l != 0.f;  // nothing seen: O may hold anything
        } else {
          const float m0 = sh->m[0][r], m1 = sh->m[1][r];
          const float l0 = sh->sum[0][0][r] + sh->sum[0][1][r], l1 = sh->sum[1][0][r] + sh->sum[1][1][r];
          m = fmaxf(m0, m1);
          const float m_use = m == -INFINITY ? 0.f : m;
          use0 = l0 != 0.f;
          use1 = l1 != 0.f;  // also false where stream 1 had no tile
          f0 = use0 ? ex2(m0 - m_use) : 0.f;
          f1 = use1 ? ex2(m1 - m_use) : 0.f;
          l = l0 * f0 + l1 * f1;
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const bool mine = r < my_rows;
        int t, hl;
        query(t, hl);
        const int unit_row = block * kRows + r;
        T* out = static_cast<T*>(p.out) +
                 (mine ? seg.o_base + t * p.o_st + hl * p.o_sh : int64_t(0));
        const int64_t slot = int64_t(blockIdx.x) * 2 + (seg.first ? 0 : 1);
#pragma unroll 1
        for (int c = 0; c < kGroups; ++c) {
          const int col = col0 + c * 32;
          float f[32];
          {
            uint32_t o[32];
            tmem_ld32(from + col, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) f[e] = use0 ? __uint_as_float(o[e]) * f0 : 0.f;
          }
          if constexpr (!kDual) {
            if (n > 1) {  // warp-uniform
              uint32_t o[32];
              tmem_ld32(from + 128 + col, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (use1) f[e] = fmaf(__uint_as_float(o[e]), f1, f[e]);
            }
          }
          if (kDual && seg.whole && kp.o_vec) {
            // four lanes exchange 16-byte pieces of their rows, so that a store writes 64 bytes in a
            // row of 8 rows each, not 16 of 32 (8 x 256 nodes: 126.5 -> 124 us; with one row block,
            // of which often few rows exist, 64 x 16 nodes 202 -> 203, so those store directly)
            uint4 w[4];
#pragma unroll
            for (int v = 0; v < 4; ++v)
              w[v] = make_uint4(Elem<T>::pack2(f[8 * v] * inv, f[8 * v + 1] * inv),
                                Elem<T>::pack2(f[8 * v + 2] * inv, f[8 * v + 3] * inv),
                                Elem<T>::pack2(f[8 * v + 4] * inv, f[8 * v + 5] * inv),
                                Elem<T>::pack2(f[8 * v + 6] * inv, f[8 * v + 7] * inv));
            swap_pieces<2>(w, lane);
            swap_pieces<1>(w, lane);  // w[k]: piece lane % 4 of row k of the four
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int owner = (lane & ~3) | k;
              T* row = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(out), owner));
              const int at = col + (lane & 3) * 8;
              if (quarter * 32 + owner < my_rows && at < D) *reinterpret_cast<uint4*>(row + at) = w[k];
            }
            __syncwarp();  // before values that are not finite are added
          } else if (mine) {
            if (seg.whole) {
#pragma unroll
              for (int v = 0; v < 4; ++v) {
                if (col + v * 8 >= D) break;
                const uint4 w = make_uint4(Elem<T>::pack2(f[8 * v] * inv, f[8 * v + 1] * inv),
                                           Elem<T>::pack2(f[8 * v + 2] * inv, f[8 * v + 3] * inv),
                                           Elem<T>::pack2(f[8 * v + 4] * inv, f[8 * v + 5] * inv),
                                           Elem<T>::pack2(f[8 * v + 6] * inv, f[8 * v + 7] * inv));
                if (!kDual && kp.o_vec) *reinterpret_cast<uint4*>(out + col + v * 8) = w;
                else store_unaligned16(out + col + v * 8, w);
              }
            } else {
              float4* wo = chunk_partial_o(P, slot);
#pragma unroll
              for (int v = 0; v < 8; ++v)
                if (col + v * 4 < D)
                  wo[int64_t(col / 4 + v) * P.unit_rows + unit_row] =
                      make_float4(f[4 * v], f[4 * v + 1], f[4 * v + 2], f[4 * v + 3]);
              if (col == 0) chunk_partial_ml(P, slot)[unit_row] = make_float2(m, l);
            }
          }
          if (fix && mine)
            add_not_finite<T>(P, seg, t, col, min(32, D - col), out + col,
                              reinterpret_cast<float*>(chunk_partial_o(P, slot)) + unit_row * 4);
          __syncwarp();
        }
      }
      tc_fence_before();
      n0 = end;
      ++segs;
    }
  }

  // ---- release TMEM once every warp is done with it
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <typename T, bool kDual, int kChunks>
cudaError_t launch_tree(const TreeKernelParams& kp, const CUtensorMap& k_map, const CUtensorMap& v_map,
                        const CUtensorMap& q_map, cudaStream_t stream) {
  auto kernel = tree_attention_kernel<T, kDual, kChunks>;
  constexpr int smem = Layout<kDual>::kBytes;
  static_assert(smem <= 227 * 1024, "shared memory");
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  if (kp.c.after_selection) return launch_after(kernel, dim3(kp.c.ctas), kThreads, smem, stream, k_map, v_map, q_map, kp);
  kernel<<<kp.c.ctas, kThreads, smem, stream>>>(k_map, v_map, q_map, kp);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_tree_shape(const TreeKernelParams& kp, const CUtensorMap& k_map, const CUtensorMap& v_map,
                              const CUtensorMap& q_map, cudaStream_t stream) {
  const bool dual = kp.c.unit_rows > kRows;
  if (kp.c.a.head_dim <= 64)
    return dual ? launch_tree<T, true, 1>(kp, k_map, v_map, q_map, stream) : launch_tree<T, false, 1>(kp, k_map, v_map, q_map, stream);
  return dual ? launch_tree<T, true, 2>(kp, k_map, v_map, q_map, stream) : launch_tree<T, false, 2>(kp, k_map, v_map, q_map, stream);
}

}  // namespace

ChunkShape chunk_shape_tensor(int64_t max_rows, int num_sms) {
  return {max_rows <= kRows ? kRows : 2 * kRows, kKeys, kUnitCost, num_sms};
}

cudaError_t run_chunk_attention_tensor(const ChunkParams& p, bool q_vec, bool o_vec, const CUtensorMap& k_map,
                                       const CUtensorMap& v_map, const CUtensorMap* q, int dtype, cudaStream_t stream) {
  const TreeKernelParams kp{p, q_vec ? 1 : 0, o_vec ? 1 : 0, q != nullptr ? 1 : 0};
  const CUtensorMap& q_map = q != nullptr ? *q : k_map;
  return dtype == HYT_DTYPE_F16 ? launch_tree_shape<__half>(kp, k_map, v_map, q_map, stream)
                                : launch_tree_shape<__nv_bfloat16>(kp, k_map, v_map, q_map, stream);
}

}  // namespace hyt
