// Tree attention for few rows: bfloat16, at most 32 rows (drafted tokens times the query heads that
// share a key/value head), pages of 8, 16 or 32 keys, heads of 64 to 128.  What it computes and how the
// work is cut is told in hx_tree_attention.cu and hx_tree_attention.cuh.
//
// With few rows the cache's bytes are the bound, and what counts is that copies never stop: not for the
// softmax, not at the end of an item.  On the tcgen05 kernel an item's end costs 10,000 cycles (the last
// product, the rows' way out, the next queries' way in, one behind the other), a fifth of 20 key tiles'
// time, and a tile's softmax takes four warps as long for 16 rows as for 128.  Here a CTA is one or
// two warps of 16 rows each over one ring of chunks of 32 keys, and several CTAs share an SM: while one
// ends an item the others stream.  A warp is all by itself: queries are the A operand of mma.sync
// (m16n8k16) in registers, keys the B operand straight from the blocks as they landed (ldmatrix), the
// softmax stays in registers and is the A operand of the second product, values again from their
// blocks (ldmatrix.trans).  Shared memory is written by the copy engine alone.
//
// Probabilities enter the second product as two bfloat16 terms (hi + lo, 16 bits), which costs nothing for up to
// 16 rows; for more, one term alone (2^-8 of each weight off) would save a tenth (64 requests x 32 drafts, two
// terms 306 to 331 us, one 290).  The reference of a row's exponentials is raised when a chunk exceeds it by more than 2^8,
// each row by itself.
//
// Measured (32 heads of 128, pages of 16): 64 requests x 16 drafts behind 1,200 keys 219 us, 5.8 TB/s of the 6.55 that a
// copy reaches: memory.  8 x 32 behind 640 keys 40 us, 2.3 TB/s: a run of 4 chunks a CTA is too short to hide how
// it starts (5,000 cycles) and is joined.  One request x 8 behind 509 keys 17 us: two launches and the call.
//
// Masks matter in the chunks that hold drafted keys; there values that are not finite are taken as
// zero in the product (what lies behind the last key may be anything, and 0 x infinity would reach
// rows that do not see a drafted one) and drafted ones are added, as what they are, to the rows that see them.
#include "hx_mma.cuh"
#include "hx_tree_attention.cuh"

namespace {

constexpr int KEYS = 32;
constexpr int LEAST = 2;                      // chunks of the shortest run
constexpr float RAISE_MAXIMUM_BY = 8.0f;      // log2 units a chunk must exceed a row's reference by

template <int D, int WARPS>
struct StreamConfig {
  static constexpr int kRows = 16 * WARPS;
  static constexpr int kHalfBytes = KEYS * D * 2;      // keys (or values) of a chunk
  static constexpr int kSlotBytes = 2 * kHalfBytes;
  // (two warps: a ring of 2 or 4 and as many CTAs as fit then took 350 us where this takes 280)
  static constexpr int kRing = (WARPS == 1 ? 2 : 3) * (D <= 64 ? 2 : 1);
  static constexpr int kSmemBytes = kRing * kSlotBytes;
  static constexpr int kFit = 227 * 1024 / (kSmemBytes + 2048);      // CTAs an SM has shared memory for
  static constexpr int kMost = WARPS == 1 ? 6 : 4;                   // ... and registers
  static constexpr int kCtas = kFit < kMost ? kFit : kMost;
};

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
      ::"r"(dst), "l"(src), "r"(bytes), "r"(hx_shared_address(bar))
      : "memory");
}
// The values of keys `key` and `key + 1` of a chunk, those that are infinite or not a number (all ones in
// the exponent) as zero: for keys from `drafted` on, which not every row sees, or which (from `there` on)
// nobody does.  `found`: a drafted one was.
__device__ __forceinline__ uint32_t finite_part(uint32_t pair, int key, int drafted, int there, bool& found) {
  if ((pair & 0x7f80u) == 0x7f80u && key >= drafted) {
    pair &= 0xffff0000u;
    found |= key < there;
  }
  if ((pair & 0x7f800000u) == 0x7f800000u && key + 1 >= drafted) {
    pair &= 0x0000ffffu;
    found |= key + 1 < there;
  }
  return pair;
}

// What is not finite among the drafted values that a row sees in the segment [c.tile, c.tile + count) is
// added to its coordinates d = first + 8 m, + 1: whatever their weight, the sum is not finite either.
template <int D>
__device__ __noinline__ void add_not_finite(const TreeArgs& a, TreeCursor c, int count, int token, int first,
                                            float* sums) {
  const int begin = max(c.context, c.tile * KEYS), end = min(c.context + c.nodes, (c.tile + count) * KEYS);
  const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(a.v_cache);
  for (int key = begin; key < end; ++key) {
    if (!(tree_mask(a, c, token, key / KEYS * KEYS) >> (key % KEYS) & 1)) continue;
    const int index = key / a.page_size;
    if (index >= a.table_stride) continue;
    const int page = a.block_tables[static_cast<size_t>(a.request_table_row[c.request]) * a.table_stride + index];
    if (page < 0 || page >= a.num_pages) continue;
    for (int i = 0; i < D / 4; ++i) {
      const int d = first + i / 2 * 8 + i % 2;
      const float x = __bfloat162float(v[hx_cache_offset(page, c.kv_head(a), key % a.page_size, d, a.kv_heads,
                                                         a.page_size, D, 8)]);
      if (!isfinite(x)) sums[i] += x;
    }
  }
}

template <int D, int WARPS>
__global__ __launch_bounds__(WARPS * 32, StreamConfig<D, WARPS>::kCtas) void tree_stream_kernel(
    const __grid_constant__ TreeArgs a) {
  using Config = StreamConfig<D, WARPS>;
  constexpr int RING = Config::kRing, ROWS = Config::kRows;
  constexpr int D_STEPS = D / 16, D_TILES = D / 8;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint64_t full[RING], empty[RING];
  // the run is found from the step's description, which was there before the kernel in front
  hx_pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const TreeRun run = tree_run<KEYS>(a, blockIdx.x, gridDim.x, LEAST);
  TreeCursor c;
  if (run.count == 0) {
    hx_pdl_wait();
    if (threadIdx.x == 0) tree_tell_none<ROWS>(a);
    return;
  }
  tree_locate<KEYS>(a, run.begin, c);
  if (threadIdx.x == 0) {
    for (int s = 0; s < RING; ++s) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(hx_shared_address(&full[s])));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(hx_shared_address(&empty[s])), "n"(WARPS));
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }

  // ---- warp 0 asks for chunks, `ahead` of the one it works on.  Page numbers are read 32 at a time,
  // the next 32 while these are used.
  const int page_size = a.page_size, pages_per_chunk = KEYS / page_size;
  const uint32_t page_bytes = static_cast<uint32_t>(page_size) * D * 2;
  TreeCursor ahead = c;
  int asked = 0;
  const int* table = nullptr;
  int window = 0, pages = -1, next_pages = -1;
  auto pages_from = [&](int first) {
    const int index = first + lane;
    return index < a.table_stride && index * page_size < ahead.context + ahead.nodes ? table[index] : -1;
  };
  auto enter_item = [&]() {      // `ahead` stands on an item whose pages have not been looked at
    table = a.block_tables + static_cast<size_t>(a.request_table_row[ahead.request]) * a.table_stride;
    window = ahead.tile * pages_per_chunk / 32 * 32;
    pages = pages_from(window);
    next_pages = pages_from(window + 32);
  };
  auto ask = [&]() {
    const int index = ahead.tile * pages_per_chunk;
    if (index - window >= 32) {
      window += 32;
      pages = next_pages;
      next_pages = pages_from(window + 32);
    }
    const int page = __shfl_sync(0xffffffffu, pages, (index - window + lane) & 31);
    long long block = -1;
    if (lane < pages_per_chunk && (index + lane) * page_size < ahead.context + ahead.nodes) {
      if (page >= 0 && page < a.num_pages)
        block = (page * static_cast<long long>(a.kv_heads) + ahead.kv_head(a)) * page_bytes;
      else
        atomicOr(a.status, HX_FLAG_BAD_PAGE);
    }
    const int slot = asked % RING;
    uint64_t* bar = &full[slot];
    const unsigned there = __ballot_sync(0xffffffffu, block >= 0);
    if (lane == 0)
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(hx_shared_address(bar)),
                   "r"(2 * __popc(there) * page_bytes) : "memory");
    __syncwarp();
    if (block >= 0) {
      const uint32_t target = hx_shared_address(ring + static_cast<size_t>(slot) * Config::kSlotBytes) + lane * page_bytes;
      bulk_copy(target, static_cast<const uint8_t*>(a.k_cache) + block, page_bytes, bar);
      bulk_copy(target + Config::kHalfBytes, static_cast<const uint8_t*>(a.v_cache) + block, page_bytes, bar);
    }
    ++asked;
    if (asked < run.count && ++ahead.tile == ahead.tiles) {
      const int request = ahead.request;
      tree_next_item<KEYS>(a, ahead);
      if (ahead.request != request) {
        enter_item();
      } else {
        if (window != 0) pages = pages_from(0), next_pages = pages_from(32);
        window = 0;
      }
    }
  };

  if (warp == 0) enter_item();      // (tables are part of the description, too)
  hx_pdl_wait();
  if (threadIdx.x == 0) tree_tell_none<ROWS>(a);
  __syncthreads();
  if (warp == 0)
    while (asked < RING && asked < run.count) ask();

  // where this lane's ldmatrix rows sit in a slot: keys as matrices (keys 0-7, d lo), (keys 0-7, d
  // hi), (keys 8-15, d lo), (keys 8-15, d hi) of 16 keys, values (transposed) as (keys 0-7, d lo),
  // (keys 8-15, d lo), (keys 0-7, d hi), (keys 8-15, d hi)
  const int matrix = lane >> 3, group = lane >> 2, quad = lane & 3;
  const uint32_t piece_step = static_cast<uint32_t>(page_size) * 32;      // two 16-byte pieces on
  uint32_t k_offset[2], v_offset[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int k_key = 16 * h + (matrix >> 1) * 8 + (lane & 7), v_key = 16 * h + (matrix & 1) * 8 + (lane & 7);
    k_offset[h] = (k_key / page_size) * page_bytes + (((matrix & 1) * page_size + k_key % page_size) << 4);
    v_offset[h] = (v_key / page_size) * page_bytes + (((matrix >> 1) * page_size + v_key % page_size) << 4);
  }
  const float scale_log2 = a.scale * HX_LOG2E;
  const int row_low = 16 * warp + group, row_high = row_low + 8;      // this lane's rows
  int i = 0;      // chunk of the run
  bool ok = true;
  for (int left = run.count; left > 0 && ok;) {
    const int count = min(c.tiles - c.tile, left);
    const TreeRows rows(a, c);
    const bool live = 16 * warp < rows.count;
    const int token_low = rows.token0 + min(row_low, rows.count - 1) / rows.heads;
    const int token_high = rows.token0 + min(row_high, rows.count - 1) / rows.heads;
    const int head_low = rows.head0 + row_low % rows.heads, head_high = rows.head0 + row_high % rows.heads;
    // the queries as A operand: rows group and group + 8, d 16 k + 2 quad and 8 on
    uint32_t q_frag[D_STEPS][4];
    float o[D_TILES][4];
    float max_low = -INFINITY, max_high = -INFINITY, sum_low = 0.0f, sum_high = 0.0f;
    bool poisoned = false;
    // the first words of the rows' masks, which are wanted at the item's end
    unsigned long long first_low = 0, first_high = 0;
    if (live) {
      first_low = __ldg(tree_words(a, c, token_low));
      first_high = __ldg(tree_words(a, c, token_high));
      const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) + 2 * quad;
      const __nv_bfloat16* q_low = q + static_cast<size_t>(c.q_begin + token_low) * a.ldq + static_cast<size_t>(head_low) * D;
      const __nv_bfloat16* q_high = q + static_cast<size_t>(c.q_begin + token_high) * a.ldq + static_cast<size_t>(head_high) * D;
#pragma unroll
      for (int k = 0; k < D_STEPS; ++k) {
        q_frag[k][0] = *reinterpret_cast<const uint32_t*>(q_low + 16 * k);
        q_frag[k][1] = *reinterpret_cast<const uint32_t*>(q_high + 16 * k);
        q_frag[k][2] = *reinterpret_cast<const uint32_t*>(q_low + 16 * k + 8);
        q_frag[k][3] = *reinterpret_cast<const uint32_t*>(q_high + 16 * k + 8);
      }
#pragma unroll
      for (int m = 0; m < D_TILES; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[m][e] = 0.0f;
    }
    for (int t = 0; t < count; ++t, ++i) {
      const int slot = i % RING;
      int arrived = 1;
      if (lane == 0) arrived = tree_wait(&full[slot], static_cast<uint32_t>(i / RING) & 1u);
      ok = __shfl_sync(0xffffffffu, arrived, 0) != 0;
      if (!ok) break;
      if constexpr (WARPS > 1) {
        // the slot of the chunk before, which the other warps have had this long to get through with
        if (warp == 0 && i > 0 && asked < run.count) {
          int freed = 1;
          if (lane == 0) freed = tree_wait(&empty[(i - 1) % RING], static_cast<uint32_t>((i - 1) / RING) & 1u);
          ok = __shfl_sync(0xffffffffu, freed, 0) != 0;
          if (!ok) break;
          ask();
        }
      }
      if (live) {
        const uint32_t k_half = hx_shared_address(ring + static_cast<size_t>(slot) * Config::kSlotBytes);
        const uint32_t v_half = k_half + Config::kHalfBytes;
        const int key0 = (c.tile + t) * KEYS;
        const bool drafted = key0 + KEYS > c.context;
        // ---- scores: rows group, group + 8 (elements 2, 3); keys 8 j + 2 quad, + 1
        float s[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[j][e] = 0.0f;
#pragma unroll
        for (int k = 0; k < D_STEPS; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t b[4];
            hx_ldmatrix_x4(b, k_half + k_offset[h] + k * piece_step);
            hx_mma_bf16(s[2 * h], q_frag[k], b[0], b[1]);
            hx_mma_bf16(s[2 * h + 1], q_frag[k], b[2], b[3]);
          }
        if (drafted) {
          const unsigned long long* words_low = tree_words(a, c, token_low);
          const unsigned long long* words_high = tree_words(a, c, token_high);
          const uint32_t low = static_cast<uint32_t>(tree_mask_of(
                                   a, c, key0, first_low, [&](int word) { return words_low[word]; })) >> (2 * quad);
          const uint32_t high = static_cast<uint32_t>(tree_mask_of(
                                    a, c, key0, first_high, [&](int word) { return words_high[word]; })) >> (2 * quad);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (!(low >> (8 * j) & 1)) s[j][0] = -INFINITY;
            if (!(low >> (8 * j + 1) & 1)) s[j][1] = -INFINITY;
            if (!(high >> (8 * j) & 1)) s[j][2] = -INFINITY;
            if (!(high >> (8 * j + 1) & 1)) s[j][3] = -INFINITY;
          }
        }
        float top_low = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])),
                              fmaxf(fmaxf(s[2][0], s[2][1]), fmaxf(s[3][0], s[3][1])));
        float top_high = fmaxf(fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3])),
                               fmaxf(fmaxf(s[2][2], s[2][3]), fmaxf(s[3][2], s[3][3])));
#pragma unroll
        for (int offset = 1; offset <= 2; offset <<= 1) {
          top_low = fmaxf(top_low, __shfl_xor_sync(0xffffffffu, top_low, offset));
          top_high = fmaxf(top_high, __shfl_xor_sync(0xffffffffu, top_high, offset));
        }
        top_low *= scale_log2;
        top_high *= scale_log2;
        // (a row that has seen nothing yet keeps -inf as its reference and zeros as its probabilities)
        const bool exceeds_low = top_low > max_low + RAISE_MAXIMUM_BY || (t == 0 && top_low != -INFINITY);
        const bool exceeds_high = top_high > max_high + RAISE_MAXIMUM_BY || (t == 0 && top_high != -INFINITY);
        if (__any_sync(0xffffffffu, exceeds_low || exceeds_high)) {
          const float correct_low = exceeds_low ? fast_exp2(max_low - top_low) : 1.0f;
          const float correct_high = exceeds_high ? fast_exp2(max_high - top_high) : 1.0f;
          if (exceeds_low) max_low = top_low;
          if (exceeds_high) max_high = top_high;
          sum_low *= correct_low;
          sum_high *= correct_high;
#pragma unroll
          for (int m = 0; m < D_TILES; ++m) {
            o[m][0] *= correct_low;
            o[m][1] *= correct_low;
            o[m][2] *= correct_high;
            o[m][3] *= correct_high;
          }
        }
        const float against_low = max_low == -INFINITY ? 0.0f : max_low;
        const float against_high = max_high == -INFINITY ? 0.0f : max_high;
        // ---- probabilities, in two terms, as A operand: keys 16 h + 2 quad and 8 on
        uint32_t p_hi[2][4], p_lo[2][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p0 = fast_exp2(fmaf(s[j][0], scale_log2, -against_low));
          const float p1 = fast_exp2(fmaf(s[j][1], scale_log2, -against_low));
          const float p2 = fast_exp2(fmaf(s[j][2], scale_log2, -against_high));
          const float p3 = fast_exp2(fmaf(s[j][3], scale_log2, -against_high));
          sum_low += p0 + p1;
          sum_high += p2 + p3;
          hx_split_bf16(p0, p1, p_hi[j >> 1][2 * (j & 1)], p_lo[j >> 1][2 * (j & 1)]);
          hx_split_bf16(p2, p3, p_hi[j >> 1][2 * (j & 1) + 1], p_lo[j >> 1][2 * (j & 1) + 1]);
        }
        // ---- the weighted values: d tiles 2 m and 2 m + 1
        if (!drafted) {
#pragma unroll
          for (int m = 0; m < D_STEPS; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t b[4];
              hx_ldmatrix_x4_trans(b, v_half + v_offset[h] + m * piece_step);
              hx_mma_bf16(o[2 * m], p_hi[h], b[0], b[1]);
              hx_mma_bf16(o[2 * m + 1], p_hi[h], b[2], b[3]);
              hx_mma_bf16(o[2 * m], p_lo[h], b[0], b[1]);
              hx_mma_bf16(o[2 * m + 1], p_lo[h], b[2], b[3]);
            }
        } else {
          bool found = false;
          const int first_drafted = c.context - key0, there = first_drafted + c.nodes;
#pragma unroll
          for (int m = 0; m < D_STEPS; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t b[4];
              hx_ldmatrix_x4_trans(b, v_half + v_offset[h] + m * piece_step);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                b[e] = finite_part(b[e], 16 * h + 8 * (e & 1) + 2 * quad, first_drafted, there, found);
              hx_mma_bf16(o[2 * m], p_hi[h], b[0], b[1]);
              hx_mma_bf16(o[2 * m + 1], p_hi[h], b[2], b[3]);
              hx_mma_bf16(o[2 * m], p_lo[h], b[0], b[1]);
              hx_mma_bf16(o[2 * m + 1], p_lo[h], b[2], b[3]);
            }
          poisoned |= __any_sync(0xffffffffu, found) != 0;
        }
      }
      // ---- this warp is through with the slot
      __syncwarp();
      if constexpr (WARPS == 1) {
        if (asked < run.count) ask();
      } else if (lane == 0) {
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(hx_shared_address(&empty[slot])) : "memory");
      }
    }
    if (!ok) break;
    // ---- the segment's rows: finished, or this CTA's part of them
    if (live) {
#pragma unroll
      for (int offset = 1; offset <= 2; offset <<= 1) {
        sum_low += __shfl_xor_sync(0xffffffffu, sum_low, offset);
        sum_high += __shfl_xor_sync(0xffffffffu, sum_high, offset);
      }
      if (poisoned) {
        float sums[D / 4];
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
#pragma unroll
          for (int e = 0; e < D / 4; ++e) sums[e] = 0.0f;
          add_not_finite<D>(a, c, count, half == 0 ? token_low : token_high, 2 * quad, sums);
#pragma unroll
          for (int m = 0; m < D_TILES; ++m)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if (half == 0) o[m][e] += sums[2 * m + e];
              else o[m][2 + e] += sums[2 * m + e];
            }
        }
      }
      const bool whole = c.tile == 0 && count == c.tiles;
      if (whole) {
        const float inverse_low = tree_inverse(sum_low);
        const float inverse_high = tree_inverse(sum_high);
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + 2 * quad;
        __nv_bfloat16* out_low = out + static_cast<size_t>(c.q_begin + token_low) * a.ldo + static_cast<size_t>(head_low) * D;
        __nv_bfloat16* out_high = out + static_cast<size_t>(c.q_begin + token_high) * a.ldo + static_cast<size_t>(head_high) * D;
#pragma unroll
        for (int m = 0; m < D_TILES; ++m) {
          if (row_low < rows.count)
            *reinterpret_cast<uint32_t*>(out_low + 8 * m) = hx_pack_bf16(o[m][0] * inverse_low, o[m][1] * inverse_low);
          if (row_high < rows.count)
            *reinterpret_cast<uint32_t*>(out_high + 8 * m) = hx_pack_bf16(o[m][2] * inverse_high, o[m][3] * inverse_high);
        }
      } else {
        float* part = tree_part<ROWS>(a, blockIdx.x, c.tile == 0);
#pragma unroll
        for (int m = 0; m < D_TILES; ++m) {
          float* at = part + (4 * m + quad) * ROWS * 2;
          *reinterpret_cast<float2*>(at + 2 * row_low) = make_float2(o[m][0], o[m][1]);
          *reinterpret_cast<float2*>(at + 2 * row_high) = make_float2(o[m][2], o[m][3]);
        }
        if (quad == 0) {
          part[D * ROWS + row_low] = max_low;
          part[D * ROWS + row_high] = max_high;
          part[(D + 1) * ROWS + row_low] = sum_low;
          part[(D + 1) * ROWS + row_high] = sum_high;
        }
      }
    }
    left -= count;
    if (left > 0) tree_next_item<KEYS>(a, c);
    else if (threadIdx.x == 0) tree_tell_cut<ROWS>(a, run, c, count);
  }
  if (!ok) {
    if (lane == 0) atomicOr(a.status, HX_FLAG_WAIT_TIMEOUT);
    // a CTA does not leave while copies into its shared memory are in flight
    if (threadIdx.x == 0)
      for (int n = max(0, asked - RING); n < asked; ++n) tree_wait(&full[n % RING], static_cast<uint32_t>(n / RING) & 1u);
    __syncwarp();
  }
}

template <int D, int WARPS>
int launch(const TreeArgs& a, cudaStream_t stream) {
  using Config = StreamConfig<D, WARPS>;
  static std::atomic<unsigned long long> ready{0};
  const bool reserved = hx_once_a_device(ready, [] {
    return cudaFuncSetAttribute(tree_stream_kernel<D, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                Config::kSmemBytes) == cudaSuccess &&
           // (else the driver keeps more of it for L1 than leaves room for kCtas)
           cudaFuncSetAttribute(tree_stream_kernel<D, WARPS>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                cudaSharedmemCarveoutMaxShared) == cudaSuccess;
  });
  HX_REQUIRE(reserved, "hx_tree_attention: cannot reserve %d bytes of shared memory", Config::kSmemBytes);
  const int ctas = hx_device_sm_count() * Config::kCtas;
  hx_launch(tree_stream_kernel<D, WARPS>, ctas, WARPS * 32, Config::kSmemBytes, stream, a);
  HX_CHECK_LAUNCH("hx_tree_attention");
  return hx_tree_join(a, HX_BF16, ctas, Config::kRows, 2, stream);
}

template <int D>
int launch_for(TreeArgs& a, int warps, cudaStream_t stream) {
  tree_fill_rows(a, 16 * warps);
  return warps == 1 ? launch<D, 1>(a, stream) : launch<D, 2>(a, stream);
}

template <int D>
long long floats_for(int sms) {
  const long long one = tree_scratch_floats<16>(D, sms * StreamConfig<D, 1>::kCtas);
  const long long two = tree_scratch_floats<32>(D, sms * StreamConfig<D, 2>::kCtas);
  return one > two ? one : two;
}

}  // namespace

bool hx_tree_stream_takes(int head_dim, int page_size) {
  return head_dim >= 64 && head_dim <= 128 && head_dim % 16 == 0 &&
         (page_size == 8 || page_size == 16 || page_size == 32);
}

long long hx_tree_stream_floats(int head_dim) {
  const int sms = hx_device_sm_count();
  switch (head_dim) {
    case 64: return floats_for<64>(sms);
    case 80: return floats_for<80>(sms);
    case 96: return floats_for<96>(sms);
    case 112: return floats_for<112>(sms);
    default: return floats_for<128>(sms);
  }
}

int hx_tree_stream_launch(TreeArgs a, int rows, cudaStream_t stream) {
  const int warps = rows <= 16 ? 1 : 2;
  switch (a.head_dim) {
    case 64: return launch_for<64>(a, warps, stream);
    case 80: return launch_for<80>(a, warps, stream);
    case 96: return launch_for<96>(a, warps, stream);
    case 112: return launch_for<112>(a, warps, stream);
    default: return launch_for<128>(a, warps, stream);
  }
}
