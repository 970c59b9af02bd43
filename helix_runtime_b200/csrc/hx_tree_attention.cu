// Attention of a tree of drafted tokens over the paged cache.
//
// A request brings `nodes` drafted tokens to a step.  Token n's key and value lie in the request's
// pages at place context + n (whatever position it was rotated for); it attends to the context
// cached keys and to the drafted tokens its bit mask names, usually itself and its ancestors in the
// tree:
//     o_n = sum_j w_nj v_j / sum_j w_nj,   w_nj = exp(scale q_n . k_j),   j cached or named.
// A token that sees nothing (no cached key, no bit) gets zeros.
//
// The causal kernels take one position per token and everything in front of it; here the order of
// the drafted keys says nothing, and all tokens of a request read the same cached keys.  So a
// CTA takes the tokens of a request (and the query heads that share a key/value head) as rows of
// one tile and reads every key once for all of them; a long context is cut over CTAs (see
// hx_tree_attention.cuh).  Four kernels:
//   * hx_tree_attention_stream.cu: bfloat16, heads of 64 to 128, pages of 8, 16 or 32 keys, few rows;
//   * hx_tree_attention_tc.cu: the same with many rows, and pages of 64;
//   * tree_tile_kernel: any other page size, float32 or bfloat16, heads up to 256 in steps of 4.
//     32 rows by 64 keys at a time on the CUDA cores, all in float32;
//   * tree_row_kernel: what is left (heads up to 1,024, even), a row a warp.
#include "hx_mma.cuh"
#include "hx_tree_attention.cuh"

namespace {

// ------------------------------------------------------------------ 32 rows x 64 keys

constexpr int TILE_ROWS = 32, TILE_KEYS = 64, TILE_WARPS = 4, ROWS_A_WARP = TILE_ROWS / TILE_WARPS;
constexpr int TILE_LEAST = 2;      // key tiles of the shortest run

template <int D_MAX>
struct TileConfig {
  // queries [32][D], keys [D / 4][64][4] and then, in the same place, values [64][D + 4], probabilities [32][64]
  static constexpr int floats(int d) { return TILE_ROWS * d + TILE_KEYS * (d + 4) + TILE_ROWS * TILE_KEYS; }
  static constexpr int kCtas = D_MAX <= 128 ? 4 : 2;
};

// Four consecutive coordinates of a cached row, wherever the cache's pieces put them.
template <typename T> __device__ __forceinline__ float4 load_four(const T* p);
template <> __device__ __forceinline__ float4 load_four<float>(const float* p) {
  return *reinterpret_cast<const float4*>(p);
}
template <> __device__ __forceinline__ float4 load_four<__nv_bfloat16>(const __nv_bfloat16* p) {
  const uint2 raw = *reinterpret_cast<const uint2*>(p);
  const __nv_bfloat162 low = *reinterpret_cast<const __nv_bfloat162*>(&raw.x);
  const __nv_bfloat162 high = *reinterpret_cast<const __nv_bfloat162*>(&raw.y);
  return make_float4(__bfloat162float(low.x), __bfloat162float(low.y), __bfloat162float(high.x),
                     __bfloat162float(high.y));
}

// 16 bytes of float32, or four bfloat16 as float32, on their way into shared memory.
template <typename T> __device__ __forceinline__ void bring_four(float* place, const T* from, bool there);
template <> __device__ __forceinline__ void bring_four<float>(float* place, const float* from, bool there) {
  hx_cp_async_16(hx_shared_address(place), from, there ? 16 : 0);
}
template <> __device__ __forceinline__ void bring_four<__nv_bfloat16>(float* place, const __nv_bfloat16* from, bool there) {
  *reinterpret_cast<float4*>(place) = there ? load_four<__nv_bfloat16>(from) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
}

// a += w x and b += w y, one instruction.
__device__ __forceinline__ void two_fma(float w, float x, float y, float& a, float& b) {
  asm("{\n\t.reg .b64 w, v, s;\n\t"
      "mov.b64 w, {%2, %2};\n\tmov.b64 v, {%3, %4};\n\tmov.b64 s, {%0, %1};\n\t"
      "fma.rn.f32x2 s, w, v, s;\n\tmov.b64 {%0, %1}, s;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(w), "f"(x), "f"(y));
}

// A weight that stands for a key which its row does not see (weights themselves are never negative).
constexpr uint32_t NOT_SEEN = 0x80000000u;

// acc[i] += a tile's values by the probabilities of row i: coordinates 4 lane .. of a warp's rows.  MASKED: a
// (drafted) key that a row does not see adds nothing to it, not even an infinity times zero.  One that it sees
// adds what its weight makes of it, also a weight of zero, as in tiles without drafted keys.
template <bool MASKED, int PIECES>
__device__ __forceinline__ void tile_weigh(float4 (&acc)[ROWS_A_WARP][PIECES], const float4* my_p, const float* values,
                                           int D, int lane, int keys) {
  for (int key4 = 0; key4 * 4 < keys; ++key4) {
    float4 v[4][PIECES];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int j = 0; j < PIECES; ++j) {
        const int d = 4 * lane + 128 * j;
        if (d < D) v[k][j] = *reinterpret_cast<const float4*>(values + (4 * key4 + k) * (D + 4) + d);
      }
#pragma unroll
    for (int i = 0; i < ROWS_A_WARP; ++i) {
      const float4 p = my_p[i * (TILE_KEYS / 4) + key4];
      const float w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
          if (MASKED && __float_as_uint(w[k]) == NOT_SEEN) continue;
          two_fma(w[k], v[k][j].x, v[k][j].y, acc[i][j].x, acc[i][j].y);
          two_fma(w[k], v[k][j].z, v[k][j].w, acc[i][j].z, acc[i][j].w);
        }
    }
  }
}

// A warp has 8 rows of the tile.  Scores: a lane has 4 keys (16 apart) of 4 rows, so that 12 reads of 128
// bytes of shared memory feed 64 multiply-adds of a warp.  Values: a lane has 4 (8, above 128)
// coordinates of all 8 rows.  A tile of heads of 112 is 3,900 cycles of multiply-adds, 15,600 for an SM's four
// CTAs, of the 35,000 that these take: the rest is what its phases wait for, copies, shared memory and one another, as the
// CTAs run in step.  What counts is that enough warps are there to fill such waits: a tile's values take the place of its
// keys, so that four CTAs share an SM.  4 requests x 24 drafts behind 700 keys, 32 heads of 112, float32: 80 us
// (1.1 TB/s, 12 TFLOP/s).  Two CTAs, with keys and values side by side and the next ones on their way, took 95, the
// same rows spread evenly over the warps 97, 2 keys by 8 rows a lane 90; weighted values without a question for masks where no key is
// drafted, two multiply-adds an instruction, 79 instead of 84 (the same for the scores took registers it has not: 90).  Of a tile's
// 35,000 cycles, CTAs in step, scores are 12,000, weighted values 10,000, copies 8,500, the softmax 4,000.  A thread copies half a key, whose page it has looked up a tile before.
template <typename T, int D_MAX>
__global__ __launch_bounds__(TILE_WARPS * 32, TileConfig<D_MAX>::kCtas) void tree_tile_kernel(
    const TreeArgs a) {
  extern __shared__ float4 tile_shared[];
  constexpr int OUT_PIECES = (D_MAX + 127) / 128;
  static_assert(TILE_KEYS == 64 && TILE_WARPS * 32 == 2 * TILE_KEYS, "two threads copy a key");
  hx_pdl_prologue();
  const int D = a.head_dim, D4 = D / 4;
  float* q_rows = reinterpret_cast<float*>(tile_shared);
  float* keys = q_rows + TILE_ROWS * D;
  float* values = keys;
  float* probabilities = keys + TILE_KEYS * (D + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const TreeRun run = tree_run<TILE_KEYS>(a, blockIdx.x, gridDim.x, TILE_LEAST);
  if (threadIdx.x == 0) tree_tell_none<TILE_ROWS>(a);
  if (run.count == 0) return;
  TreeCursor c;
  tree_locate<TILE_KEYS>(a, run.begin, c);
  const int chunk = hx_cache_chunk(sizeof(T), D);
  const T* q = static_cast<const T*>(a.q);
  const T* k_cache = static_cast<const T*>(a.k_cache);
  const T* v_cache = static_cast<const T*>(a.v_cache);
  const float scale_log2 = a.scale * HX_LOG2E;
  const int my_key = threadIdx.x % TILE_KEYS, my_half = threadIdx.x / TILE_KEYS;      // of a tile's copies
  const int key_x = lane & 15, row_y = lane >> 4;                                     // of a tile's scores
  // four coordinates on: the next piece of `chunk`, or further in the same one
  const int pieces_a_chunk = chunk / 4;

  for (int left = run.count; left > 0;) {
    const int count = min(c.tiles - c.tile, left);
    const TreeRows rows(a, c);
    const int rows_here = rows.count, kv_head = rows.kv_head;
    const int last_key = c.context + c.nodes - 1;
    const int* table = a.block_tables + static_cast<size_t>(a.request_table_row[c.request]) * a.table_stride;
    auto page_of = [&](int key) {
      const int index = key / a.page_size;
      return key <= last_key && index < a.table_stride ? table[index] : -1;
    };
    // the pieces of a key (or value) of this thread; one that does not exist or has no page is zeros
    auto bring = [&](int key, int page, const T* cache, float* place, int stride) {
      const bool there = page >= 0 && page < a.num_pages && key <= last_key;
      const T* from = cache + (there ? hx_cache_offset(page, kv_head, key % a.page_size, 0, a.kv_heads, a.page_size, D, chunk) : 0);
      const size_t step = there ? static_cast<size_t>(a.page_size) * chunk : 0;
#pragma unroll 4
      for (int d4 = my_half; d4 < D4; d4 += 2)      // (coordinates 4 d4: a chunk's first, or further on in it)
        bring_four<T>(place + d4 * stride, from + d4 / pieces_a_chunk * step + (there ? d4 % pieces_a_chunk * 4 : 0), there);
      hx_cp_async_commit();
      return there || key > last_key;
    };
    float* my_keys = keys + my_key * 4;
    float* my_values = values + my_key * (D + 4);
    int key = c.tile * TILE_KEYS + my_key;      // of the tile that is copied next
    int page = page_of(key), page_after = count > 1 ? page_of(key + TILE_KEYS) : -1;
    __syncthreads();      // the last item's tiles have been read
    if (!bring(key, page, k_cache, my_keys, 4 * TILE_KEYS)) atomicOr(a.status, HX_FLAG_BAD_PAGE);
    for (int i = threadIdx.x; i < TILE_ROWS * D4; i += blockDim.x) {
      const int row = i / D4, d4 = i - row * D4;
      float4 value = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (row < rows_here)
        value = load_four<T>(q + static_cast<size_t>(c.q_begin + rows.token0 + row / rows.heads) * a.ldq +
                             static_cast<size_t>(rows.head0 + row % rows.heads) * D + 4 * d4);
      reinterpret_cast<float4*>(q_rows)[row * D4 + d4] = value;
    }
    float row_max[4], row_sum[4];      // of the rows whose scores this lane has
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      row_max[j] = -INFINITY;
      row_sum[j] = 0.0f;
    }
    float4 acc[ROWS_A_WARP][OUT_PIECES];
#pragma unroll
    for (int i = 0; i < ROWS_A_WARP; ++i)
#pragma unroll
      for (int j = 0; j < OUT_PIECES; ++j) acc[i][j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const bool live = warp * ROWS_A_WARP < rows_here;      // this warp has rows
    for (int t = 0; t < count; ++t) {
      const int key0 = (c.tile + t) * TILE_KEYS;
      hx_cp_async_wait<0>();      // this tile's keys
      __syncthreads();            // everybody's; and the queries are written
      // ---- scores of rows 4 row_y + j against keys key_x + 16 i
      float s[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[j][i] = 0.0f;
      const float4* my_q = reinterpret_cast<const float4*>(q_rows) + (warp * ROWS_A_WARP + 4 * row_y) * D4;
      const float4* my_k = reinterpret_cast<const float4*>(keys) + key_x;
#pragma unroll 1
      for (int d4 = 0; d4 < (live ? D4 : 0); ++d4) {
        float4 k[4], w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = my_k[d4 * TILE_KEYS + 16 * i];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = my_q[j * D4 + d4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[j][i] = fmaf(w[j].x, k[i].x, s[j][i]);
            s[j][i] = fmaf(w[j].y, k[i].y, s[j][i]);
            s[j][i] = fmaf(w[j].z, k[i].z, s[j][i]);
            s[j][i] = fmaf(w[j].w, k[i].w, s[j][i]);
          }
      }
      __syncthreads();      // the keys have been read
      bring(key, page, v_cache, my_values, 4);
      const bool more = t + 1 < count;
      key += TILE_KEYS;
      page = page_after;
      if (t + 2 < count) page_after = page_of(key + TILE_KEYS);
      // ---- the running maximum and sum of every row (sixteen lanes have one)
      const bool drafted = key0 + TILE_KEYS > c.context;
      float correction[4];
      if (live) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = warp * ROWS_A_WARP + 4 * row_y + j;
        unsigned seen = ~0u;      // bit 16 (i % 2) + i / 2 of it: the row sees key key_x + 16 i
        if (drafted) {
          const unsigned long long mask =
              (row < rows_here ? tree_mask(a, c, rows.token0 + row / rows.heads, key0) : 0ull) >> key_x;
          seen = (static_cast<unsigned>(mask) & 0x00010001u) | (static_cast<unsigned>(mask >> 32) & 0x00010001u) << 1;
        }
        auto sees = [&](int i) { return (seen >> (16 * (i % 2) + i / 2)) & 1; };
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[j][i] = sees(i) ? s[j][i] * scale_log2 : -INFINITY;
          top = fmaxf(top, s[j][i]);
        }
#pragma unroll
        for (int offset = 8; offset > 0; offset >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, offset));
        const float new_max = fmaxf(row_max[j], top);
        const float against = new_max == -INFINITY ? 0.0f : new_max;
        correction[j] = exp2f(row_max[j] - against);
        row_max[j] = new_max;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = exp2f(s[j][i] - against);
          sum += p;
          probabilities[row * TILE_KEYS + key_x + 16 * i] = sees(i) ? p : __uint_as_float(NOT_SEEN);
        }
#pragma unroll
        for (int offset = 8; offset > 0; offset >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, offset);
        row_sum[j] = fmaf(row_sum[j], correction[j], sum);
      }
#pragma unroll
      for (int i = 0; i < ROWS_A_WARP; ++i) {
        const float factor = __shfl_sync(0xffffffffu, correction[i % 4], i / 4 * 16);
#pragma unroll
        for (int j = 0; j < OUT_PIECES; ++j) {
          acc[i][j].x *= factor;
          acc[i][j].y *= factor;
          acc[i][j].z *= factor;
          acc[i][j].w *= factor;
        }
      }
      }
      hx_cp_async_wait<0>();      // this tile's values
      __syncthreads();
      // ---- the weighted values: coordinates 4 lane .. of 8 rows, four keys at a time
      const float4* my_p = reinterpret_cast<const float4*>(probabilities) + warp * ROWS_A_WARP * (TILE_KEYS / 4);
      const int keys_here = live ? min(TILE_KEYS, last_key + 1 - key0) : 0;
      if (drafted) tile_weigh<true>(acc, my_p, values, D, lane, keys_here);
      else tile_weigh<false>(acc, my_p, values, D, lane, keys_here);
      if (more) {
        __syncthreads();      // the values have been read
        if (!bring(key, page, k_cache, my_keys, 4 * TILE_KEYS)) atomicOr(a.status, HX_FLAG_BAD_PAGE);
      }
    }
    // ---- the rows, or this CTA's part of them
    if (live) {
      const bool whole = c.tile == 0 && count == c.tiles;
      float* part = tree_part<TILE_ROWS>(a, blockIdx.x, c.tile == 0);
#pragma unroll
      for (int i = 0; i < ROWS_A_WARP; ++i) {
        const float top = __shfl_sync(0xffffffffu, row_max[i % 4], i / 4 * 16);
        const float sum = __shfl_sync(0xffffffffu, row_sum[i % 4], i / 4 * 16);
        const int row = warp * ROWS_A_WARP + i;
        if (row >= rows_here) continue;
        const float inverse = tree_inverse(sum);
        T* out = static_cast<T*>(a.out) + static_cast<size_t>(c.q_begin + rows.token0 + row / rows.heads) * a.ldo +
                 static_cast<size_t>(rows.head0 + row % rows.heads) * D;
#pragma unroll
        for (int j = 0; j < OUT_PIECES; ++j) {
          const int d = 4 * lane + 128 * j;
          if (d >= D) continue;
          const float4 v = acc[i][j];
          if (whole) {
            out[d] = hx_from_float<T>(v.x * inverse);
            out[d + 1] = hx_from_float<T>(v.y * inverse);
            out[d + 2] = hx_from_float<T>(v.z * inverse);
            out[d + 3] = hx_from_float<T>(v.w * inverse);
          } else {
            *reinterpret_cast<float4*>(part + (static_cast<size_t>(d / 4) * TILE_ROWS + row) * 4) = v;
          }
        }
        if (!whole && lane == 0) {
          part[static_cast<size_t>(D) * TILE_ROWS + row] = top;
          part[static_cast<size_t>(D + 1) * TILE_ROWS + row] = sum;
        }
      }
    }
    left -= count;
    if (left > 0) tree_next_item<TILE_KEYS>(a, c);
    else if (threadIdx.x == 0) tree_tell_cut<TILE_ROWS>(a, run, c, count);
  }
}

// ------------------------------------------------------------------ a row a warp

constexpr int ROW_WARPS = 4, ROW_KEYS = 64, ROW_MAX_DIM = 1024, ROW_CTAS = 4, ROW_LEAST = 2;

// Lane j owns keys j and j + 32 of a tile for the scores and pairs of coordinates 2 lane + 64 i for
// the values.  No shared keys: for head sizes that no model here has, right rather than fast.
template <typename T>
__global__ __launch_bounds__(ROW_WARPS * 32) void tree_row_kernel(const TreeArgs a) {
  __shared__ float q_shared[ROW_WARPS][ROW_MAX_DIM];
  constexpr int PAIRS = ROW_MAX_DIM / 64;
  hx_pdl_prologue();
  const int D = a.head_dim, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const TreeRun run = tree_run<ROW_KEYS>(a, blockIdx.x, gridDim.x, ROW_LEAST);
  if (threadIdx.x == 0) tree_tell_none<ROW_WARPS>(a);
  if (run.count == 0) return;
  TreeCursor c;
  tree_locate<ROW_KEYS>(a, run.begin, c);
  const int chunk = hx_cache_chunk(sizeof(T), D);
  const T* k_cache = static_cast<const T*>(a.k_cache);
  const T* v_cache = static_cast<const T*>(a.v_cache);
  const float scale_log2 = a.scale * HX_LOG2E;
  for (int left = run.count; left > 0;) {
    const int count = min(c.tiles - c.tile, left);
    const TreeRows rows(a, c);
    const int rows_here = rows.count, kv_head = rows.kv_head;
    const int last_key = c.context + c.nodes - 1;
    const int* table = a.block_tables + static_cast<size_t>(a.request_table_row[c.request]) * a.table_stride;
    const int row = warp;
    if (row < rows_here) {
      const int token = rows.token0 + row / rows.heads, head = rows.head0 + row % rows.heads;
      const T* q = static_cast<const T*>(a.q) + static_cast<size_t>(c.q_begin + token) * a.ldq +
                   static_cast<size_t>(head) * D;
      float* qs = q_shared[warp];
      __syncwarp();
      for (int d = lane; d < D; d += 32) qs[d] = hx_to_float<T>(q[d]);
      __syncwarp();
      float acc[PAIRS][2];
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) acc[i][0] = acc[i][1] = 0.0f;
      float row_max = -INFINITY, row_sum = 0.0f;
      for (int t = 0; t < count; ++t) {
        const int key0 = (c.tile + t) * ROW_KEYS;
        const unsigned long long mask = tree_mask(a, c, token, key0);
        for (int half = 0; half < 2; ++half) {
          const int key = key0 + 32 * half + lane;
          int page = -1;
          if (key <= last_key) {
            const int index = key / a.page_size;
            page = index < a.table_stride ? table[index] : -1;
            if (page < 0 || page >= a.num_pages) {
              atomicOr(a.status, HX_FLAG_BAD_PAGE);
              page = -1;
            }
          }
          float score = -INFINITY;
          if (page >= 0 && ((mask >> (32 * half + lane)) & 1)) {
            float dot = 0.0f;
            for (int d = 0; d < D; d += 2) {
              const T* k = k_cache + hx_cache_offset(page, kv_head, key % a.page_size, d, a.kv_heads,
                                                     a.page_size, D, chunk);
              dot = fmaf(qs[d], hx_to_float<T>(k[0]), dot);
              dot = fmaf(qs[d + 1], hx_to_float<T>(k[1]), dot);
            }
            score = dot * scale_log2;
          }
          const unsigned seen = __ballot_sync(0xffffffffu, score != -INFINITY);
          if (seen == 0u) continue;
          float top = score;
#pragma unroll
          for (int offset = 16; offset > 0; offset >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, offset));
          const float new_max = fmaxf(row_max, top);
          const float correction = exp2f(row_max - new_max);
          const float p = score == -INFINITY ? 0.0f : exp2f(score - new_max);
          float sum = p;
#pragma unroll
          for (int offset = 16; offset > 0; offset >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, offset);
          row_sum = fmaf(row_sum, correction, sum);
          row_max = new_max;
#pragma unroll
          for (int i = 0; i < PAIRS; ++i) {
            acc[i][0] *= correction;
            acc[i][1] *= correction;
          }
          for (unsigned rest = seen; rest != 0u; rest &= rest - 1) {
            const int j = __ffs(rest) - 1;
            const float w = __shfl_sync(0xffffffffu, p, j);
            const int v_page = __shfl_sync(0xffffffffu, page, j);
            const int slot = (key0 + 32 * half + j) % a.page_size;
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
              const int d = 2 * lane + 64 * i;
              if (d >= D) continue;
              const T* v = v_cache + hx_cache_offset(v_page, kv_head, slot, d, a.kv_heads, a.page_size, D, chunk);
              acc[i][0] = fmaf(w, hx_to_float<T>(v[0]), acc[i][0]);
              acc[i][1] = fmaf(w, hx_to_float<T>(v[1]), acc[i][1]);
            }
          }
        }
      }
      const bool whole = c.tile == 0 && count == c.tiles;
      const float inverse = tree_inverse(row_sum);
      T* out = static_cast<T*>(a.out) + static_cast<size_t>(c.q_begin + token) * a.ldo +
               static_cast<size_t>(head) * D;
      float* part = tree_part<ROW_WARPS>(a, blockIdx.x, c.tile == 0);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        const int d = 2 * lane + 64 * i;
        if (d >= D) continue;
        if (whole) {
          out[d] = hx_from_float<T>(acc[i][0] * inverse);
          out[d + 1] = hx_from_float<T>(acc[i][1] * inverse);
        } else {
          *reinterpret_cast<float2*>(part + (static_cast<size_t>(d / 2) * ROW_WARPS + row) * 2) =
              make_float2(acc[i][0], acc[i][1]);
        }
      }
      if (!whole && lane == 0) {
        part[static_cast<size_t>(D) * ROW_WARPS + row] = row_max;
        part[static_cast<size_t>(D + 1) * ROW_WARPS + row] = row_sum;
      }
    }
    left -= count;
    if (left > 0) tree_next_item<ROW_KEYS>(a, c);
    else if (threadIdx.x == 0) tree_tell_cut<ROW_WARPS>(a, run, c, count);
  }
}

// ------------------------------------------------------------------ joining parts

constexpr int JOIN_WARPS = 8, JOIN_THREADS = 32 * JOIN_WARPS;
constexpr int JOIN_FEW = 4;        // parts that a thread joins for many coordinates
constexpr int JOIN_SOME = 32;      // ... and for few
constexpr int JOIN_CTAS = 3;       // an SM

// COUNT coordinates of a row out of some parts: sums against the largest of their maxima.
template <int COUNT>
struct Joined {
  float top = -INFINITY, sum = 0.0f, acc[COUNT] = {};
  __device__ __forceinline__ void add(float m, float l, const float (&o)[COUNT]) {
    // no part, or one whose row saw nothing.  (Scores that are no numbers leave no maximum either, but a sum
    // that is none: it goes on into the row's.)
    if (m == -INFINITY && !(l != l)) return;
    const float new_top = fmaxf(top, m);
    const float keep = exp2f(top - new_top), take = exp2f(m - new_top);
    top = new_top;
    sum = fmaf(sum, keep, l * take);
#pragma unroll
    for (int e = 0; e < COUNT; ++e) acc[e] = fmaf(acc[e], keep, o[e] * take);
  }
};

// Parts [begin, end) of a row's coordinates from COUNT * group on; the loads of LOADS parts are in
// flight together.  A piece (VEC coordinates) behind the last is the last one again.
template <int ROWS, int VEC, int COUNT, int LOADS>
__device__ __forceinline__ Joined<COUNT> join_parts(const TreeArgs& a, int owner, int begin, int end, int row,
                                                    int group) {
  const int D = a.head_dim;
  const long long stride = tree_part_floats<ROWS>(D);
  Joined<COUNT> joined;
  for (int base = begin; base < end; base += LOADS) {
    float m[LOADS], l[LOADS], o[LOADS][COUNT];
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      m[u] = -INFINITY;
      l[u] = 0.0f;
      if (base + u < end) {
        const int index = base + u;
        const float* part = a.partial + (index == 0 ? 2ll * owner + 1 : 2ll * (owner + index)) * stride;
        m[u] = __ldcg(part + D * ROWS + row);
        l[u] = __ldcg(part + (D + 1) * ROWS + row);
#pragma unroll
        for (int p = 0; p < COUNT / VEC; ++p) {
          const float* at = part + (min(group * (COUNT / VEC) + p, D / VEC - 1) * ROWS + row) * VEC;
          if constexpr (VEC == 4) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(at));
            o[u][4 * p] = v.x; o[u][4 * p + 1] = v.y; o[u][4 * p + 2] = v.z; o[u][4 * p + 3] = v.w;
          } else {
            const float2 v = __ldcg(reinterpret_cast<const float2*>(at));
            o[u][2 * p] = v.x; o[u][2 * p + 1] = v.y;
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < LOADS; ++u) joined.add(m[u], l[u], o[u]);
  }
  return joined;
}

template <typename T, int COUNT>
__device__ __forceinline__ void store_joined(const TreeArgs& a, const TreeCut& cut, int row, int group,
                                             const Joined<COUNT>& joined) {
  const float inverse = tree_inverse(joined.sum);
  T* out = static_cast<T*>(a.out) + static_cast<size_t>(cut.token + row / cut.heads) * a.ldo +
           static_cast<size_t>(cut.head0 + row % cut.heads) * a.head_dim + group * COUNT;
  const int here = a.head_dim - group * COUNT;
  // (where whole vectors fit: the tensor cores' kernels see to it that rows are aligned)
  if (sizeof(T) == 2 && COUNT % 4 == 0 && a.head_dim % COUNT == 0 &&
      (reinterpret_cast<uintptr_t>(out) & 7) == 0) {
#pragma unroll
    for (int e = 0; e + 3 < COUNT; e += 4) {
      const __nv_bfloat162 low = __floats2bfloat162_rn(joined.acc[e] * inverse, joined.acc[e + 1] * inverse);
      const __nv_bfloat162 high = __floats2bfloat162_rn(joined.acc[e + 2] * inverse, joined.acc[e + 3] * inverse);
      *reinterpret_cast<uint2*>(out + e) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&low), *reinterpret_cast<const uint32_t*>(&high));
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < COUNT; ++e)
    if (e < here) out[e] = hx_from_float<T>(joined.acc[e] * inverse);
}

// Every block makes lists of the cut items and the blocks share them out.  An item of few parts (there
// are many such items): a thread joins them all, for 16 coordinates of a row, so that maxima and weights
// are read once for them.  One of some more: the same for 4 coordinates, with more parts in flight.
// One of many (a long context of few requests): the warps of a block take runs of the parts.
// Neighbouring lanes have neighbouring rows.  Always joined in ascending order of the keys.
template <typename T, int ROWS, int VEC>
__global__ __launch_bounds__(JOIN_THREADS, JOIN_CTAS) void tree_join_kernel(const TreeArgs a, int ctas) {
  constexpr int WIDE = 16, SLIM = 4;      // coordinates of a thread
  __shared__ short lists[3][TREE_MOST_CTAS];
  __shared__ short parts_of[TREE_MOST_CTAS];
  __shared__ TreeCut cuts[TREE_MOST_CTAS];
  __shared__ int of_warp[3][JOIN_WARPS];
  __shared__ float met[JOIN_WARPS][SLIM + 2][32];
  hx_pdl_prologue();
  const int D = a.head_dim, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int length[3] = {0, 0, 0};
  for (int base = 0; base < ctas; base += JOIN_THREADS) {
    const int owner = base + threadIdx.x;
    int parts = 0;
    if (owner < ctas) {      // (a cut that is none may be anything)
      parts = __ldcg(tree_cut_parts<ROWS>(a, ctas) + owner);
      const int4 cut = __ldcg(reinterpret_cast<const int4*>(tree_cuts<ROWS>(a, ctas) + owner));
      cuts[owner] = TreeCut{cut.x, cut.y, cut.z, cut.w};
      parts_of[owner] = static_cast<short>(parts);
    }
    const int which = parts == 0 ? -1 : parts <= JOIN_FEW ? 0 : parts <= JOIN_SOME ? 1 : 2;
    unsigned mine[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      mine[k] = __ballot_sync(0xffffffffu, which == k);
      if (lane == 0) of_warp[k][warp] = __popc(mine[k]);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      int place = length[k] + __popc(mine[k] & ((1u << lane) - 1));
      for (int w = 0; w < JOIN_WARPS; ++w) {
        if (w < warp) place += of_warp[k][w];
        length[k] += of_warp[k][w];
      }
      if (which == k) lists[k][place] = static_cast<short>(owner);
    }
    __syncthreads();
  }
  const int thread = blockIdx.x * JOIN_THREADS + threadIdx.x, threads = gridDim.x * JOIN_THREADS;
  const int wide_slots = ROWS * ((D + WIDE - 1) / WIDE), groups = (D + SLIM - 1) / SLIM;
  for (int s = thread; s < length[0] * wide_slots; s += threads) {
    const int owner = lists[0][s / wide_slots], at = s % wide_slots, group = at / ROWS, row = at % ROWS;
    const TreeCut cut = cuts[owner];
    if (row < cut.rows)
      store_joined<T, WIDE>(a, cut, row, group,
                            join_parts<ROWS, VEC, WIDE, 2>(a, owner, 0, parts_of[owner], row, group));
  }
  for (int s = thread; s < length[1] * ROWS * groups; s += threads) {
    const int owner = lists[1][s / (ROWS * groups)], at = s % (ROWS * groups), group = at / ROWS, row = at % ROWS;
    const TreeCut cut = cuts[owner];
    if (row < cut.rows)
      store_joined<T, SLIM>(a, cut, row, group,
                            join_parts<ROWS, VEC, SLIM, 8>(a, owner, 0, parts_of[owner], row, group));
  }
  constexpr int LANE_ROWS = ROWS < 32 ? ROWS : 32, LANE_GROUPS = 32 / LANE_ROWS;      // of a warp
  const int units = (ROWS / LANE_ROWS) * ((groups + LANE_GROUPS - 1) / LANE_GROUPS);
  for (int u = blockIdx.x; u < length[2] * units; u += gridDim.x) {
    const int owner = lists[2][u / units], parts = parts_of[owner], unit = u % units;
    const TreeCut cut = cuts[owner];
    const int row = unit % (ROWS / LANE_ROWS) * LANE_ROWS + lane % LANE_ROWS;
    const int group = unit / (ROWS / LANE_ROWS) * LANE_GROUPS + lane / LANE_ROWS;
    const bool mine = row < cut.rows && group < groups;
    Joined<SLIM> joined;
    if (mine)
      joined = join_parts<ROWS, VEC, SLIM, 8>(a, owner, parts * warp / JOIN_WARPS, parts * (warp + 1) / JOIN_WARPS,
                                              row, group);
    met[warp][0][lane] = joined.top;
    met[warp][1][lane] = joined.sum;
#pragma unroll
    for (int e = 0; e < SLIM; ++e) met[warp][2 + e][lane] = joined.acc[e];
    __syncthreads();
    if (warp == 0 && mine) {
      Joined<SLIM> total;
#pragma unroll
      for (int w = 0; w < JOIN_WARPS; ++w) {
        float o[SLIM];
#pragma unroll
        for (int e = 0; e < SLIM; ++e) o[e] = met[w][2 + e][lane];
        total.add(met[w][0][lane], met[w][1][lane], o);
      }
      store_joined<T, SLIM>(a, cut, row, group, total);
    }
    __syncthreads();
  }
}

// CTAs of the tile kernel that an SM has registers and shared memory for: heads of 128 leave three.
int tile_ctas_an_sm(int head_dim) {
  const int most = head_dim <= 128 ? TileConfig<128>::kCtas : TileConfig<256>::kCtas;
  const int fit = 227 * 1024 / (TileConfig<128>::floats(head_dim) * 4 + 1024);
  return fit < most ? fit : most;
}

template <typename T, int D_MAX>
int launch_tile(const TreeArgs& a, int ctas, cudaStream_t stream) {
  const int bytes = TileConfig<D_MAX>::floats(a.head_dim) * 4;
  static std::atomic<unsigned long long> ready{0};
  const bool reserved = hx_once_a_device(ready, [] {
    return cudaFuncSetAttribute(tree_tile_kernel<T, D_MAX>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                TileConfig<D_MAX>::floats(D_MAX) * 4) == cudaSuccess &&
           cudaFuncSetAttribute(tree_tile_kernel<T, D_MAX>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                cudaSharedmemCarveoutMaxShared) == cudaSuccess;
  });
  HX_REQUIRE(reserved, "hx_tree_attention: cannot reserve shared memory");
  hx_launch(tree_tile_kernel<T, D_MAX>, ctas, TILE_WARPS * 32, bytes, stream, a);
  HX_CHECK_LAUNCH("hx_tree_attention");
  return HX_OK;
}

// Up to here the streaming kernel beats the tcgen05 one, whose tile of 128 rows is mostly empty then (32 heads of 128;
// streaming against tcgen05): 64 requests x 8 or 16 drafts behind 1,200 keys 215 and 219 us against 321 and 332, x 32
// drafts 306 to 331 against 345 to 358; 8 requests behind 640 keys 33, 31 and 40 us against 49, 44 and 45; one request, 32 rows
// behind 32,701 keys, 56 against 53 to 58.  It has no tiles of more rows: a warp's 16 rows fill its registers.
constexpr int STREAM_MOST_ROWS = 32;

// Which kernel: the tensor cores', the tile kernel, or the row kernel.
enum TreeKernel { TREE_TC, TREE_TILE, TREE_ROW };
TreeKernel kernel_for(int dtype, int head_dim, int page_size) {
  if (dtype == HX_BF16 && hx_tree_tc_takes(head_dim, page_size)) return TREE_TC;
  if (head_dim % 4 == 0 && head_dim <= 256) return TREE_TILE;
  return TREE_ROW;
}

}  // namespace

int hx_tree_join(const TreeArgs& a, int dtype, int ctas, int rows, int vec, cudaStream_t stream) {
  HX_REQUIRE(ctas <= TREE_MOST_CTAS, "hx_tree_attention: a grid of %d CTAs", ctas);
  const int grid = hx_device_sm_count() * JOIN_CTAS;
  const bool half = dtype == HX_BF16;
  auto run = [&](auto kernel) { hx_launch(kernel, grid, JOIN_THREADS, 0, stream, a, ctas); };
  if (half && rows == 128) run(tree_join_kernel<__nv_bfloat16, 128, 4>);
  else if (half && rows == 32 && vec == 2) run(tree_join_kernel<__nv_bfloat16, 32, 2>);
  else if (half && rows == 16) run(tree_join_kernel<__nv_bfloat16, 16, 2>);
  else if (half && rows == TILE_ROWS) run(tree_join_kernel<__nv_bfloat16, TILE_ROWS, 4>);
  else if (rows == TILE_ROWS) run(tree_join_kernel<float, TILE_ROWS, 4>);
  else if (half) run(tree_join_kernel<__nv_bfloat16, ROW_WARPS, 2>);
  else run(tree_join_kernel<float, ROW_WARPS, 2>);
  HX_CHECK_LAUNCH("hx_tree_attention");
  return HX_OK;
}

// Floats of scratch that hx_tree_attention needs for these sizes, whatever the step brings; negative:
// there is no kernel for them.
HX_API long long hx_tree_attention_scratch_floats(int dtype, int heads, int kv_heads, int head_dim,
                                                  int page_size) {
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || head_dim <= 0 || head_dim % 2 != 0 ||
      head_dim > ROW_MAX_DIM || page_size <= 0 || (dtype != HX_F32 && dtype != HX_BF16))
    return -1;
  const int sms = hx_device_sm_count();
  if (sms <= 0) return -1;
  switch (kernel_for(dtype, head_dim, page_size)) {
    case TREE_TC: {      // (or the streaming kernel, as the trees are)
      const long long tc = hx_tree_tc_floats(head_dim);
      const long long stream = hx_tree_stream_takes(head_dim, page_size) ? hx_tree_stream_floats(head_dim) : 0;
      return tc > stream ? tc : stream;
    }
    case TREE_TILE: return tree_scratch_floats<TILE_ROWS>(head_dim, sms * tile_ctas_an_sm(head_dim));
    default: return tree_scratch_floats<ROW_WARPS>(head_dim, sms * ROW_CTAS);
  }
}

// out[t, h D .. (h + 1) D) for every token t of the requests; see the head of this file.  visible:
// [tokens, ld_visible] of 64-bit words, `words` of them a token, bit j of word w: the token sees
// drafted token 64 w + j of its request.  max_nodes: the most tokens a request brings, which a kernel
// is chosen by (any number gives the right result; 0: not known).  partial: hx_tree_attention_scratch_floats() floats.  Rows of
// `out` behind request_start[requests] are left as they are.
HX_API int hx_tree_attention(const void* q, int ldq, const void* k_cache, const void* v_cache, int dtype,
                             const long long* visible, int ld_visible, int words,
                             const int* request_start, const int* request_context,
                             const int* request_table_row, const int* block_tables, int table_stride,
                             void* out, int ldo, float* partial, int requests, int heads, int kv_heads,
                             int head_dim, int page_size, int num_pages, float scale, int max_nodes,
                             int* status, cudaStream_t stream) {
  HX_REQUIRE(dtype == HX_F32 || dtype == HX_BF16, "hx_tree_attention: unknown dtype %d", dtype);
  HX_REQUIRE(requests >= 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && page_size > 0,
             "hx_tree_attention: bad sizes");
  HX_REQUIRE(head_dim > 0 && head_dim % 2 == 0 && head_dim <= ROW_MAX_DIM,
             "hx_tree_attention: head_dim %d (even, at most %d)", head_dim, ROW_MAX_DIM);
  HX_REQUIRE(words > 0 && ld_visible >= words, "hx_tree_attention: a token has at least one word of 64 bits");
  HX_REQUIRE(num_pages > 0 && table_stride > 0 && static_cast<long long>(num_pages) * kv_heads < (1ll << 31),
             "hx_tree_attention: bad cache geometry");
  HX_REQUIRE(scale > 0.0f && scale <= 3.0e38f, "hx_tree_attention: the scale must be positive and finite");
  HX_REQUIRE(status != nullptr && partial != nullptr, "hx_tree_attention: status word or scratch missing");
  const int size = dtype == HX_BF16 ? 2 : 4;
  const int piece = hx_cache_chunk(size, head_dim) * size;      // bytes the cache is read in
  auto aligned = [](const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; };
  HX_REQUIRE(aligned(k_cache, piece) && aligned(v_cache, piece) && aligned(partial, 16) && aligned(visible, 8),
             "hx_tree_attention: cache, scratch or masks are not aligned");
  if (requests == 0) return HX_OK;
  TreeArgs a{q, ldq, k_cache, v_cache, visible, ld_visible, words, request_start, request_context,
             request_table_row, block_tables, table_stride, out, ldo, partial, requests, heads, kv_heads,
             head_dim, page_size, num_pages, scale, status, 1, 1, 1};
  const TreeKernel kernel = kernel_for(dtype, head_dim, page_size);
  const int sms = hx_device_sm_count();
  HX_REQUIRE(sms > 0, "hx_tree_attention: the device cannot be asked");
  if (kernel == TREE_TC) {
    HX_REQUIRE(ldq % 8 == 0 && ldo % 8 == 0 && aligned(q, 16) && aligned(out, 16),
               "hx_tree_attention: q and out must be 16-byte aligned, row strides multiples of 8");
    const long long rows = static_cast<long long>(max_nodes) * (heads / kv_heads);
    if (hx_tree_stream_takes(head_dim, page_size) && rows > 0 && rows <= STREAM_MOST_ROWS)
      return hx_tree_stream_launch(a, static_cast<int>(rows), stream);
    return hx_tree_tc_launch(a, stream);
  }
  if (kernel == TREE_TILE) {
    HX_REQUIRE(ldq % 4 == 0 && aligned(q, 4 * size), "hx_tree_attention: q must be aligned to four elements");
    tree_fill_rows(a, TILE_ROWS);
    const int ctas = sms * tile_ctas_an_sm(head_dim);
    int rc;
    if (dtype == HX_BF16)
      rc = head_dim <= 128 ? launch_tile<__nv_bfloat16, 128>(a, ctas, stream)
                           : launch_tile<__nv_bfloat16, 256>(a, ctas, stream);
    else
      rc = head_dim <= 128 ? launch_tile<float, 128>(a, ctas, stream) : launch_tile<float, 256>(a, ctas, stream);
    if (rc != HX_OK) return rc;
    return hx_tree_join(a, dtype, ctas, TILE_ROWS, 4, stream);
  }
  tree_fill_rows(a, ROW_WARPS);
  const int ctas = sms * ROW_CTAS;
  if (dtype == HX_BF16) hx_launch(tree_row_kernel<__nv_bfloat16>, ctas, ROW_WARPS * 32, 0, stream, a);
  else hx_launch(tree_row_kernel<float>, ctas, ROW_WARPS * 32, 0, stream, a);
  HX_CHECK_LAUNCH("hx_tree_attention");
  return hx_tree_join(a, dtype, ctas, ROW_WARPS, 2, stream);
}
