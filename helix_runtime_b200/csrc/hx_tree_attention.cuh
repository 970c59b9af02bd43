// What the kernels of tree attention share: their arguments, how the work is cut into equal runs,
// which keys a token sees, and where a run leaves the parts of rows that it did not finish.
//
// The work.  A request's drafted tokens and the query heads of a key/value head (in groups, where they
// are more than a tile has rows) make up rows, token by token; `tile_tokens` tokens fill a tile of rows.  An ITEM is one tile of rows against
// one key/value head: it walks all the keys of its request, cached and drafted, in tiles of `keys`
// anchored at key 0.  The key tiles of all items lie end to end in one list (requests in order;
// in a request key/value heads in order and under each its tiles of rows, so that CTAs which read
// the same keys do so at about the same time), and every CTA of a grid that fills the GPU once takes an
// equal run of that list, whatever the mix of lengths.  An item inside a run is finished by its
// CTA; one that is cut by run borders leaves parts (unnormalised sums, maxima, weights) in the
// caller's scratch, at most two a CTA, which a second kernel joins in ascending order.  Nothing in
// the scratch outlives the call and nothing in it has to be zero.
#pragma once

#include "hx_common.cuh"

struct TreeArgs {
  const void* q;
  int ldq;
  const void* k_cache;
  const void* v_cache;
  const long long* visible;     // [tokens, ld_visible] bit j of a token's words: it sees token j of its request
  int ld_visible;
  int words;                    // words a token has
  const int* request_start;     // [requests + 1] first token of each request
  const int* request_context;   // [requests] cached keys in front of the tree: seen by every token
  const int* request_table_row;
  const int* block_tables;
  int table_stride;
  void* out;
  int ldo;
  float* partial;
  int requests;
  int heads;
  int kv_heads;
  int head_dim;
  int page_size;
  int num_pages;
  float scale;
  int* status;
  int group;                    // query heads of a key/value head that an item takes at most
  int groups;                   // groups of them a key/value head
  int tile_tokens;              // tokens whose heads fill a tile of rows
};

namespace {

constexpr float HX_LOG2E = 1.4426950408889634f;

// An item of the list and a key tile of it; every field is the same in all threads that hold it.
struct TreeCursor {
  int request, item, items;     // item: (kv_head * groups + group) * row_tiles + row_tile
  int tile, tiles;              // key tiles
  int row_tiles;
  int q_begin, nodes, context;

  __device__ __forceinline__ int kv_head(const TreeArgs& a) const { return item / row_tiles / a.groups; }
};

// An item's rows: row r is query head head0 + r % heads of drafted token token0 + r / heads.
struct TreeRows {
  int kv_head, head0, heads, token0, count;
  __device__ __forceinline__ TreeRows(const TreeArgs& a, const TreeCursor& c) {
    const int slot = c.item / c.row_tiles, of_kv = a.heads / a.kv_heads;
    kv_head = slot / a.groups;
    const int first = (slot - kv_head * a.groups) * a.group;
    head0 = kv_head * of_kv + first;
    heads = min(a.group, of_kv - first);
    token0 = (c.item - slot * c.row_tiles) * a.tile_tokens;
    count = min(a.tile_tokens, c.nodes - token0) * heads;
  }
};

// Sizes of a request: key tiles of an item in `tiles`, 0 where it brings no token.
template <int KEYS>
__device__ __forceinline__ void tree_request(const TreeArgs& a, int request, TreeCursor& c) {
  c.request = request;
  c.q_begin = a.request_start[request];
  c.nodes = a.request_start[request + 1] - c.q_begin;
  c.context = max(a.request_context[request], 0);
  c.row_tiles = (max(c.nodes, 0) + a.tile_tokens - 1) / a.tile_tokens;
  c.items = c.row_tiles * a.kv_heads * a.groups;
  c.tiles = c.nodes > 0 ? (c.context + c.nodes + KEYS - 1) / KEYS : 0;
}

// Key tiles of all items of the list; every lane of a converged warp gets the sum.
template <int KEYS>
__device__ __forceinline__ long long tree_total(const TreeArgs& a) {
  const int lane = threadIdx.x & 31;
  long long mine = 0;
  for (int r = lane; r < a.requests; r += 32) {
    TreeCursor c;
    tree_request<KEYS>(a, r, c);
    mine += static_cast<long long>(c.items) * c.tiles;
  }
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, offset);
  return mine;
}

// The item and key tile at place `at` of the list (0 <= at < total).  Called by a converged warp.
template <int KEYS>
__device__ __forceinline__ void tree_locate(const TreeArgs& a, long long at, TreeCursor& c) {
  const int lane = threadIdx.x & 31;
  long long before = 0;
  int found = -1;
  for (int base = 0; base < a.requests && found < 0; base += 32) {
    long long work = 0;
    if (base + lane < a.requests) {
      tree_request<KEYS>(a, base + lane, c);
      work = static_cast<long long>(c.items) * c.tiles;
    }
    long long inclusive = work;
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1) {
      const long long other = __shfl_up_sync(0xffffffffu, inclusive, offset);
      if (lane >= offset) inclusive += other;
    }
    const unsigned beyond = __ballot_sync(0xffffffffu, before + inclusive > at);
    if (beyond != 0u) {
      const int source = __ffs(beyond) - 1;
      found = base + source;
      before += __shfl_sync(0xffffffffu, inclusive - work, source);
    } else {
      before += __shfl_sync(0xffffffffu, inclusive, 31);
    }
  }
  tree_request<KEYS>(a, max(found, 0), c);
  const long long inside = at - before;
  c.item = static_cast<int>(inside / c.tiles);
  c.tile = static_cast<int>(inside - static_cast<long long>(c.item) * c.tiles);
}

// On to the next item (there is one: callers count the tiles that are left to them).
template <int KEYS>
__device__ __forceinline__ void tree_next_item(const TreeArgs& a, TreeCursor& c) {
  c.tile = 0;
  if (++c.item < c.items) return;
  c.item = 0;
  int request = c.request;
  do {
    ++request;
    if (request >= a.requests) return;
    tree_request<KEYS>(a, request, c);
  } while (c.tiles == 0);
}

// Bounded wait: false when the limit ran out (some seconds).  A poll may sleep for 16 us: without that
// time the waiting warps of a tcgen05 CTA issued ten times the instructions of those that work, and
// held them up.
__device__ __forceinline__ bool tree_wait(uint64_t* bar, uint32_t parity) {
  const uint32_t address = static_cast<uint32_t>(__cvta_generic_to_shared(bar));
  for (uint32_t poll = 0; poll < 400u * 1000u; ++poll) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(address), "r"(parity), "r"(16u * 1024u)
        : "memory");
    if (done) return true;
  }
  return false;
}

// One over a row's sum of weights; a row that saw nothing becomes zeros, one whose scores are no numbers stays none.
__device__ __forceinline__ float tree_inverse(float sum) { return sum == 0.0f ? 0.0f : 1.0f / sum; }

// A CTA's run of the list.  Runs are at least `least` tiles long, so that a short list does not
// become more parts than it is worth.
struct TreeRun {
  long long begin, per_cta, total;
  int count;
};

// What the join needs to know of the item that begins in a CTA's run and goes on behind it.
struct alignas(16) TreeCut {
  int token, head0;      // the row of `out` and the head of row 0
  int heads, rows;       // heads a token, rows
};
constexpr int TREE_MOST_CTAS = 1024;
template <int KEYS>
__device__ __forceinline__ TreeRun tree_run(const TreeArgs& a, int cta, int ctas, int least) {
  TreeRun run;
  run.total = tree_total<KEYS>(a);
  run.per_cta = (run.total + ctas - 1) / ctas;
  if (run.per_cta < least) run.per_cta = least;
  run.begin = cta * run.per_cta;
  const long long rest = run.total - run.begin;
  run.count = rest <= 0 ? 0 : static_cast<int>(rest < run.per_cta ? rest : run.per_cta);
  return run;
}

// Which of the 64 keys from key0 on does a drafted token of the cursor's request see?  Bit i is key
// key0 + i: a cached key, or a drafted one whose bit is set.  `first_word`: the first of the token's
// words; `word_at` gives the others.
template <typename Words>
__device__ __forceinline__ unsigned long long tree_mask_of(const TreeArgs& a, const TreeCursor& c, int key0,
                                                           unsigned long long first_word, Words word_at) {
  const int cached = c.context - key0;      // of the tile's keys, so many are cached ones
  if (cached >= 64) return ~0ull;
  unsigned long long mask;
  if (cached >= 0) {
    mask = first_word << cached;
    if (cached > 0) mask |= (1ull << cached) - 1;
  } else {
    const int first = -cached, word = first >> 6, shift = first & 63;
    mask = word == 0 ? first_word >> shift : word < a.words ? word_at(word) >> shift : 0ull;
    // (words behind the last token's say nothing)
    if (shift > 0 && word + 1 < a.words && 64 * (word + 1) < c.nodes) mask |= word_at(word + 1) << (64 - shift);
  }
  const int there = cached + c.nodes;       // keys of the tile that exist
  if (there < 64) mask &= there > 0 ? (1ull << there) - 1 : 0ull;
  return mask;
}
__device__ __forceinline__ const unsigned long long* tree_words(const TreeArgs& a, const TreeCursor& c, int token) {
  return reinterpret_cast<const unsigned long long*>(a.visible) + static_cast<size_t>(c.q_begin + token) * a.ld_visible;
}
__device__ __forceinline__ unsigned long long tree_mask(const TreeArgs& a, const TreeCursor& c, int token, int key0) {
  if (c.context - key0 >= 64) return ~0ull;
  const unsigned long long* words = tree_words(a, c, token);
  return tree_mask_of(a, c, key0, words[0], [&](int word) { return words[word]; });
}

// How the heads of a key/value head and the tokens fill tiles of `rows` rows.
inline void tree_fill_rows(TreeArgs& a, int rows) {
  const int of_kv = a.heads / a.kv_heads;
  a.group = of_kv < rows ? of_kv : rows;
  a.groups = (of_kv + a.group - 1) / a.group;
  a.tile_tokens = rows / a.group;
}

// A part of an item: VEC coordinates of a row side by side, [head_dim / VEC][ROWS][VEC], then the
// rows' maxima (log2 units of the scaled scores) and weights.
template <int ROWS>
__host__ __device__ constexpr long long tree_part_floats(int head_dim) {
  return static_cast<long long>(ROWS) * (head_dim + 2);
}
// The scratch: two parts a CTA, behind them what each says about its cut item and, last, how many parts
// that item has (0: there is none).
template <int ROWS>
__host__ __device__ constexpr long long tree_scratch_floats(int head_dim, int ctas) {
  return ctas * (2 * tree_part_floats<ROWS>(head_dim) + static_cast<long long>(sizeof(TreeCut) / 4) + 1);
}
template <int ROWS>
__device__ __forceinline__ TreeCut* tree_cuts(const TreeArgs& a, int ctas) {
  return reinterpret_cast<TreeCut*>(a.partial + ctas * 2 * tree_part_floats<ROWS>(a.head_dim));
}
template <int ROWS>
__device__ __forceinline__ int* tree_cut_parts(const TreeArgs& a, int ctas) {
  return reinterpret_cast<int*>(tree_cuts<ROWS>(a, ctas) + ctas);
}
template <int ROWS>
__device__ __forceinline__ float* tree_part(const TreeArgs& a, int cta, bool item_begins) {
  return a.partial + (2ll * cta + (item_begins ? 1 : 0)) * tree_part_floats<ROWS>(a.head_dim);
}

// One thread says that the CTA's run leaves nothing to the join: first of all, so that it holds
// whatever comes between, ...
template <int ROWS>
__device__ __forceinline__ void tree_tell_none(const TreeArgs& a) {
  tree_cut_parts<ROWS>(a, gridDim.x)[blockIdx.x] = 0;
}
// ... and at the run's end what it does leave, looked at from the last segment.
template <int ROWS>
__device__ __forceinline__ void tree_tell_cut(const TreeArgs& a, const TreeRun& run, const TreeCursor& last,
                                              int last_count) {
  if (last.tile != 0 || last_count == last.tiles) return;
  const TreeRows rows(a, last);
  const long long item_end = run.begin + run.count - last_count + last.tiles;
  tree_cuts<ROWS>(a, gridDim.x)[blockIdx.x] = TreeCut{last.q_begin + rows.token0, rows.head0, rows.heads, rows.count};
  tree_cut_parts<ROWS>(a, gridDim.x)[blockIdx.x] =
      static_cast<int>((item_end - 1) / run.per_cta) - static_cast<int>(blockIdx.x) + 1;
}

}  // namespace

// Joins the parts that `ctas` CTAs of tiles of `rows` rows left (`vec` coordinates side by side), on the
// same stream behind them.
int hx_tree_join(const TreeArgs& a, int dtype, int ctas, int rows, int vec, cudaStream_t stream);

// The tcgen05 kernel (bfloat16): whether it takes these sizes, its scratch, its launch.
bool hx_tree_tc_takes(int head_dim, int page_size);
long long hx_tree_tc_floats(int head_dim);
int hx_tree_tc_launch(TreeArgs a, cudaStream_t stream);

// The streaming kernel (bfloat16), tiles of 16 or 32 rows; `rows`: of the largest tree.
bool hx_tree_stream_takes(int head_dim, int page_size);
long long hx_tree_stream_floats(int head_dim);
int hx_tree_stream_launch(TreeArgs a, int rows, cudaStream_t stream);
