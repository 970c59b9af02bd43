// Tree attention on the 5th-generation tensor cores (tcgen05), bfloat16 storage; what it computes and
// how the work is cut into runs is told in hx_tree_attention.cu and hx_tree_attention.cuh.
//
// A tile of 128 rows (the M of a product) holds the drafted tokens of a request, each with the
// query heads of one key/value head; the item walks its keys 64 at a time.  Warp roles:
//   warp 0      asks for keys and values, a whole (page, head) block a copy (see below);
//   warp 1      one lane issues S = Q K^T into one of two score buffers in tensor memory;
//   warp 2      one lane issues O += P V;
//   warp 3      loads the queries of an item, as soon as the item before has read its own;
//   warps 4-11  softmax: two threads own a row, one the first 32 scores of a tile, the other the last 32 (with one
//               thread a row the softmax took 2,000 cycles a tile, a chain of instructions that no
//               product or copy was long enough to hide: 64 requests x 64 drafts 405 us).  They tell each other their
//               maxima, so both keep the same reference.  P goes back
//               over the scores they have read as two bfloat16 terms (hi + lo, 16 bits of each weight, as in
//               the kernels of prompts and single tokens: one term alone is 2^-8 of each weight off, as much again as the
//               output's rounding).  They fill the score buffer, also the columns that the maxima are told
//               through, so the low terms wait until the other thread has read.  P is the A
//               operand of O += P V straight from tensor memory; the reference of the exponentials is
//               raised when a tile exceeds it by more than 2^8, O stays in tensor memory.
// Keys and values keep flowing across items: the rings go by TURNS, the key tiles of the CTA's run in
// order.  Two CTAs share an SM and fill each other's gaps.
//
// Operands as they land.  A block of the cache is [piece][slot][16 bytes], so eight slots of a piece
// are a core matrix (8 rows x 16 bytes) of an operand that is not swizzled.  What a product's descriptor
// wants is one stride from eight keys to the next eight.  Pages of 64: 128 bytes.  Pages of 32: two
// products of 32 keys.  Pages of 8: the stride is the block's size.  Pages of 16: the first eight
// slots of the four pages lie a block apart, and so do the second eight: two products of 32 keys,
// whose scores stand in that order, column 32 a + 8 p + s for key 16 p + 8 a + s.  The output product
// takes 16 columns at a time, eight keys each of two pages, again a block apart.  (Copying keys piece by
// piece into one stride instead took a copy of 256 bytes 80 cycles of the warp that asks, 6,500 cycles a tile.)
//
// Masks matter in the tiles that hold drafted keys, the last one or two of an item.  There values
// are looked at, too: a probability of zero does not stop one that is not finite (0 x infinity), be it a
// drafted one that other rows see or what a page holds behind the last key.  Such a value is taken as zero
// in the product; a drafted one is added, as what it is, to the rows that do see it.
//
// Measured (32 heads of 128): one request x 64 drafts behind 32,701 keys, 4 query heads a key/value head, 85 to 91 us, 380
// to 400 TFLOP/s: scores, softmax and output product of a tile are one behind the other, 2,900 cycles a tile and SM with two
// CTAs an SM (the tensor pipe is active 30 % of the time); tensor memory has no room for a third.  64 requests x 64 drafts behind
// 1,200 keys, as many key/value heads, 376 to 390 us, 3.4 TB/s.  With one term of a weight these took 78 and 333 us.
//
// Every wait is bounded; a wait that runs out sets a status bit, the CTA lets its copies land, frees its
// tensor memory and returns.
#include "hx_mma.cuh"
#include "hx_tcgen05.cuh"
#include "hx_tree_attention.cuh"

namespace {

constexpr int BLOCK_M = 128, BLOCK_N = 64;
constexpr int WARP_PAGES = 0, WARP_SCORES = 1, WARP_OUTPUT = 2, WARP_QUERIES = 3;      // and 4 to 11: softmax
constexpr int THREADS = 384;
constexpr int GROUP_STRIDE = 128;             // bytes from one 8-row core matrix to the next row group
constexpr int CHUNK_STRIDE = BLOCK_M * 16;    // bytes from one 16-byte column of Q to the next
constexpr float RAISE_MAXIMUM_BY = 8.0f;      // log2 units a tile must exceed a row's reference by
constexpr int CTAS_AN_SM = 2;
constexpr int LEAST = 2;                      // key tiles of the shortest run

template <int D>
struct TreeTcConfig {
  static constexpr int kKeyStages = 3, kValueStages = 2;
  static constexpr int kQBytes = BLOCK_M * D * 2;
  static constexpr int kHalfBytes = BLOCK_N * D * 2;          // keys (or values) of a tile
  static constexpr int kBarrierBytes = 256;
  static constexpr int kSmemBytes = kQBytes + (kKeyStages + kValueStages) * kHalfBytes + 128 + kBarrierBytes;
  static constexpr int kOutputColumn = 2 * BLOCK_N;
  static constexpr int kTmemColumns = 256;
  static_assert(2 * BLOCK_N + D <= kTmemColumns, "tensor memory of a CTA");
  static_assert(CTAS_AN_SM * (kSmemBytes + 1024) <= 228 * 1024, "an SM has 228 KB of shared memory");
};

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two float32 operations in one instruction, and the largest of three: the softmax is bound by the
// instructions it issues.
__device__ __forceinline__ uint64_t pair_of(float low, float high) {
  uint64_t pair;
  asm("mov.b64 %0, {%1, %2};" : "=l"(pair) : "f"(low), "f"(high));
  return pair;
}
__device__ __forceinline__ void halves_of(uint64_t pair, float& low, float& high) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(low), "=f"(high) : "l"(pair));
}
__device__ __forceinline__ uint64_t pair_fma(uint64_t x, uint64_t y, uint64_t z) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return r;
}
__device__ __forceinline__ uint64_t pair_add(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
__device__ __forceinline__ float max_of_3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float low, float high) {
  const __nv_bfloat162 pair = __floats2bfloat162_rn(low, high);
  return *reinterpret_cast<const uint32_t*>(&pair);
}
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
      ::"r"(dst), "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}
// A number of this thread's lane to and from a column of tensor memory.
__device__ __forceinline__ void tmem_store1(uint32_t address, float value) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(address), "r"(__float_as_uint(value)) : "memory");
}
__device__ __forceinline__ float tmem_load1(uint32_t address) {
  uint32_t value;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(value) : "r"(address) : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  return __uint_as_float(value);
}
// All ones in those of two bfloat16 that are infinite or not a number (all ones in the exponent).
__device__ __forceinline__ uint32_t exponents_of(uint32_t pair) { return __vcmpeq2(pair & 0x7f807f80u, 0x7f807f80u); }

// What is not finite among the drafted values that a row sees in the segment [c.tile, c.tile + count) is
// added to the row as stored: whatever their weight, the sum is not finite either.
template <int D>
__device__ __noinline__ void add_not_finite(const TreeArgs& a, TreeCursor c, int count, int token, int row, int half,
                                            __nv_bfloat16* out, float* part) {
  const int first = max(c.context, c.tile * BLOCK_N);
  const int end = min(c.context + c.nodes, (c.tile + count) * BLOCK_N);
  const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(a.v_cache);
  for (int key = first; key < end; ++key) {
    if (!(tree_mask(a, c, token, key / BLOCK_N * BLOCK_N) >> (key % BLOCK_N) & 1)) continue;
    const int index = key / a.page_size;
    if (index >= a.table_stride) continue;
    const int page = a.block_tables[static_cast<size_t>(a.request_table_row[c.request]) * a.table_stride + index];
    if (page < 0 || page >= a.num_pages) continue;
    for (int d = 0; d < D; ++d) {
      if ((d / 16) % 2 != half) continue;      // (another thread's)
      const float x = __bfloat162float(v[hx_cache_offset(page, c.kv_head(a), key % a.page_size, d, a.kv_heads,
                                                         a.page_size, D, 8)]);
      if (isfinite(x)) continue;
      if (out != nullptr) out[d] = __float2bfloat16_rn(__bfloat162float(out[d]) + x);
      else part[(static_cast<size_t>(d / 4) * BLOCK_M + row) * 4 + d % 4] += x;
    }
  }
}

template <int D>
__global__ __launch_bounds__(THREADS, CTAS_AN_SM) void tree_attention_tc_kernel(
    const __grid_constant__ TreeArgs a) {
  using Config = TreeTcConfig<D>;
  constexpr int K_STAGES = Config::kKeyStages, V_STAGES = Config::kValueStages;
  constexpr int PIECES = D / 8;

  // the run is found from the step's description, which was there before the kernel in front
  const TreeRun run = tree_run<BLOCK_N>(a, blockIdx.x, gridDim.x, LEAST);
  TreeCursor at;
  if (run.count == 0) {      // before any barrier or allocation: the whole CTA leaves
    hx_pdl_wait();
    if (threadIdx.x == 0) tree_tell_none<BLOCK_M>(a);
    return;
  }
  tree_locate<BLOCK_N>(a, run.begin, at);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~static_cast<uintptr_t>(127));
  uint8_t* q_tile = smem;
  uint8_t* k_stages = q_tile + Config::kQBytes;
  uint8_t* v_stages = k_stages + K_STAGES * Config::kHalfBytes;
  uint64_t* k_full = reinterpret_cast<uint64_t*>(v_stages + V_STAGES * Config::kHalfBytes);
  uint64_t* k_done = k_full + K_STAGES;        // its scores have read them
  uint64_t* v_full = k_done + K_STAGES;
  uint64_t* v_done = v_full + V_STAGES;
  uint64_t* s_full = v_done + V_STAGES;        // [2] scores of turn t in buffer t % 2
  uint64_t* p_full = s_full + 2;               // [2] its probabilities are in place
  uint64_t* o_full = p_full + 2;               // [2] its output product is done
  uint64_t* q_ready = o_full + 2;              // the queries of a segment are in shared memory
  uint64_t* q_done = q_ready + 1;              // the last score product of a segment has read them
  uint64_t* met = q_done + 1;                  // [4] both softmax warps of 32 rows have told
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(met + 4);
  volatile int* failed = reinterpret_cast<volatile int*>(tmem_holder + 1);
  // [2] the last even and the last odd segment with a drafted value that is not finite.  (A warp without rows may
  // already look at the first tiles of segment n + 1 while others write rows of segment n, but comes no
  // further: their probabilities of n + 1 are wanted for its products.)
  volatile int* poisoned = failed + 1;
  static_assert((2 * K_STAGES + 2 * V_STAGES + 12) * 8 + 16 <= Config::kBarrierBytes, "the place of barriers and flags");

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int page_size = a.page_size;
  const int pages_per_tile = BLOCK_N / page_size;
  const int page_shift = __ffs(page_size) - 1;      // (pages of 8, 16, 32 or 64)
  const uint32_t page_bytes = static_cast<uint32_t>(page_size) * D * 2;
  const uint32_t piece_stride = static_cast<uint32_t>(page_size) * 16;   // next 16-byte piece of a key

  if (threadIdx.x == 0) {
    for (int s = 0; s < K_STAGES; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_done[s], 1);
    }
    for (int s = 0; s < V_STAGES; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_done[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&s_full[b], 1);
      mbar_init(&p_full[b], 8);   // one arrival per softmax warp
      mbar_init(&o_full[b], 1);
    }
    mbar_init(q_ready, 1);
    mbar_init(q_done, 1);
    for (int quarter = 0; quarter < 4; ++quarter) mbar_init(&met[quarter], 2);
    *failed = 0;
    poisoned[0] = poisoned[1] = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == WARP_SCORES) {
    tmem_alloc(tmem_holder, Config::kTmemColumns);
    // Only now may the kernel behind come in: it could else take the tensor memory that this one still
    // waits for, and hold it until this one is done.
    hx_pdl_trigger();
  }
  hx_pdl_wait();
  if (threadIdx.x == 0) tree_tell_none<BLOCK_M>(a);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;

  // One lane waits and looks at the failure flag, all lanes get the same answer.
  auto wait_for = [&](uint64_t* bar, uint32_t parity) {
    int state = 0;      // 0: go on, 1: this wait ran out, 2: somebody else failed
    if (lane == 0) state = *failed ? 2 : (tree_wait(bar, parity & 1u) ? 0 : 1);
    state = __shfl_sync(0xffffffffu, state, 0);
    if (state == 1 && lane == 0) {
      atomicOr(a.status, HX_FLAG_WAIT_TIMEOUT);
      *failed = 1;
    }
    return state == 0;
  };

  if (warp == WARP_PAGES) {
    // ------------------------------------------------------------ page requests
    auto request_values = [&](int turn, long long block) {
      const int stage = turn % V_STAGES;
      if (!wait_for(&v_done[stage], static_cast<uint32_t>(turn / V_STAGES) + 1u)) return false;
      const unsigned there = __ballot_sync(0xffffffffu, block >= 0);
      if (lane == 0) mbar_expect_tx(&v_full[stage], __popc(there) * page_bytes);
      __syncwarp();
      if (block >= 0)
        bulk_copy(smem_u32(v_stages + stage * Config::kHalfBytes) + lane * page_bytes,
                  static_cast<const uint8_t*>(a.v_cache) + block, page_bytes, &v_full[stage]);
      return true;
    };
    // Turn t asks for the keys of turn t and for the values of turn t - 1, which are wanted later.
    // Lane p < pages_per_tile holds the block (of bytes into the layer's cache) of the turn's page p,
    // -1 where there is none.  Page numbers are read 32 at a time, the next 32 while these are used, and the
    // first of the next item while this one's are (a read at each turn held the copies up: 2,400 cycles a tile).
    TreeCursor c = at;
    int asked = 0, keys_asked = 0;      // key tiles whose copies are on their way
    auto table_of = [&](const TreeCursor& of) {
      return a.block_tables + static_cast<size_t>(a.request_table_row[of.request]) * a.table_stride;
    };
    auto pages_from = [&](const int* table, const TreeCursor& of, int first) {
      const int index = first + lane;
      return index < a.table_stride && index * page_size < of.context + of.nodes ? table[index] : -1;
    };
    const uint8_t* k_cache = static_cast<const uint8_t*>(a.k_cache);
    const int* table = table_of(c);
    int pages = pages_from(table, c, c.tile * pages_per_tile / 32 * 32);
    long long value_block = -1;
    int turn = 0, left = run.count;
    bool going = true;
    while (left > 0 && going) {
      const int count = min(c.tiles - c.tile, left);
      TreeCursor next = c;
      const int* next_table = table;
      int next_item_pages = -1;
      if (left > count) {
        tree_next_item<BLOCK_N>(a, next);
        if (next.request != c.request) next_table = table_of(next);
        next_item_pages = pages_from(next_table, next, 0);
      }
      int window = c.tile * pages_per_tile / 32 * 32;
      int next_pages = pages_from(table, c, window + 32);
      const long long kv_head = c.kv_head(a);
      for (int t = 0; t < count; ++t, ++turn) {
        const int index = (c.tile + t) * pages_per_tile;      // of the tile's first page
        if (index - window >= 32) {
          window += 32;
          pages = next_pages;
          next_pages = pages_from(table, c, window + 32);
        }
        const int page = __shfl_sync(0xffffffffu, pages, (index - window + lane) & 31);
        long long block = -1;
        if (lane < pages_per_tile && (index + lane) * page_size < c.context + c.nodes) {
          if (page >= 0 && page < a.num_pages) block = (page * static_cast<long long>(a.kv_heads) + kv_head) * page_bytes;
          else atomicOr(a.status, HX_FLAG_BAD_PAGE);
        }
        const int stage = turn % K_STAGES;
        going = wait_for(&k_done[stage], static_cast<uint32_t>(turn / K_STAGES) + 1u);
        if (!going) break;
        const unsigned there = __ballot_sync(0xffffffffu, block >= 0);
        if (lane == 0) mbar_expect_tx(&k_full[stage], __popc(there) * page_bytes);
        __syncwarp();
        if (block >= 0)
          bulk_copy(smem_u32(k_stages + stage * Config::kHalfBytes) + lane * page_bytes, k_cache + block, page_bytes,
                    &k_full[stage]);
        ++keys_asked;
        if (turn > 0) {
          going = request_values(turn - 1, value_block);
          if (!going) break;
          ++asked;
        }
        value_block = block;
      }
      left -= count;
      c = next;
      table = next_table;
      pages = next_item_pages;
    }
    if (going && request_values(turn - 1, value_block)) ++asked;
    // a CTA does not leave while copies into its shared memory are in flight
    if (*failed) {
      for (int t = max(0, keys_asked - K_STAGES); t < keys_asked; ++t)
        if (lane == 0) tree_wait(&k_full[t % K_STAGES], static_cast<uint32_t>(t / K_STAGES) & 1u);
      for (int t = max(0, asked - V_STAGES); t < asked; ++t)
        if (lane == 0) tree_wait(&v_full[t % V_STAGES], static_cast<uint32_t>(t / V_STAGES) & 1u);
      __syncwarp();
    }
  } else if (warp == WARP_QUERIES) {
    // ------------------------------------------------------------------ queries
    // [D / 8 pieces][16 row groups][8 rows][16 bytes]; rows behind the last keep what lay there (a row's
    // scores concern no other row)
    // (q_done has a phase a segment: a barrier that completes one a turn would have to be waited for
    // turn by turn, a parity says nothing about phases further back)
    TreeCursor c = at;
    int segment = 0;
    for (int left = run.count; left > 0; ++segment) {
      const int count = min(c.tiles - c.tile, left);
      if (segment > 0 && !wait_for(q_done, static_cast<uint32_t>(segment - 1))) break;
      const TreeRows rows(a, c);
      const int rows_here = rows.count;
      const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) +
                               static_cast<size_t>(c.q_begin + rows.token0) * a.ldq + static_cast<size_t>(rows.head0) * D;
      // (asynchronous copies: all of a lane's are in flight together, without registers.  Eight at a time
      // through registers took 25,000 cycles for 128 rows; one division a copy another 500 each)
#pragma unroll 2
      for (int row_group = 0; row_group * 8 < rows_here; ++row_group) {
        const int row = row_group * 8 + (lane & 7), token = row / rows.heads;
        const bool there = row < rows_here;
        const __nv_bfloat16* from =
            there ? q + static_cast<size_t>(token) * a.ldq + static_cast<size_t>(row - token * rows.heads) * D : q;
        const uint32_t target = smem_u32(q_tile + row_group * GROUP_STRIDE + (lane & 7) * 16);
#pragma unroll
        for (int j = 0; j < (PIECES + 3) / 4; ++j) {
          const int piece = 4 * j + (lane >> 3);
          if (piece < PIECES) hx_cp_async_16(target + piece * CHUNK_STRIDE, from + piece * 8, there ? 16 : 0);
        }
      }
      hx_cp_async_commit();
      hx_cp_async_wait<0>();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);
      left -= count;
      if (left > 0) tree_next_item<BLOCK_N>(a, c);
    }
  } else if (warp == WARP_SCORES) {
    // ------------------------------------------------------------ score products
    if (hx_elect_one()) {
      // pages of 16 and 32: two products of 32 keys, the second `apart` bytes on
      const bool halves = page_size == 16 || page_size == 32;
      const uint32_t idesc = halves ? make_idesc(BLOCK_M, BLOCK_N / 2) : make_idesc(BLOCK_M, BLOCK_N);
      const uint32_t apart = (page_size == 16 ? GROUP_STRIDE : page_bytes) >> 4;
      const uint32_t key_step = (2 * piece_stride) >> 4;      // 16 coordinates on
      const uint64_t desc_q = make_smem_desc_plain(smem_u32(q_tile), CHUNK_STRIDE, GROUP_STRIDE);
      const uint64_t desc_k0 =
          make_smem_desc_plain(smem_u32(k_stages), piece_stride, page_size >= 32 ? GROUP_STRIDE : page_bytes);
      TreeCursor c = at;
      int turn = 0, segment = 0;
      for (int left = run.count; left > 0 && !*failed; ++segment) {
        const int count = min(c.tiles - c.tile, left);
        bool ok = tree_wait(q_ready, static_cast<uint32_t>(segment) & 1u);
        for (int t = 0; t < count && ok && !*failed; ++t, ++turn) {
          const int b = turn & 1, stage = turn % K_STAGES;
          // (the buffer held the probabilities of two turns ago, which the output product must have read)
          ok = tree_wait(&k_full[stage], static_cast<uint32_t>(turn / K_STAGES) & 1u) &&
               (turn < 2 || tree_wait(&o_full[b], static_cast<uint32_t>(turn / 2 - 1) & 1u));
          if (!ok) break;
          tc_fence_after();
          const uint64_t desc_k = desc_k0 + stage * (Config::kHalfBytes >> 4);
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            umma_bf16(tmem_base + b * BLOCK_N, desc_q + k * ((2 * CHUNK_STRIDE) >> 4), desc_k + k * key_step, idesc,
                      k > 0 ? 1u : 0u);
          if (halves) {
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
              umma_bf16(tmem_base + b * BLOCK_N + BLOCK_N / 2, desc_q + k * ((2 * CHUNK_STRIDE) >> 4),
                        desc_k + apart + k * key_step, idesc, k > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[b]);
          umma_commit(&k_done[stage]);
          if (t == count - 1) umma_commit(q_done);
        }
        if (!ok) {
          atomicOr(a.status, HX_FLAG_WAIT_TIMEOUT);
          *failed = 1;
        }
        left -= count;
        if (left > 0) tree_next_item<BLOCK_N>(a, c);
      }
    }
  } else if (warp == WARP_OUTPUT) {
    // ----------------------------------------------------------- output products
    if (hx_elect_one()) {
      constexpr uint32_t idesc = make_idesc_b_mn_major(BLOCK_M, D);
      // values: MN-major, the next 8 keys are 128 bytes or a block on, the next 8 coordinates one piece on
      const uint64_t desc_v0 =
          make_smem_desc_plain(smem_u32(v_stages), page_size >= 32 ? GROUP_STRIDE : page_bytes, piece_stride);
      uint32_t value_step[BLOCK_N / 16];
#pragma unroll
      for (int g = 0; g < BLOCK_N / 16; ++g)
        value_step[g] = (page_size == 16 ? 2 * (g & 1) * page_bytes + (g >> 1) * GROUP_STRIDE
                                         : (g * 16 / page_size) * page_bytes + (g * 16 % page_size) * 16) >> 4;
      const uint32_t target = tmem_base + Config::kOutputColumn;
      TreeCursor c = at;
      int turn = 0;
      for (int left = run.count; left > 0 && !*failed;) {
        const int count = min(c.tiles - c.tile, left);
        for (int t = 0; t < count && !*failed; ++t, ++turn) {
          const int b = turn & 1, stage = turn % V_STAGES;
          // (the first probabilities of a segment come when the rows of the one before have left)
          if (!tree_wait(&p_full[b], static_cast<uint32_t>(turn / 2) & 1u) ||
              !tree_wait(&v_full[stage], static_cast<uint32_t>(turn / V_STAGES) & 1u)) {
            atomicOr(a.status, HX_FLAG_WAIT_TIMEOUT);
            *failed = 1;
            break;
          }
          tc_fence_after();
          const uint64_t desc_v = desc_v0 + stage * (Config::kHalfBytes >> 4);
          // (from either half's first column on 16 columns of P's high terms, and 16 of its low ones)
          const uint32_t probabilities = tmem_base + b * BLOCK_N;
#pragma unroll
          for (int g = 0; g < BLOCK_N / 16; ++g) {
            const uint32_t high = probabilities + (g >> 1) * (BLOCK_N / 2) + (g & 1) * 8;
            umma_bf16_a_tmem(target, high, desc_v + value_step[g], idesc, (t > 0 || g > 0) ? 1u : 0u);
            umma_bf16_a_tmem(target, high + BLOCK_N / 4, desc_v + value_step[g], idesc, 1u);
          }
          umma_commit(&v_done[stage]);
          umma_commit(&o_full[b]);
        }
        left -= count;
        if (left > 0) tree_next_item<BLOCK_N>(a, c);
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax
    constexpr int HALF = BLOCK_N / 2;
    const int quarter = warp & 3;      // tensor-memory lanes [32 * quarter, 32 * quarter + 32)
    const int half = (warp - 4) >> 2;  // which 32 columns of a tile, and which half of O's
    const int row = quarter * 32 + lane;
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t output_base = lane_base + Config::kOutputColumn;
    const float scale_log2 = a.scale * HX_LOG2E;      // positive: it does not change which score is largest
    const uint64_t factor_pair = pair_of(scale_log2, scale_log2), minus_one = pair_of(-1.0f, -1.0f);
    uint32_t meetings = 0;
    // The two warps of 32 rows meet: each arrives, and waits for both.
    auto arrive = [&]() {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&met[quarter]);
    };
    auto meet = [&]() {
      const bool there = wait_for(&met[quarter], meetings++);
      tc_fence_after();
      return there;
    };
    // This thread's number for the one that the other thread of the row tells, through a column of the score
    // buffer whose score has been read.  The arrival behind it says that the other's has been read, too: before
    // anything else goes into that column (the low terms of the probabilities, the next scores, which wait for
    // them) the threads have met once more.
    auto exchange = [&](uint32_t columns, float mine, float& other) {
      tmem_store1(columns + half * HALF, mine);
      tmem_store_wait();
      arrive();
      if (!meet()) return false;
      other = tmem_load1(columns + (half ^ 1) * HALF);
      arrive();
      return true;
    };
    TreeCursor c = at;
    int turn = 0, segment = 0;
    bool ok = true;
    for (int left = run.count; left > 0 && ok; ++segment) {
      const int count = min(c.tiles - c.tile, left);
      const TreeRows rows(a, c);
      const int rows_here = rows.count;
      const int my_token = rows.token0 + min(row, rows_here - 1) / rows.heads;      // (rows behind the last: any)
      const int my_head = rows.head0 + row % rows.heads;
      const bool live = quarter * 32 < rows_here;                         // the warp has rows
      // the first word of the row's mask, which is wanted at the item's end, is on its way from its beginning on
      const unsigned long long* words_of_row = tree_words(a, c, my_token);
      const unsigned long long first_word = live ? __ldg(words_of_row) : 0ull;
      float row_max = -INFINITY;      // the reference of this row's exponentials, in log2 units
      float row_sum = 0.0f;           // of this thread's columns, from the last tile on of both
      for (int t = 0; t < count && ok; ++t, ++turn) {
        const int b = turn & 1;
        ok = wait_for(&s_full[b], static_cast<uint32_t>(turn / 2));
        if (!ok) break;
        const int key0 = (c.tile + t) * BLOCK_N;
        const bool drafted = key0 + BLOCK_N > c.context;
        if (live) {
          tc_fence_after();
          const uint32_t score_base = lane_base + b * BLOCK_N;
          float p[HALF];
          {
            uint32_t r[2][16];
            tmem_load16_issue(score_base + half * HALF, r[0]);
            tmem_load16_issue(score_base + half * HALF + 16, r[1]);
            tmem_load_wait();
#pragma unroll
            for (int i = 0; i < HALF; ++i) p[i] = __uint_as_float(r[i / 16][i % 16]);
          }
          if (drafted) {
            const unsigned long long mask =
                tree_mask_of(a, c, key0, first_word, [&](int word) { return words_of_row[word]; });
            uint32_t seen = static_cast<uint32_t>(mask >> (HALF * half));
            if (page_size == 16)      // the order of the columns
              seen = __byte_perm(static_cast<uint32_t>(mask), static_cast<uint32_t>(mask >> 32),
                                 half == 0 ? 0x6420 : 0x7531);
#pragma unroll
            for (int i = 0; i < HALF; ++i)
              if (!((seen >> i) & 1)) p[i] = -INFINITY;
          }
          float part_max[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) part_max[u] = max_of_3(p[u], p[u + 4], p[u + 8]);
#pragma unroll
          for (int i = 12; i + 8 <= HALF; i += 8)
#pragma unroll
            for (int u = 0; u < 4; ++u) part_max[u] = max_of_3(part_max[u], p[i + u], p[i + 4 + u]);
#pragma unroll
          for (int u = 0; u < 4; ++u) part_max[u] = fmaxf(part_max[u], p[HALF - 4 + u]);
          const float own_max = scale_log2 * fmaxf(max_of_3(part_max[0], part_max[1], part_max[2]), part_max[3]);
          float other_max = 0.0f;
          ok = exchange(score_base + HALF / 2, own_max, other_max);
          if (!ok) break;
          const float tile_max = fmaxf(own_max, other_max);
          // a row that has seen nothing yet keeps -inf as its reference and zeros as its probabilities
          const float old_max = row_max;
          // (each row by itself, so that what another row sees does not reach this one, not even by rounding)
          const bool exceeds = row < rows_here && tile_max > old_max + RAISE_MAXIMUM_BY;
          const bool raised = t > 0 && __any_sync(0xffffffffu, exceeds);
          if (t == 0 || exceeds) row_max = tile_max;
          if (raised) {
            // what O holds was taken against the old reference; the product of the last turn must have landed
            const float correction = !exceeds ? 1.0f : old_max == -INFINITY ? 0.0f : fast_exp2(old_max - row_max);
            row_sum *= correction;
            ok = wait_for(&o_full[(turn - 1) & 1], static_cast<uint32_t>((turn - 1) / 2));
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1      // (rare: the loop that runs every time keeps the instruction cache)
            for (int d0 = 16 * half; d0 < D; d0 += 32) {
              uint32_t r[16];
              tmem_load16_issue(output_base + d0, r);
              tmem_load_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * correction);
              tmem_store16_raw(output_base + d0, r);
            }
          }
          // P = hi + lo, two keys per column, the earlier key in the lower half
          uint64_t part_sum[2] = {0, 0};
          const float reference = row_max == -INFINITY ? 0.0f : row_max;
          const uint64_t reference_pair = pair_of(-reference, -reference);
          uint32_t high[16], low[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float x0, x1;
            halves_of(pair_fma(pair_of(p[2 * i], p[2 * i + 1]), factor_pair, reference_pair), x0, x1);
            const uint64_t weights = pair_of(fast_exp2(x0), fast_exp2(x1));
            part_sum[i % 2] = pair_add(part_sum[i % 2], weights);
            halves_of(weights, x0, x1);
            high[i] = pack_bf16(x0, x1);
            halves_of(pair_fma(pair_of(__uint_as_float(high[i] << 16), __uint_as_float(high[i] & 0xffff0000u)), minus_one,
                               weights), x0, x1);
            low[i] = pack_bf16(x0, x1);
          }
          {
            float even, odd;
            halves_of(pair_add(part_sum[0], part_sum[1]), even, odd);
            row_sum += even + odd;
          }
          tmem_store16_raw(score_base + half * HALF, high);
          ok = meet();
          if (!ok) break;
          if (t == count - 1) {
            float other_sum = 0.0f;
            ok = exchange(score_base + HALF / 2 + 1, row_sum, other_sum) && meet();
            if (!ok) break;
            row_sum = half == 0 ? row_sum + other_sum : other_sum + row_sum;
          }
          tmem_store16_raw(score_base + half * HALF + HALF / 2, low);
          tmem_store_wait();
        }
        if (drafted) {
          ok = wait_for(&v_full[turn % V_STAGES], static_cast<uint32_t>(turn / V_STAGES));
          if (!ok) break;
          // a thread has a key and every fourth piece of its value
          const int number = half * 128 + row, key = number & (BLOCK_N - 1);
          bool wrote = false, found = false;
          if (key >= c.context - key0) {
            uint8_t* at_key = v_stages + (turn % V_STAGES) * Config::kHalfBytes + (key >> page_shift) * page_bytes +
                              (key & (page_size - 1)) * 16;
#pragma unroll
            for (int j = 0; j < (PIECES + 3) / 4; ++j) {
              const int piece = 4 * j + number / BLOCK_N;
              if (piece >= PIECES) break;
              uint4* place = reinterpret_cast<uint4*>(at_key + piece * piece_stride);
              uint4 value = *place;
              if ((exponents_of(value.x) | exponents_of(value.y) | exponents_of(value.z) | exponents_of(value.w)) == 0u)
                continue;
              value.x &= ~exponents_of(value.x);
              value.y &= ~exponents_of(value.y);
              value.z &= ~exponents_of(value.z);
              value.w &= ~exponents_of(value.w);
              *place = value;
              wrote = true;
            }
            found = wrote && key < c.context + c.nodes - key0;
          }
          if (found) poisoned[segment & 1] = segment;
          if (__any_sync(0xffffffffu, wrote)) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[b]);
      }
      if (!ok) break;

      // ---- the segment's rows: finished, or this CTA's part of them; a thread has half of the coordinates
      ok = wait_for(&o_full[(turn - 1) & 1], static_cast<uint32_t>((turn - 1) / 2));
      if (!ok) break;
      if (live) {
        tc_fence_after();
        const bool whole = c.tile == 0 && count == c.tiles;
        const float inverse = tree_inverse(row_sum);
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + static_cast<size_t>(c.q_begin + my_token) * a.ldo +
                             static_cast<size_t>(my_head) * D;
        float* part = tree_part<BLOCK_M>(a, blockIdx.x, c.tile == 0);
#pragma unroll 1      // (instructions that are met once an item come at 40 cycles for eight)
        for (int d0 = 16 * half; d0 < D; d0 += 32) {
          float o[16];
          __syncwarp();
          tmem_load16(output_base + d0, o);
          if (row < rows_here) {
            if (row_sum == 0.0f) {
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = 0.0f;
            }
            if (whole) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint4 packed;
                packed.x = pack_bf16(o[8 * h] * inverse, o[8 * h + 1] * inverse);
                packed.y = pack_bf16(o[8 * h + 2] * inverse, o[8 * h + 3] * inverse);
                packed.z = pack_bf16(o[8 * h + 4] * inverse, o[8 * h + 5] * inverse);
                packed.w = pack_bf16(o[8 * h + 6] * inverse, o[8 * h + 7] * inverse);
                *reinterpret_cast<uint4*>(out + d0 + 8 * h) = packed;
              }
            } else {
#pragma unroll
              for (int h = 0; h < 4; ++h)
                *reinterpret_cast<float4*>(part + (static_cast<size_t>(d0 / 4 + h) * BLOCK_M + row) * 4) =
                    make_float4(o[4 * h], o[4 * h + 1], o[4 * h + 2], o[4 * h + 3]);
            }
          }
        }
        if (!whole && half == 0 && row < rows_here) {
          part[static_cast<size_t>(D) * BLOCK_M + row] = row_max;
          part[static_cast<size_t>(D + 1) * BLOCK_M + row] = row_sum;
        }
        // (told before the arrivals that the last output product waited for)
        if (poisoned[segment & 1] == segment && row < rows_here)
          add_not_finite<D>(a, c, count, my_token, row, half, whole ? out : nullptr, whole ? nullptr : part);
        tc_fence_before();
      }
      left -= count;
      if (left > 0) tree_next_item<BLOCK_N>(a, c);
      else if (threadIdx.x == 128) tree_tell_cut<BLOCK_M>(a, run, c, count);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == WARP_SCORES) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Config::kTmemColumns);
  }
}

template <int D>
int launch(const TreeArgs& a, int ctas, cudaStream_t stream) {
  using Config = TreeTcConfig<D>;
  static std::atomic<unsigned long long> ready{0};
  const bool reserved = hx_once_a_device(ready, [] {
    return cudaFuncSetAttribute(tree_attention_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                Config::kSmemBytes) == cudaSuccess &&
           cudaFuncSetAttribute(tree_attention_tc_kernel<D>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                cudaSharedmemCarveoutMaxShared) == cudaSuccess;
  });
  HX_REQUIRE(reserved, "hx_tree_attention: cannot reserve %d bytes of shared memory", Config::kSmemBytes);
  hx_launch(tree_attention_tc_kernel<D>, ctas, THREADS, Config::kSmemBytes, stream, a);
  HX_CHECK_LAUNCH("hx_tree_attention");
  return HX_OK;
}

}  // namespace

bool hx_tree_tc_takes(int head_dim, int page_size) {
  return head_dim >= 64 && head_dim <= 128 && head_dim % 16 == 0 &&
         (page_size == 8 || page_size == 16 || page_size == 32 || page_size == 64);
}

long long hx_tree_tc_floats(int head_dim) {
  return tree_scratch_floats<BLOCK_M>(head_dim, hx_device_sm_count() * CTAS_AN_SM);
}

int hx_tree_tc_launch(TreeArgs a, cudaStream_t stream) {
  tree_fill_rows(a, BLOCK_M);
  const int ctas = hx_device_sm_count() * CTAS_AN_SM;
  int rc;
  switch (a.head_dim) {
    case 64: rc = launch<64>(a, ctas, stream); break;
    case 80: rc = launch<80>(a, ctas, stream); break;
    case 96: rc = launch<96>(a, ctas, stream); break;
    case 112: rc = launch<112>(a, ctas, stream); break;
    default: rc = launch<128>(a, ctas, stream); break;
  }
  if (rc != HX_OK) return rc;
  return hx_tree_join(a, HX_BF16, ctas, BLOCK_M, 4, stream);
}
