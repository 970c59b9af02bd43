// Moving what the paged cache holds: whole pages to other pages, and the rows of accepted drafted
// tokens to where they belong.  Both work on all layers of a group of layers at once:
// storage [layer, key|value, page, kv_head, (head_dim / c, slot, c)], see hx_cache_offset.
//
// Both are bound by memory: every byte is read once and written once.  Measured (32 layers of 32 heads of 128): 64
// pages to 64 others 159 us, 6.7 TB/s, as fast as any copy; one page 7 us, the call.  Kept rows of 32 requests, up to 6 each, 48 to
// 56 us: 16 bytes of each 32-byte sector are wanted, 64 bytes at a time leave memory, and what is
// wanted moves at 1.9 TB/s; one request's 9 us.
//
// Neither lets the next kernel in before it has completed.  Attention fetches what earlier steps have left
// in the cache before it waits for the kernel in front of it, and that one may have been let in
// early, too: behind a kernel that moves cached rows nothing may start early.
#include "hx_common.cuh"

namespace {

constexpr int THREADS = 256;

// ------------------------------------------------------------------------- whole pages

// A page of one plane (a layer's keys, or its values) is one contiguous block.  A CTA copies
// UNROLL x THREADS units of one page of one plane: its loads are all in flight before it
// looks whether the pair may be copied at all, and before the first store.
template <typename Unit, int UNROLL>
__global__ __launch_bounds__(THREADS) void copy_pages_kernel(uint8_t* storage, const int* source, const int* target,
                                                             int pairs, int num_pages, long long page_bytes,
                                                             int* status) {
  hx_pdl_wait();      // (and lets nobody in early, see above)
  const int pair = blockIdx.y;
  const size_t plane = static_cast<size_t>(blockIdx.z) * num_pages;
  const int from = source[pair], to = target[pair];
  if (from == to && from >= 0 && from < num_pages) return;
  const bool there = from >= 0 && from < num_pages && to >= 0 && to < num_pages;
  if (!there) {
    if (threadIdx.x == 0) atomicOr(status, HX_FLAG_BAD_PAGE);
    return;
  }
  const Unit* in = reinterpret_cast<const Unit*>(storage + (plane + from) * page_bytes);
  Unit* out = reinterpret_cast<Unit*>(storage + (plane + to) * page_bytes);
  const long long units = page_bytes / static_cast<long long>(sizeof(Unit));
  const long long first = static_cast<long long>(blockIdx.x) * UNROLL * THREADS + threadIdx.x;
  Unit value[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u)
    if (first + u * THREADS < units) value[u] = __ldcs(in + first + u * THREADS);
  // a page that another pair writes, or reads, is not written: what it would hold depends on who is first
  bool taken = false;
  for (int other = threadIdx.x; other < pairs; other += THREADS)
    taken |= other != pair && (target[other] == to || (source[other] == to && target[other] != to));
  if (__syncthreads_or(taken)) {
    if (threadIdx.x == 0) atomicOr(status, HX_FLAG_BAD_MOVE);
    return;
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u)
    if (first + u * THREADS < units) __stcs(out + first + u * THREADS, value[u]);
}

template <typename Unit>
int launch_copy(uint8_t* storage, const int* source, const int* target, int pairs, int planes, int num_pages,
                long long page_bytes, int* status, cudaStream_t stream) {
  constexpr int UNROLL = 4;
  const long long blocks = (page_bytes / static_cast<long long>(sizeof(Unit)) + UNROLL * THREADS - 1) / (UNROLL * THREADS);
  HX_REQUIRE(blocks <= 0x7fffffffll, "hx_copy_pages: pages of %lld bytes", page_bytes);
  hx_launch(copy_pages_kernel<Unit, UNROLL>, dim3(static_cast<unsigned>(blocks), pairs, planes), THREADS, 0, stream,
            storage, source, target, pairs, num_pages, page_bytes, status);
  HX_CHECK_LAUNCH("hx_copy_pages");
  return HX_OK;
}

// ---------------------------------------------------------------------------- kept rows

struct KeepArgs {
  uint8_t* storage;
  const int* block_tables;
  int table_stride;
  const int* request_table_row;
  const int* request_context;
  const int* path;
  int ld_path;
  int width;
  const int* kept;
  int kv_heads, page_size, num_pages;
  int pieces;            // units of a row: head_dim / c
  int planes;
  int* status;
};

// Row k of a request moves from place context + path[k] to place context + k.  The path ascends, so
// path[k] >= k, and a row's new place is the old one of an earlier row or of none: a warp that
// reads its rows before it writes them, in ascending order, overwrites nothing that is still wanted.
// Leading rows that stay where they are (path[k] = k) are left out.
//
// A CTA has a request and a share of its (plane, head, unit) items: what it has to find out first (how many
// rows, which, in which pages: a chain of loads) it finds out once for many of them.  A warp's
// lanes hold the rows of an item side by side (neighbouring slots of a page are neighbouring units), as
// many items as fit, and eight such loads are in flight.  A unit is 16 bytes of a sector of 32, so
// that rows which move alone move twice their bytes.
template <typename Unit>
__global__ __launch_bounds__(THREADS) void keep_rows_kernel(const KeepArgs a) {
  constexpr int LOADS = 8;      // items whose rows are in flight together
  hx_pdl_wait();      // (and lets nobody in early, see above)
  const int request = blockIdx.y;
  const int kept = a.kept[request];
  const int context = a.request_context[request];
  const int* path = a.path + static_cast<size_t>(request) * a.ld_path;
  const int* table = a.block_tables + static_cast<size_t>(a.request_table_row[request]) * a.table_stride;
  if (kept <= 0) return;
  // ---- the whole path is looked at before anything moves
  auto page_at = [&](int place, int& slot) {
    const int index = place / a.page_size;
    slot = place - index * a.page_size;
    const int page = place >= 0 && index < a.table_stride ? table[index] : -1;
    return page < a.num_pages ? page : -1;
  };
  bool bad_path = kept > a.width || context < 0, bad_page = false;
  int first = 0;      // rows in front that stay
  for (int base = 0; base < min(kept, a.width); base += THREADS) {
    const int k = base + threadIdx.x;
    int stays = 0;
    if (k < min(kept, a.width)) {
      const int from = path[k];
      bad_path |= from < 0 || (k > 0 && from <= path[k - 1]) || from > 0x7fffffff - max(context, 0);
      stays = from == k;
      if (!bad_path && !stays) {
        int slot;
        bad_page |= page_at(context + from, slot) < 0 || page_at(context + k, slot) < 0;
      }
    }
    first += __syncthreads_count(stays);
  }
  bad_path = __syncthreads_or(bad_path) != 0;
  bad_page = __syncthreads_or(bad_page) != 0;
  if (bad_path || bad_page) {
    if (threadIdx.x == 0) atomicOr(a.status, bad_path ? HX_FLAG_BAD_MOVE : HX_FLAG_BAD_PAGE);
    return;
  }
  const int moved = kept - first;
  if (moved <= 0) return;
  int lanes = 1;      // of a warp, for the rows of an item
  while (lanes < moved && lanes < 32) lanes *= 2;
  const int lane = threadIdx.x & 31, warps = THREADS / 32;
  const int items = a.kv_heads * a.pieces, items_a_warp = 32 / lanes;
  const size_t plane_units = static_cast<size_t>(a.num_pages) * items * a.page_size;
  Unit* storage = reinterpret_cast<Unit*>(a.storage);
  const int all_items = items * a.planes;
  const int stride = gridDim.x * warps * items_a_warp;
  for (int chunk = 0; chunk < moved; chunk += lanes) {
    const int k = first + chunk + lane % lanes;
    const bool mine = k < kept;
    int from_slot = 0, to_slot = 0;
    size_t from_block = 0, to_block = 0;      // of the page's first item in the first plane, in units
    if (mine) {
      const int from_page = page_at(context + path[k], from_slot), to_page = page_at(context + k, to_slot);
      from_block = static_cast<size_t>(from_page) * items * a.page_size + from_slot;
      to_block = static_cast<size_t>(to_page) * items * a.page_size + to_slot;
    }
    for (int item = (blockIdx.x * warps + (threadIdx.x >> 5)) * items_a_warp + lane / lanes;
         __any_sync(0xffffffffu, item < all_items); item += LOADS * stride) {
      Unit value[LOADS];
      size_t place[LOADS];
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        const int at = item + u * stride, plane = at / items;
        place[u] = plane * plane_units + static_cast<size_t>(at - plane * items) * a.page_size;
        if (mine && at < all_items) value[u] = storage[from_block + place[u]];
      }
      __syncwarp();
#pragma unroll
      for (int u = 0; u < LOADS; ++u)
        if (mine && item + u * stride < all_items) storage[to_block + place[u]] = value[u];
    }
    __syncwarp();
  }
}

}  // namespace

// Copies page source[i] to page target[i], i < pairs, in every one of `planes` planes of num_pages pages
// of page_bytes bytes.  A pair whose page lies outside the pool is left out (HX_FLAG_BAD_PAGE), and
// so is one whose target another pair writes or reads (HX_FLAG_BAD_MOVE).
HX_API int hx_copy_pages(void* storage, int planes, int num_pages, long long page_bytes, const int* source,
                         const int* target, int pairs, int* status, cudaStream_t stream) {
  HX_REQUIRE(planes > 0 && planes <= 65535 && num_pages > 0 && page_bytes > 0 && page_bytes % 4 == 0,
             "hx_copy_pages: bad cache geometry");
  HX_REQUIRE(pairs >= 0 && pairs <= 65535, "hx_copy_pages: %d pairs of pages (at most 65535)", pairs);
  HX_REQUIRE(status != nullptr && (reinterpret_cast<uintptr_t>(storage) & 3) == 0,
             "hx_copy_pages: status word missing or storage not aligned");
  if (pairs == 0) return HX_OK;
  uint8_t* bytes = static_cast<uint8_t*>(storage);
  if (page_bytes % 16 == 0 && (reinterpret_cast<uintptr_t>(storage) & 15) == 0)
    return launch_copy<uint4>(bytes, source, target, pairs, planes, num_pages, page_bytes, status, stream);
  return launch_copy<uint32_t>(bytes, source, target, pairs, planes, num_pages, page_bytes, status, stream);
}

// Request r keeps kept[r] of the rows behind its request_context[r] cached ones: row k moves from
// place context + path[r][k] to place context + k, in every plane.  path[r] ascends from at least 0 (the
// way down a tree whose tokens stand behind their parents).  A request whose path does not ascend or is
// longer than `width` (HX_FLAG_BAD_MOVE), or leads outside its pages (HX_FLAG_BAD_PAGE), is left as it is.
HX_API int hx_keep_rows(void* storage, int dtype, int planes, int num_pages, int kv_heads, int page_size,
                        int head_dim, const int* block_tables, int table_stride, const int* request_table_row,
                        const int* request_context, const int* path, int ld_path, int width, const int* kept,
                        int requests, int* status, cudaStream_t stream) {
  HX_REQUIRE(dtype == HX_F32 || dtype == HX_BF16, "hx_keep_rows: unknown dtype %d", dtype);
  HX_REQUIRE(planes > 0 && num_pages > 0 && kv_heads > 0 && page_size > 0 && head_dim > 0 &&
                 head_dim % 2 == 0 && table_stride > 0,
             "hx_keep_rows: bad cache geometry");
  HX_REQUIRE(requests >= 0 && requests <= 65535 && width > 0 && ld_path >= width, "hx_keep_rows: bad sizes");
  const int size = dtype == HX_BF16 ? 2 : 4, chunk = hx_cache_chunk(size, head_dim), unit = chunk * size;
  HX_REQUIRE(status != nullptr && (reinterpret_cast<uintptr_t>(storage) & (unit - 1)) == 0,
             "hx_keep_rows: status word missing or storage not aligned");
  HX_REQUIRE(static_cast<long long>(kv_heads) * (head_dim / chunk) < (1 << 24), "hx_keep_rows: rows too long");
  if (requests == 0) return HX_OK;
  KeepArgs a{static_cast<uint8_t*>(storage), block_tables, table_stride, request_table_row, request_context, path,
             ld_path, width, kept, kv_heads, page_size, num_pages, head_dim / chunk, planes, status};
  // eight CTAs an SM together, and no more than have a round of loads each
  const long long items = static_cast<long long>(kv_heads) * (head_dim / chunk) * planes;
  HX_REQUIRE(items < (1ll << 30), "hx_keep_rows: too many heads and planes");
  const int sms = hx_device_sm_count();
  HX_REQUIRE(sms > 0, "hx_keep_rows: the device cannot be asked");
  const long long wanted = (8ll * sms + requests - 1) / requests, most = (items + 8 * THREADS / 4 - 1) / (8 * THREADS / 4);
  const dim3 grid(static_cast<unsigned>(wanted < most ? wanted : most), requests);
  if (unit == 16) hx_launch(keep_rows_kernel<uint4>, grid, THREADS, 0, stream, a);
  else if (unit == 8) hx_launch(keep_rows_kernel<uint2>, grid, THREADS, 0, stream, a);
  else hx_launch(keep_rows_kernel<uint32_t>, grid, THREADS, 0, stream, a);
  HX_CHECK_LAUNCH("hx_keep_rows");
  return HX_OK;
}
