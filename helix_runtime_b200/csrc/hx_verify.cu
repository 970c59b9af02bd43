// Verification of drafted tokens against the target model, from given uniform numbers.
//
// A request's step held a tree: token 0 is the last one it was given, every other is a draft for
// what follows its parent, drawn from a draft distribution q of that parent.  The walk starts at
// token 0.  At a token with target distribution p = softmax(logits / T) its children are tried in
// order; one that stands is walked to, and when none stands the next token is drawn from what is
// left of p.  The tokens then follow the target's own distribution, whatever q is.
//
// The mathematics.  With r the distribution that is left (p at first) a child x with number u stands
// when u q(x) < r(x); when it falls, r becomes max(r - q, 0) over its sum.  Children that were drawn without
// putting back: q loses x and is scaled by c = 1 / (1 - q of the fallen).  Both are followed in two
// numbers instead of a distribution: r = max(p - b q, 0) / S with S its sum, and b += S c, S = sum max(p -
// b q, 0) when a child falls (b = 0 and S = 1 at first; where r is zero it stays zero, as b
// only grows; a fallen x had r(x) <= u c q(x), so that what is left of it is zero without a list of the
// fallen).  Without a draft model q is one at the drafted token: it stands when u S < p(x), and S
// loses p(x) when it falls, so only the fallen have to be remembered.
//
// Numbers.  A decision is a comparison of two products, and the next token the place where a
// running sum over tens of thousands of tokens passes a number: with sums in float32 about one draw in a
// hundred would land beside the exact place.  Logits are float32, exponentials and sums 64-bit:
// 2^n times a table of 2^(j / 64) times a polynomial in what is left (after P. T. P. Tang,
// "Table-driven implementation of the exponential function", 1989), whose error of a few 1e-16 is what
// the sums have anyway, in a dozen instructions.
//
// Layout.  A request is a cluster of CTAs; every warp owns a stretch of the vocabulary, which it
// reads for the largest logit and again for the exponentials; those stay
// in shared memory, in 64 bits, so that a fallen child costs no second exponential (a vocabulary too long for
// that: they are computed again).  A visited token takes
// one exchange through distributed shared memory, one more a fallen child: a CTA adds up its warps and tells
// the others, and then each takes the same decisions from the same numbers.  What a chain of visited tokens
// takes is latency, so the tree lies in shared memory, the logits of all children are asked for
// together with the row, and the row that comes next if the first child stands is fetched into the L2
// meanwhile.  Only rows of tokens that are walked over are read.
//
// Measured (32,000 tokens): 64 requests x 32 drafts, with the drafts' logits, 100 to 118 us by the walks drawn; one request x 8 16
// to 32; 32 x 16 without a draft model 27 to 34.  A visited token takes about 13,000 cycles (two passes over its
// stretch, an exchange, and one more with each child that falls), the deepest walk of a batch sets the time.  Its bytes,
// 25 MB, would take 4 us.
#include "hx_common.cuh"

#include <atomic>

namespace {

constexpr int WARPS = 16, THREADS = WARPS * 32;
constexpr int MAX_CLUSTER = 8;
constexpr int TABLE = 64;
constexpr int MOST_CACHED = 200 * 1024;
constexpr int TREE = 256;      // tokens of a tree that shared memory holds (a larger one is read where it lies)

struct VerifyArgs {
  const float* logits;      // [tokens, ld]
  int ld;
  const float* draft;       // [tokens, ld_draft]: row t, what the children of token t were drawn from; null: none
  int ld_draft;
  const int* ids;           // [tokens] the drafted tokens
  const int* parents;       // [tokens] within the request, in front of the child; -1: token 0
  const int* request_start;
  const float* heat;        // [requests]; not above zero: greedy
  const float* uniform;     // [tokens] a token's number; token 0's: the next token's
  int* path;                // [requests, ld_path]
  int ld_path;
  int width;
  int* kept;
  int* next;
  int vocab;
  int span;                 // tokens of the vocabulary a warp owns, a multiple of 128
  int put_back;             // children were drawn with putting back
  int cached;               // shared memory holds the exponentials of a CTA's stretches
  int* status;
};

// What a warp (and then a CTA) says of its stretch: maximum and sum of exponentials against it, of target
// and draft.
struct Told {
  double p_sum, q_sum;
  float p_max, q_max;
  int best;                 // the lowest id of p_max
  int bad;                  // 1: a logit that is none
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  return rank;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t size;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
  return size;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t address_in(const void* p, uint32_t rank) {
  uint32_t address;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(address)
               : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
  return address;
}
__device__ __forceinline__ void store_in(uint32_t address, uint64_t value) {
  asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(address), "l"(value) : "memory");
}

// e^((x - top) / T) for x <= top: `unit` is 64 / (T ln 2).
struct Exponential {
  const double* table;      // 2^(j / 64)
  double unit, top;
  __device__ __forceinline__ double operator()(float x) const {
    constexpr double ROUND = 6755399441055744.0;      // 1.5 * 2^52: the sum's low bits are a whole number
    constexpr double C1 = 0.010830424696249145;       // ln 2 / 64 and its powers over the factorials
    const double y = (static_cast<double>(x) - top) * unit;      // in units of 1 / 64 octave
    if (!(y > -64.0 * 1000.0)) return 0.0;             // below 2^-1000, and minus infinity
    const double whole = y + ROUND;
    const double rest = y - (whole - ROUND);
    const int n = __double2loint(whole);
    constexpr double C2 = C1 * C1 / 2.0, C3 = C2 * C1 / 3.0, C4 = C3 * C1 / 4.0, C5 = C4 * C1 / 5.0;
    double p = fma(rest, C5, C4);
    p = fma(rest, p, C3);
    p = fma(rest, p, C2);
    p = fma(rest, p, C1);
    p = fma(rest, p, 1.0);
    const double base = table[n & (TABLE - 1)];
    return __hiloint2double(__double2hiint(base) + (n >> 6) * (1 << 20), __double2loint(base)) * p;
  }
};

__device__ __forceinline__ double warp_sum(double value) {
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) value += __shfl_xor_sync(0xffffffffu, value, offset);
  return value;
}

__device__ __forceinline__ void take_larger(float& value, int& id, float other, int other_id) {
  if (other > value || (other == value && other_id < id)) {
    value = other;
    id = other_id;
  }
}

__device__ __forceinline__ double sum_of(double value, int width) {
  for (int offset = width / 2; offset > 0; offset >>= 1) value += __shfl_xor_sync(0xffffffffu, value, offset);
  return value;
}

// `width` (a power of two) of these, one a lane, as one: sums against the common maxima.  All lanes below
// `width` get the result.
__device__ __forceinline__ Told join_told(const Told& mine, int width, const double* table, double unit) {
  Told all;
  all.p_max = mine.p_max;
  all.q_max = mine.q_max;
  all.best = mine.best;
  all.bad = mine.bad;
  for (int offset = width / 2; offset > 0; offset >>= 1) {
    take_larger(all.p_max, all.best, __shfl_xor_sync(0xffffffffu, all.p_max, offset),
                __shfl_xor_sync(0xffffffffu, all.best, offset));
    all.q_max = fmaxf(all.q_max, __shfl_xor_sync(0xffffffffu, all.q_max, offset));
    all.bad |= __shfl_xor_sync(0xffffffffu, all.bad, offset);
  }
  all.p_sum = sum_of(mine.p_sum > 0.0 ? mine.p_sum * Exponential{table, unit, all.p_max}(mine.p_max) : 0.0, width);
  all.q_sum = sum_of(mine.q_sum > 0.0 ? mine.q_sum * Exponential{table, unit, all.q_max}(mine.q_max) : 0.0, width);
  return all;
}

// (two CTAs an SM: with one, and no registers spilled, the same 64 walks took 120 us instead of 106)
__global__ __launch_bounds__(THREADS, 2) void verify_kernel(const __grid_constant__ VerifyArgs a) {
  extern __shared__ double exponentials[];          // [WARPS][span / 4 lanes ...]: of p and, behind all of them, of q
  __shared__ double table[TABLE];
  __shared__ Told of_warp[WARPS], of_cta[2][MAX_CLUSTER];
  __shared__ double sums_of_warp[WARPS];            // of the last exchange, for the draw
  __shared__ int parent_of[TREE], id_of[TREE];
  __shared__ float number_of[TREE];
  hx_pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = cluster_rank(), ctas = cluster_size();
  const int request = blockIdx.x / ctas;
  const int me = rank * WARPS + warp;
  if (threadIdx.x < TABLE) table[threadIdx.x] = exp2(threadIdx.x * (1.0 / TABLE));
  hx_pdl_wait();
  const int begin = a.request_start[request];
  const int nodes = a.request_start[request + 1] - begin;
  const bool held_tree = nodes <= TREE;
  if (held_tree)
    for (int j = threadIdx.x; j < nodes; j += THREADS) {
      parent_of[j] = a.parents[begin + j];
      id_of[j] = a.ids[begin + j];
      number_of[j] = a.uniform[begin + j];
    }
  cluster_sync();      // every CTA's shared memory is there, and the tree in it

  int* path = a.path + static_cast<size_t>(request) * a.ld_path;
  const bool writes = rank == 0 && warp == 0;
  if (nodes <= 0) {      // (the same in the whole cluster)
    if (writes) {
      for (int k = lane; k < a.width; k += 32) path[k] = -1;
      if (lane == 0) {
        a.kept[request] = 0;
        a.next[request] = -1;
      }
    }
    return;
  }
  const float heat = a.heat[request];
  const bool greedy = !(heat > 0.0f);
  const double unit = greedy ? 0.0 : TABLE / (0.693147180559945309 * static_cast<double>(heat));
  const int first = min(static_cast<long long>(me) * a.span, static_cast<long long>(a.vocab));
  const int last = min(static_cast<long long>(first) + a.span, static_cast<long long>(a.vocab));
  const bool wide = a.ld % 4 == 0 && a.ld_draft % 4 == 0 && (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 &&
                    (reinterpret_cast<uintptr_t>(a.draft) & 15) == 0;
  double* p_cache = exponentials + warp * a.span;
  double* q_cache = p_cache + WARPS * a.span;
  int phase = 0;       // which half of `of_cta` the next exchange uses

  // One exchange: the CTA's warps as one, told to every CTA; all warps of the cluster get the
  // cluster's.  (A half is written again two exchanges later: everyone has passed the barrier between.)
  auto tell = [&](const Told& mine, bool plain_sums) {
    phase ^= 1;
    if (lane == 0) {
      of_warp[warp] = mine;
      sums_of_warp[warp] = mine.p_sum;
    }
    __syncthreads();
    if (warp == 0) {
      Told cta = of_warp[lane % WARPS];
      if (plain_sums) cta.p_sum = sum_of(cta.p_sum, WARPS);
      else cta = join_told(cta, WARPS, table, unit);
      if (lane < ctas) {
        const uint32_t place = address_in(&of_cta[phase][rank], lane);
        store_in(place, __double_as_longlong(cta.p_sum));
        store_in(place + 8, __double_as_longlong(cta.q_sum));
        store_in(place + 16, static_cast<uint64_t>(__float_as_uint(cta.p_max)) |
                                 static_cast<uint64_t>(__float_as_uint(cta.q_max)) << 32);
        store_in(place + 24, static_cast<uint64_t>(static_cast<uint32_t>(cta.best)) |
                                 static_cast<uint64_t>(static_cast<uint32_t>(cta.bad)) << 32);
      }
    }
    cluster_sync();
  };
  auto cache_place = [&](int id) { return (id & 3) * (a.span / 4) + ((id - first) >> 2); };
  auto parent_at = [&](int j) { return held_tree ? parent_of[j] : a.parents[begin + j]; };
  auto id_at = [&](int j) { return held_tree ? id_of[j] : a.ids[begin + j]; };
  auto number_at = [&](int j) { return held_tree ? number_of[j] : a.uniform[begin + j]; };
  // the next child of `node` behind `after`, or `nodes`
  auto child_of = [&](int node, int after) {
    for (int base = after + 1; base < nodes; base += 32) {
      const int j = base + lane;
      const unsigned found = __ballot_sync(0xffffffffu, j < nodes && parent_at(j) == node);
      if (found != 0u) return base + __ffs(found) - 1;
    }
    return nodes;
  };

  int node = 0, kept = 1, bad_token = 0;
  if (writes && lane == 0) path[0] = 0;
  while (true) {
    const float* row = a.logits + static_cast<size_t>(begin + node) * a.ld;
    int child = kept < a.width ? child_of(node, node) : nodes;      // (a path that is full ends)
    const bool drafted = a.draft != nullptr && child < nodes && !greedy;
    const float* draft = drafted ? a.draft + static_cast<size_t>(begin + node) * a.ld_draft : row;

    // calls take(id, p, q) for this lane's tokens of the warp's stretch: four side by side of each 128
    auto each = [&](auto take) {
#pragma unroll 2
      for (int id = first + 4 * lane; id < last; id += 128) {
        float p[4], q[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (wide && id + 3 < last) {
          const float4 four = __ldg(reinterpret_cast<const float4*>(row + id));
          p[0] = four.x; p[1] = four.y; p[2] = four.z; p[3] = four.w;
          if (drafted) {
            const float4 other = __ldg(reinterpret_cast<const float4*>(draft + id));
            q[0] = other.x; q[1] = other.y; q[2] = other.z; q[3] = other.w;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (id + e < last) {
              p[e] = __ldg(row + id + e);
              if (drafted) q[e] = __ldg(draft + id + e);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (id + e < last) take(id + e, p[e], q[e]);
      }
    };
    // lane k: the k-th child (of the first 32) and its logits
    int my_child = nodes, my_token = -1;
    float my_p = 0.0f, my_q = 0.0f;
    if (!greedy && child < nodes) {
      int count = 0;
      for (int j = child; j < nodes && count < 32; j = child_of(node, j), ++count)
        if (lane == count) my_child = j;
      if (my_child < nodes) my_token = id_at(my_child);
      if (my_token >= 0 && my_token < a.vocab) {
        my_p = __ldg(row + my_token);
        if (drafted) my_q = __ldg(draft + my_token);
      }
    }
    // the rows that come next if the first child stands
    if (child < nodes && lane < 8 && first + 32 * lane < last) {
      const size_t ahead = static_cast<size_t>(begin + child);
      asm volatile("prefetch.global.L2 [%0];" ::"l"(a.logits + ahead * a.ld + first + 32 * lane));
      if (drafted) asm volatile("prefetch.global.L2 [%0];" ::"l"(a.draft + ahead * a.ld_draft + first + 32 * lane));
    }

    Told mine;
    mine.p_max = mine.q_max = -INFINITY;
    mine.best = 0x7fffffff;
    bool bad = false;
    each([&](int id, float p, float q) {
      bad |= !isfinite(p) || !(q < INFINITY);      // (a draft may leave tokens out: minus infinity)
      if (p > mine.p_max) {
        mine.p_max = p;
        mine.best = id;
      }
      mine.q_max = fmaxf(mine.q_max, q);
    });
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) {
      take_larger(mine.p_max, mine.best, __shfl_xor_sync(0xffffffffu, mine.p_max, offset),
                  __shfl_xor_sync(0xffffffffu, mine.best, offset));
      mine.q_max = fmaxf(mine.q_max, __shfl_xor_sync(0xffffffffu, mine.q_max, offset));
    }
    mine.bad = __any_sync(0xffffffffu, bad);
    mine.p_sum = mine.q_sum = 0.0;
    if (!greedy && !mine.bad && first < last) {
      const Exponential of_p{table, unit, mine.p_max};
      // (a stretch that the draft leaves out wholly has no maximum: its sum is zero against any)
      const Exponential of_q{table, unit, fmaxf(mine.q_max, -3.0e38f)};
      double p_sum = 0.0, q_sum = 0.0;
      // (place e * span / 4 + id / 4 of the warp's: neighbouring lanes side by side)
      each([&](int id, float p, float q) {
        const double e_p = of_p(p), e_q = drafted ? of_q(q) : 0.0;
        p_sum += e_p;
        q_sum += e_q;
        if (a.cached) {
          const int place = cache_place(id);
          p_cache[place] = e_p;
          if (drafted) q_cache[place] = e_q;
        }
      });
      mine.p_sum = warp_sum(p_sum);
      if (drafted) mine.q_sum = warp_sum(q_sum);
    }
    tell(mine, false);
    bool row_sums = true;      // what was told last is the row's own sums (and not what a fallen child leaves)
    const Told all = join_told(of_cta[phase][lane % ctas], ctas, table, unit);
    if (all.bad || (drafted && all.q_max == -INFINITY)) {
      if (writes && lane == 0) {
        a.next[request] = -1;
        atomicOr(a.status, HX_FLAG_NONFINITE);
      }
      break;
    }
    const Exponential of_p{table, unit, all.p_max}, of_q{table, unit, drafted ? all.q_max : 0.0f};
    const double p_unit = 1.0 / all.p_sum, q_unit = drafted ? 1.0 / all.q_sum : 0.0;
    // what turns this warp's exponentials, against its own maxima, into shares
    const double p_factor = first < last && !greedy ? of_p(mine.p_max) * p_unit : 0.0;
    const double q_factor = first < last && drafted ? of_q(mine.q_max) * q_unit : 0.0;
    // calls take(id, share of p, share of q) for this lane's tokens
    auto each_share = [&](auto take) {
      if (a.cached) {
#pragma unroll 2
        for (int id = first + 4 * lane; id < last; id += 128)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (id + e < last) {
              const int place = cache_place(id + e);
              take(id + e, p_cache[place] * p_factor, drafted ? q_cache[place] * q_factor : 0.0);
            }
      } else {
        each([&](int id, float p, float q) { take(id, of_p(p) * p_unit, drafted ? of_q(q) * q_unit : 0.0); });
      }
    };

    // ---- the children, in order
    double b = 0.0, left = 1.0, gone = 0.0;
    // without putting back: different tokens that fell.  (Without a draft model their p is out of `left`, with one their
    // q is in `gone`; a token that is drafted again takes nothing more.)
    int fallen = 0;
    int fallen_token = -1;     // lane f: the f-th of them
    auto fell_before = [&](int child, int token) {
      bool again = __any_sync(0xffffffffu, lane < fallen && fallen_token == token);
      if (fallen > 32)
        for (int j = child_of(node, node); j < child; j = child_of(node, j)) again |= id_at(j) == token;
      return again;
    };
    auto remember = [&](int token) {
      if (lane == fallen) fallen_token = token;
      ++fallen;
    };
    int stands = -1;
    // lane k: the k-th child's shares, before anything fell
    const double my_p_share = !greedy && my_token >= 0 ? of_p(my_p) * p_unit : 0.0;
    const double my_q_share = drafted && my_token >= 0 ? of_q(my_q) * q_unit : 0.0;
    int order = 0;
    for (; child < nodes; child = child_of(node, child), ++order) {
      const int token = id_at(child);
      if (token < 0 || token >= a.vocab) {
        bad_token = 1;      // passed over
        continue;
      }
      if (greedy) {
        if (token != all.best) continue;
        stands = child;
        break;
      }
      const double u = number_at(child);
      double p = __shfl_sync(0xffffffffu, my_p_share, order & 31), q = __shfl_sync(0xffffffffu, my_q_share, order & 31);
      if (order >= 32) {
        p = of_p(__ldg(row + token)) * p_unit;
        q = drafted ? of_q(__ldg(draft + token)) * q_unit : 0.0;
      }
      if (drafted) {
        const double rest = 1.0 - gone;
        if (!(rest > 0.0)) continue;      // nothing of q is left to have been drawn from
        const double scale = a.put_back ? 1.0 : 1.0 / rest;
        const bool again = !a.put_back && fell_before(child, token);
        if (!again && u * q * scale * left < p - b * q) {
          stands = child;
          break;
        }
        b += left * scale;
        if (!a.put_back && !again) {
          gone += q;
          remember(token);
        }
        double sum = 0.0;
        each_share([&](int, double of_target, double of_draft) {
          const double over = of_target - b * of_draft;
          if (over > 0.0) sum += over;
        });
        mine.p_sum = warp_sum(sum);
        tell(mine, true);
        row_sums = false;
        left = sum_of(of_cta[phase][lane % ctas].p_sum, ctas);
      } else {
        if (fell_before(child, token)) continue;      // nothing of it is left
        if (u * left < p) {
          stands = child;
          break;
        }
        left -= p;
        remember(token);
      }
    }
    if (stands >= 0) {
      if (writes && lane == 0) path[kept] = stands;
      ++kept;
      node = stands;
      continue;
    }

    // ---- none stands: the next token, from what is left
    if (greedy) {
      if (writes && lane == 0) a.next[request] = all.best;
      break;
    }
    const double u = number_at(0);
    const bool plain = !(left > 0.0) || (fallen == 0 && b == 0.0);      // (nothing left but by rounding: p itself)
    const bool listed = !plain && !drafted && fallen > 0;      // the fallen children's tokens weigh nothing
    // has the token fallen? (the warp asks together)
    auto fell = [&](int id) {
      bool out = false;
      for (int f = 0; f < min(fallen, 32); ++f) out |= id == __shfl_sync(0xffffffffu, fallen_token, f);
      if (fallen > 32)
        for (int j = child_of(node, node); j < nodes; j = child_of(node, j)) out |= id_at(j) == id;
      return out;
    };
    // four tokens of this lane from `id` on, of which the fallen and those behind the stretch weigh nothing
    auto weights_of = [&](int id, double (&w)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool out = listed && fell(id + e);
        w[e] = 0.0;
        if (id + e >= last || out) continue;
        const int place = cache_place(id + e);
        w[e] = a.cached ? p_cache[place] * p_factor : of_p(__ldg(row + id + e)) * p_unit;
        if (plain || listed || !drafted) continue;
        w[e] -= b * (a.cached ? q_cache[place] * q_factor : of_q(__ldg(draft + id + e)) * q_unit);
        if (!(w[e] > 0.0)) w[e] = 0.0;
      }
    };
    // every warp's sum: p's from the row's first exchange, what is over from that of the last fallen
    // child, otherwise told now
    const bool first_sums = plain && row_sums;
    if (listed || (plain && !first_sums)) {
      double sum = 0.0;
      for (int base = first; base < last; base += 128) {
        double w[4];
        weights_of(base + 4 * lane, w);
        sum += (w[0] + w[1]) + (w[2] + w[3]);
      }
      mine.p_sum = warp_sum(sum);
      tell(mine, true);
    }
    // the CTA in which the running sum passes the target, and in it the warp; all add alike and agree
    auto pick = [&](double sum, int count, double target, double& before) {
      double inclusive = lane < count ? sum : 0.0;
#pragma unroll
      for (int offset = 1; offset < 32; offset <<= 1) {
        const double other = __shfl_up_sync(0xffffffffu, inclusive, offset);
        if (lane >= offset) inclusive += other;
      }
      const bool some = lane < count && sum > 0.0;
      const unsigned beyond = __ballot_sync(0xffffffffu, some && target < before + inclusive);
      const unsigned weighs = __ballot_sync(0xffffffffu, some);
      // (a sum that falls short by rounding: the last with any weight)
      const int source = beyond != 0u ? __ffs(beyond) - 1 : 31 - __clz(weighs | 1u);
      before += __shfl_sync(0xffffffffu, inclusive - (lane < count ? sum : 0.0), source);
      return source;
    };
    double cta_sum = 0.0;
    if (lane < ctas) {
      const Told& of = of_cta[phase][lane];
      cta_sum = !first_sums ? of.p_sum : of.p_sum > 0.0 ? of.p_sum * of_p(of.p_max) * p_unit : 0.0;
    }
    const double target = u * warp_sum(cta_sum);
    double before = 0.0;
    if (pick(cta_sum, ctas, target, before) == rank) {
      double sum = 0.0;
      if (lane < WARPS) {
        sum = sums_of_warp[lane];
        if (first_sums && sum > 0.0) sum *= of_p(of_warp[lane].p_max) * p_unit;
      }
      if (pick(sum, WARPS, target, before) == warp) {
        int chosen = -1, last_with_weight = -1;
        for (int base = first; base < last && chosen < 0; base += 128) {
          const int id = base + 4 * lane;
          double w[4];
          weights_of(id, w);
          double inclusive = (w[0] + w[1]) + (w[2] + w[3]);
          const double own = inclusive;
#pragma unroll
          for (int offset = 1; offset < 32; offset <<= 1) {
            const double other = __shfl_up_sync(0xffffffffu, inclusive, offset);
            if (lane >= offset) inclusive += other;
          }
          // this lane's first token whose running sum passes the target, and its last with any weight
          int passes = -1, heavy = -1;
          double running = before + (inclusive - own);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            running += w[e];
            if (w[e] > 0.0) heavy = id + e;
            if (passes < 0 && w[e] > 0.0 && target < running) passes = id + e;
          }
          const unsigned passed = __ballot_sync(0xffffffffu, passes >= 0);
          const unsigned weighs = __ballot_sync(0xffffffffu, heavy >= 0);
          if (weighs != 0u) last_with_weight = __shfl_sync(0xffffffffu, heavy, 31 - __clz(weighs));
          if (passed != 0u) chosen = __shfl_sync(0xffffffffu, passes, __ffs(passed) - 1);
          before += __shfl_sync(0xffffffffu, inclusive, 31);
        }
        if (chosen < 0) chosen = last_with_weight;      // the running sum fell short by rounding
        if (lane == 0) a.next[request] = chosen;
      }
    }
    break;
  }
  if (writes) {
    __syncwarp();
    for (int k = kept + lane; k < a.width; k += 32) path[k] = -1;
    if (lane == 0) {
      a.kept[request] = kept;
      if (bad_token) atomicOr(a.status, HX_FLAG_BAD_TOKEN);
    }
  }
}

}  // namespace

// One walk a request (see the head of this file).  path[r]: the tokens walked over, token 0 first, -1
// behind them; kept[r]: how many; next[r]: the token that follows the last of them.  A request without
// tokens has kept 0 and next -1.  A path of `width` tokens is full: the walk ends there.  A row that is
// walked over and holds a target logit that is not finite, or draft logits that are no distribution
// (not a number, infinity, minus infinity throughout): next -1 and HX_FLAG_NONFINITE.  A child whose token
// lies outside the vocabulary is passed over (HX_FLAG_BAD_TOKEN).
HX_API int hx_verify_drafts(const float* logits, int ld, const float* draft, int ld_draft, int vocab,
                            const int* token_ids, const int* parents, const int* request_start,
                            const float* temperature, const float* uniform, int* path, int ld_path, int width,
                            int* kept, int* next_tokens, int requests, int put_back, int* status,
                            cudaStream_t stream) {
  HX_REQUIRE(requests >= 0 && vocab > 0 && ld >= vocab && (draft == nullptr || ld_draft >= vocab),
             "hx_verify_drafts: bad sizes");
  HX_REQUIRE(width > 0 && ld_path >= width, "hx_verify_drafts: a path has room for at least token 0");
  HX_REQUIRE(temperature != nullptr && uniform != nullptr && status != nullptr, "hx_verify_drafts: missing arguments");
  if (requests == 0) return HX_OK;
  const int sms = hx_device_sm_count();
  HX_REQUIRE(sms > 0, "hx_verify_drafts: the device cannot be asked");
  HX_REQUIRE(requests <= (1 << 24), "hx_verify_drafts: too many requests");
  // As many CTAs a request as leave four an SM in all, half of which run at once: what a batch waits for is the
  // deepest walk, whose length is latency, and most walks are short (64 requests with trees of 32 over 32,000
  // tokens: 8 CTAs 106 us, 4 CTAs 135).  And no more than have 32 x 4 tokens a warp.
  int ctas = MAX_CLUSTER;
  while (ctas > 1 && (static_cast<long long>(requests) * ctas > 4ll * sms || vocab <= (ctas / 2) * WARPS * 128)) ctas /= 2;
  int span = (vocab + ctas * WARPS - 1) / (ctas * WARPS);
  span = (span + 127) / 128 * 128;
  VerifyArgs a{logits, ld, draft, ld_draft, token_ids, parents, request_start, temperature, uniform, path, ld_path,
               width, kept, next_tokens, vocab, span, put_back, 0, status};
  // exponentials of target and draft (a request without drafted tokens' logits needs none of them twice)
  const long long bytes = static_cast<long long>(WARPS) * span * 16;
  a.cached = bytes <= MOST_CACHED;
  static std::atomic<unsigned long long> ready{0};
  const bool reserved = hx_once_a_device(ready, [] {
    return cudaFuncSetAttribute(verify_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_CACHED) == cudaSuccess;
  });
  HX_REQUIRE(reserved, "hx_verify_drafts: cannot reserve %d bytes of shared memory", MOST_CACHED);
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(requests * ctas);
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = a.cached ? static_cast<size_t>(bytes) : 0;
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = ctas;
  attribute[0].val.clusterDim.y = 1;
  attribute[0].val.clusterDim.z = 1;
  attribute[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = hx_pdl_enabled() ? 2 : 1;
  cudaLaunchKernelEx(&config, verify_kernel, a);
  HX_CHECK_LAUNCH("hx_verify_drafts");
  return HX_OK;
}
