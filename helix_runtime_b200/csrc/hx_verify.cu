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
// Layout.  A request is a cluster of CTAs; every warp owns a stretch of the vocabulary and reads it
// from global memory (again from L1 when a child falls), and one exchange of the warps' sums
// through distributed shared memory a visited token, one more a fallen child, is all that the
// warps tell each other: each then takes the same decisions from the same numbers.  Only rows of tokens
// that are walked over are read.
#include "hx_common.cuh"

#include <mutex>

namespace {

constexpr int WARPS = 16, THREADS = WARPS * 32;
constexpr int MAX_CLUSTER = 8;
constexpr int TABLE = 64;

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
  int* status;
};

// What a warp tells about its stretch: maximum and sum of exponentials against it, of target and draft.
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
    return __hiloint2double(__double2hiint(base) + ((n >> 6) << 20), __double2loint(base)) * p;
  }
};

__device__ __forceinline__ double warp_sum(double value) {
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) value += __shfl_xor_sync(0xffffffffu, value, offset);
  return value;
}

__global__ __launch_bounds__(THREADS) void verify_kernel(const VerifyArgs a) {
  __shared__ double table[TABLE];
  __shared__ Told told[2][MAX_CLUSTER * WARPS];
  hx_pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = cluster_rank(), ctas = cluster_size();
  const int request = blockIdx.x / ctas;
  const int owners = ctas * WARPS, me = rank * WARPS + warp;
  if (threadIdx.x < TABLE) table[threadIdx.x] = exp2(threadIdx.x * (1.0 / TABLE));
  hx_pdl_wait();
  cluster_sync();      // every CTA's shared memory is there

  const int begin = a.request_start[request];
  const int nodes = a.request_start[request + 1] - begin;
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
  int phase = 0;       // which half of `told` the next exchange uses

  // One exchange: lane r of a warp writes the warp's words to CTA r; behind the barrier they are
  // everywhere.  (A half is written again two exchanges later: everyone has passed the barrier between.)
  auto tell = [&](const Told& mine) {
    phase ^= 1;
    if (lane < ctas) {
      const uint32_t place = address_in(&told[phase][me], lane);
      store_in(place, __double_as_longlong(mine.p_sum));
      store_in(place + 8, __double_as_longlong(mine.q_sum));
      store_in(place + 16, static_cast<uint64_t>(__float_as_uint(mine.p_max)) |
                               static_cast<uint64_t>(__float_as_uint(mine.q_max)) << 32);
      store_in(place + 24, static_cast<uint64_t>(static_cast<uint32_t>(mine.best)) |
                               static_cast<uint64_t>(static_cast<uint32_t>(mine.bad)) << 32);
    }
    cluster_sync();
  };
  // the next child of `node` behind `after`, or `nodes`
  auto child_of = [&](int node, int after) {
    for (int base = after + 1; base < nodes; base += 32) {
      const int j = base + lane;
      const unsigned found = __ballot_sync(0xffffffffu, j < nodes && a.parents[begin + j] == node);
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

    // ---- this warp's stretch of both rows
    Told mine;
    mine.p_max = mine.q_max = -INFINITY;
    mine.best = 0x7fffffff;
    bool bad = false;
    auto take = [&](float p, float q, int id) {
      bad |= !isfinite(p) || !(q < INFINITY);      // (a draft may leave tokens out: minus infinity)
      if (p > mine.p_max) {
        mine.p_max = p;
        mine.best = id;
      }
      mine.q_max = fmaxf(mine.q_max, q);
    };
#pragma unroll 4
    for (int id = first + lane; id < last; id += 32) take(row[id], drafted ? draft[id] : 0.0f, id);
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) {
      const float other = __shfl_xor_sync(0xffffffffu, mine.p_max, offset);
      const int other_best = __shfl_xor_sync(0xffffffffu, mine.best, offset);
      if (other > mine.p_max || (other == mine.p_max && other_best < mine.best)) {
        mine.p_max = other;
        mine.best = other_best;
      }
      mine.q_max = fmaxf(mine.q_max, __shfl_xor_sync(0xffffffffu, mine.q_max, offset));
    }
    mine.bad = __any_sync(0xffffffffu, bad);
    mine.p_sum = mine.q_sum = 0.0;
    if (!greedy && !mine.bad && first < last) {
      const Exponential of_p{table, unit, mine.p_max};
      // (a stretch that the draft leaves out wholly has no maximum: its sum is zero)
      const bool any_q = drafted && mine.q_max > -INFINITY;
      const Exponential of_q{table, unit, any_q ? mine.q_max : 0.0f};
      for (int id = first + lane; id < last; id += 32) {
        mine.p_sum += of_p(row[id]);
        if (any_q) mine.q_sum += of_q(draft[id]);
      }
      mine.p_sum = warp_sum(mine.p_sum);
      mine.q_sum = warp_sum(mine.q_sum);
    }
    tell(mine);

    // ---- everybody's: the same sums in the same order in every warp
    const Told* all = told[phase];
    float p_top = -INFINITY, q_top = -INFINITY;
    int best = 0x7fffffff, any_bad = 0;
    for (int w = lane; w < owners; w += 32) {
      if (all[w].p_max > p_top || (all[w].p_max == p_top && all[w].best < best)) {
        p_top = all[w].p_max;
        best = all[w].best;
      }
      q_top = fmaxf(q_top, all[w].q_max);
      any_bad |= all[w].bad;
    }
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) {
      const float other = __shfl_xor_sync(0xffffffffu, p_top, offset);
      const int other_best = __shfl_xor_sync(0xffffffffu, best, offset);
      if (other > p_top || (other == p_top && other_best < best)) {
        p_top = other;
        best = other_best;
      }
      q_top = fmaxf(q_top, __shfl_xor_sync(0xffffffffu, q_top, offset));
    }
    any_bad = __any_sync(0xffffffffu, any_bad);
    if (any_bad || (drafted && q_top == -INFINITY)) {
      if (writes && lane == 0) {
        a.next[request] = -1;
        atomicOr(a.status, HX_FLAG_NONFINITE);
      }
      break;
    }
    const Exponential of_p{table, unit, p_top}, of_q{table, unit, drafted ? q_top : 0.0f};
    double p_all = 0.0, q_all = 0.0;
    if (!greedy) {
      for (int w = lane; w < owners; w += 32) {
        if (all[w].p_sum > 0.0) p_all += all[w].p_sum * of_p(all[w].p_max);
        if (all[w].q_sum > 0.0) q_all += all[w].q_sum * of_q(all[w].q_max);
      }
      p_all = warp_sum(p_all);
      q_all = warp_sum(q_all);
    }
    const double p_unit = 1.0 / p_all, q_unit = drafted ? 1.0 / q_all : 0.0;

    // ---- the children, in order
    double b = 0.0, left = 1.0, gone = 0.0;
    int fallen = 0;            // without a draft model: different tokens that fell, whose p is out of `left`
    int fallen_token = -1;     // lane f: the f-th of them
    int stands = -1;
    for (; child < nodes; child = child_of(node, child)) {
      const int token = a.ids[begin + child];
      if (token < 0 || token >= a.vocab) {
        bad_token = 1;      // passed over
        continue;
      }
      if (greedy) {
        if (token != best) continue;
        stands = child;
        break;
      }
      const double u = a.uniform[begin + child];
      const double p = of_p(row[token]) * p_unit;
      if (drafted) {
        const double rest = 1.0 - gone;
        if (!(rest > 0.0)) continue;      // nothing of q is left to have been drawn from
        const double scale = a.put_back ? 1.0 : 1.0 / rest;
        const double q = of_q(draft[token]) * q_unit;
        if (u * q * scale * left < p - b * q) {
          stands = child;
          break;
        }
        b += left * scale;
        if (!a.put_back) gone += q;
        double sum = 0.0;
        for (int id = first + lane; id < last; id += 32) {
          const double over = of_p(row[id]) * p_unit - b * (of_q(draft[id]) * q_unit);
          if (over > 0.0) sum += over;
        }
        mine.p_sum = warp_sum(sum);
        mine.p_max = p_top;
        tell(mine);
        left = 0.0;
        for (int w = lane; w < owners; w += 32) left += told[phase][w].p_sum;
        left = warp_sum(left);
      } else {
        // fell already: nothing of it is left
        bool again = __any_sync(0xffffffffu, lane < fallen && fallen_token == token);
        if (fallen > 32)
          for (int j = child_of(node, node); j < child; j = child_of(node, j)) again |= a.ids[begin + j] == token;
        if (again) continue;
        if (u * left < p) {
          stands = child;
          break;
        }
        left -= p;
        if (lane == fallen) fallen_token = token;
        ++fallen;
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
      if (writes && lane == 0) a.next[request] = best;
      break;
    }
    const double u = a.uniform[begin];
    const bool plain = !(left > 0.0) || (fallen == 0 && b == 0.0);      // (nothing left but by rounding: p itself)
    const bool listed = !plain && fallen > 0;      // the fallen children's tokens weigh nothing
    // has token base + lane fallen? (the warp asks together)
    auto fell = [&](int id) {
      bool out = false;
      for (int f = 0; f < min(fallen, 32); ++f) out |= id == __shfl_sync(0xffffffffu, fallen_token, f);
      if (fallen > 32)
        for (int j = child_of(node, node); j < nodes; j = child_of(node, j)) out |= a.ids[begin + j] == id;
      return out;
    };
    auto weight = [&](int id) {
      if (plain || listed) return of_p(row[id]) * p_unit;
      const double over = of_p(row[id]) * p_unit - b * (of_q(draft[id]) * q_unit);
      return over > 0.0 ? over : 0.0;
    };
    // every warp's sum: p's from the row's first exchange, what is over from that of the last fallen
    // child, otherwise told now
    const bool first_sums = plain && b == 0.0;
    if (listed || (plain && !first_sums)) {
      double sum = 0.0;
      for (int base = first; base < last; base += 32) {
        const bool out = listed && fell(base + lane);
        if (base + lane < last && !out) sum += weight(base + lane);
      }
      mine.p_sum = warp_sum(sum);
      tell(mine);
    }
    auto sum_of = [&](int w) {
      const Told& of = told[phase][w];
      return !first_sums ? of.p_sum : of.p_sum > 0.0 ? of.p_sum * of_p(of.p_max) * p_unit : 0.0;
    };
    // the stretch in which the running sum passes the target; all warps add alike and agree on it
    const int each = (owners + 31) / 32, own_first = min(lane * each, owners), own_last = min(own_first + each, owners);
    double lane_sum = 0.0;
    int owner = -1;
    for (int w = own_first; w < own_last; ++w) {
      const double sum = sum_of(w);
      lane_sum += sum;
      if (sum > 0.0) owner = w;
    }
    double inclusive_sum = lane_sum;
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1) {
      const double other = __shfl_up_sync(0xffffffffu, inclusive_sum, offset);
      if (lane >= offset) inclusive_sum += other;
    }
    const double target = u * __shfl_sync(0xffffffffu, inclusive_sum, 31);
    const unsigned beyond = __ballot_sync(0xffffffffu, owner >= 0 && target < inclusive_sum);
    const unsigned weighs = __ballot_sync(0xffffffffu, owner >= 0);
    // (a sum that falls short by rounding: the last stretch with any weight)
    const int source = beyond != 0u ? __ffs(beyond) - 1 : 31 - __clz(weighs | 1u);
    double before = inclusive_sum - lane_sum;
    if (beyond != 0u) {
      double running = before;
      for (int w = own_first; w < own_last; ++w) {
        const double sum = sum_of(w);
        if (sum > 0.0 && target < running + sum) {
          owner = w;
          break;
        }
        running += sum;
      }
      before = running;
    }
    owner = __shfl_sync(0xffffffffu, owner, source);
    before = __shfl_sync(0xffffffffu, before, source);
    if (owner == me) {
      int chosen = -1, last_with_weight = -1;
      for (int base = first; base < last && chosen < 0; base += 32) {
        const int id = base + lane;
        const bool out = listed && fell(id);
        const double w = id < last && !out ? weight(id) : 0.0;
        double inclusive = w;
#pragma unroll
        for (int offset = 1; offset < 32; offset <<= 1) {
          const double other = __shfl_up_sync(0xffffffffu, inclusive, offset);
          if (lane >= offset) inclusive += other;
        }
        const unsigned passed = __ballot_sync(0xffffffffu, w > 0.0 && target < before + inclusive);
        const unsigned heavy = __ballot_sync(0xffffffffu, w > 0.0);
        if (heavy != 0u) last_with_weight = base + 31 - __clz(heavy);
        if (passed != 0u) chosen = base + __ffs(passed) - 1;
        before += __shfl_sync(0xffffffffu, inclusive, 31);
      }
      if (chosen < 0) chosen = last_with_weight;      // the running sum fell short by rounding
      if (lane == 0) a.next[request] = chosen;
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
  // as many CTAs a request as leave two an SM, and no more than have 32 x 4 tokens a warp
  int ctas = MAX_CLUSTER;
  while (ctas > 1 && (static_cast<long long>(requests) * ctas > 2ll * sms || vocab <= (ctas / 2) * WARPS * 128)) ctas /= 2;
  HX_REQUIRE(requests <= (1 << 24), "hx_verify_drafts: too many requests");
  int span = (vocab + ctas * WARPS - 1) / (ctas * WARPS);
  span = (span + 127) / 128 * 128;
  VerifyArgs a{logits, ld, draft, ld_draft, token_ids, parents, request_start, temperature, uniform, path, ld_path,
               width, kept, next_tokens, vocab, span, put_back, status};
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(requests * ctas);
  config.blockDim = dim3(THREADS);
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
