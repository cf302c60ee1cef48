// Part of unpacked.hip, included inside its anonymous namespace: a router's logits to each token's experts and their weights.
//
//   s_e = softmax_e(l) or 1 / (1 + exp(-l_e));   r_e = s_e + b_e, without a bias l_e, of which s_e is a growing function
//   groups: the sum of a group's `group_best` largest s_e + b_e ranks it; experts of the best `top_groups` groups compete (one best, no bias: by l_e).  Masked experts
//   add nothing to it: a group with one expert left is as good as that one, one with none comes behind all others
//   the `top` largest r_e in descending order, ties to the lowest number;  weights s_e, over their sum if `renormalize`, times `scale`
//
// A logit or bias of -inf masks its expert: it comes behind every other, with weight 0; a token of which every expert is masked has weights 0.  NaN ranks first.
// Scores and ranks are 64 bits: experts' ranks lie within 2^-24 of each other in one token of some thousand, and an expert taken for its neighbour is another result.
// One wave to a token.  Ranks that are logits are float32 as they are; others are first formed in float32, and only those that lie within what float32 may be off of each
// other, or of what decides, are compared in 64 bits (Route); what that does not cover is done in 64 bits throughout (route_exact).  The weights of the chosen are
// 64 bits either way.
// 8 of 256 experts, sigmoid, bias, 4 of 8 groups: 16384 tokens 17 us, where their 17 MB take 2.4; 427 vector and 351 scalar instructions a token, the vector units busy in
// four fifths of the time.  6 of 64 by softmax: 1 token 2.8 us, 500 tokens 4.7, less than the host takes for the call.  In 64 bits throughout 16384 tokens take 127; four tokens
// to a wave, finished together, 19; a wave that goes on from token to token 31 (the 64-bit constants kept in registers leave it too few neighbours).
constexpr int ROUTE_MOST = 1024, ROUTE_WAVES = 4;

struct RouteArgs {
  const void* logits;                 // [tokens][experts], `stride` elements from token to token
  const float* bias;                  // [experts] or NULL
  int* ids;                           // [tokens][top]
  float* weights;
  long long stride, tokens;
  int dtype, experts, top, sigmoid, groups, top_groups, group_best, renormalize;
  double scale;
  int size, parts_log2;               // experts of a group, lanes to a group
};

// ranks as integers of the same order: -0 as 0, NaN (of either sign) above all
__device__ __forceinline__ long long order_of(double v) {
  if (!(v == v)) return 0x7FFFFFFFFFFFFFFFll;
  const long long u = __builtin_bit_cast(long long, v + 0.0);
  return u < 0 ? u ^ 0x7FFFFFFFFFFFFFFFll : u;
}
constexpr long long ORDER_MASKED = (long long)0x800FFFFFFFFFFFFFull;      // order_of(-inf)
constexpr long long ORDER_NONE = (long long)0x8000000000000000ull;        // no expert, or one that is taken
// the same of float32 that is not NaN, in unsigned numbers from 1 on (0: no expert)
__device__ __forceinline__ uint32_t key_of_sum(float v) {                // that is not -0
  const uint32_t u = __float_as_uint(v);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint32_t key_of(float v) { return key_of_sum(v + 0.f); }
__device__ __forceinline__ float value_of_key(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }
constexpr uint32_t KEY_MASKED = 0x007FFFFFu;                             // of -inf

template <typename V> __device__ __forceinline__ V wave_largest(V v) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) { const V w = __shfl_xor(v, off); v = w > v ? w : v; }
  return v;
}
// 1 / x for x from 2^-1000 to 2^1000, off by 2^-51 at most: the instruction's 24 bits doubled twice.  A quotient as the language defines it takes four times the instructions.
__device__ __forceinline__ double inverse64(double x) {
  double r = __builtin_amdgcn_rcp(x);
  r = __builtin_fma(__builtin_fma(-x, r, 1.0), r, r);
  return __builtin_fma(__builtin_fma(-x, r, 1.0), r, r);
}
// e^x for x <= 0: 2^k times the series of e^r to r^13 for r = x - k log 2, |r| <= 0.347 (the next term is 4e-18); 0 where 64 bits hold nothing else
__device__ __forceinline__ double exp64(double x) {
  const double k = rint(x * 1.4426950408889634);
  const double r = __builtin_fma(k, -2.3190468138462996e-17, __builtin_fma(k, -0.6931471805599453, x));      // log 2 in two parts
  double p = 1.0 / 6227020800.0;
  p = __builtin_fma(p, r, 1.0 / 479001600.0); p = __builtin_fma(p, r, 1.0 / 39916800.0); p = __builtin_fma(p, r, 1.0 / 3628800.0); p = __builtin_fma(p, r, 1.0 / 362880.0);
  p = __builtin_fma(p, r, 1.0 / 40320.0); p = __builtin_fma(p, r, 1.0 / 5040.0); p = __builtin_fma(p, r, 1.0 / 720.0); p = __builtin_fma(p, r, 1.0 / 120.0);
  p = __builtin_fma(p, r, 1.0 / 24.0); p = __builtin_fma(p, r, 1.0 / 6.0); p = __builtin_fma(p, r, 0.5); p = __builtin_fma(p, r, 1.0); p = __builtin_fma(p, r, 1.0);
  return x < -746.0 ? 0.0 : __builtin_ldexp(p, (int)k);
}
__device__ __forceinline__ double sigmoid64(double l) {
  const double e = exp64(-fabs(l)), r = inverse64(1.0 + e);
  return l < 0.0 ? e * r : r;
}

// ---- in 64 bits: PER consecutive experts to a lane, the largest taken one after the other
template <int PER> __device__ __forceinline__ void route_exact(const RouteArgs& a, long long token, int lane) {
  double l[PER], score[PER], most = -INFINITY;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = lane * PER + j;
    l[j] = e < a.experts ? (double)load_elem_g(a.logits, a.dtype, (size_t)(token * a.stride) + e) : -INFINITY;
    most = fmax(most, l[j]);
  }
  if (a.sigmoid) {
#pragma unroll
    for (int j = 0; j < PER; ++j) score[j] = sigmoid64(l[j]);
  } else {
    most = wave_largest(most);
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j) { score[j] = l[j] == -INFINITY ? 0.0 : exp64(l[j] - most); sum += score[j]; }
    sum = wave_sum(sum);
#pragma unroll
    for (int j = 0; j < PER; ++j) score[j] = sum == 0.0 ? 0.0 : score[j] * inverse64(sum);
  }
  long long rank[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = lane * PER + j;
    const float b = a.bias != nullptr && e < a.experts ? ((const HTR_GLOBAL float*)a.bias)[e] : 0.f;
    if (b == -INFINITY) l[j] = -INFINITY;
    rank[j] = e >= a.experts ? ORDER_NONE : l[j] == -INFINITY ? ORDER_MASKED : order_of(a.bias != nullptr ? score[j] + (double)b : l[j]);
  }
  if (a.groups > 1) {
    const int size = a.size;
    long long mine = ORDER_NONE;                    // lane g: what ranks group g
    for (int g = 0; g < a.groups; ++g) {
      double sum = 0.0;
      long long before = 0x7FFFFFFFFFFFFFFFll;
      int before_e = -1;
      for (int k = 0; k < min(a.group_best, size); ++k) {
        // the largest behind the one before, ties by number
        long long best = ORDER_NONE;
        double v[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const int e = lane * PER + j;
          if (e / size != g || e >= a.experts) continue;
          v[j] = l[j] == -INFINITY ? -INFINITY : a.bias != nullptr ? score[j] + (double)((const HTR_GLOBAL float*)a.bias)[e] : a.group_best > 1 ? score[j] : l[j];
          const long long o = order_of(v[j]);
          if ((o < before || (o == before && e > before_e)) && o > best) best = o;
        }
        const long long top = wave_largest(best);
        int first = 1 << 20;
        double value = 0.0;
#pragma unroll
        for (int j = PER - 1; j >= 0; --j) {
          const int e = lane * PER + j;
          if (e / size == g && e < a.experts && order_of(v[j]) == top && (top < before || e > before_e)) { first = e; value = v[j]; }
        }
        const int e = -wave_largest(-first);
        value = __shfl(value, e / PER);
        sum += k == 0 || top != ORDER_MASKED ? value : 0.0;
        before = top;
        before_e = e;
      }
      if (lane == g) mine = order_of(sum);
    }
    // a group is in where fewer than top_groups others are better, or as good and before it
    int better = 0;
    for (int g = 0; g < a.groups; ++g) {
      const long long other = __shfl(mine, g);
      better += other > mine || (other == mine && g < lane);
    }
    const unsigned long long in = __ballot(lane < a.groups && better < a.top_groups);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int e = lane * PER + j;
      if (e < a.experts && !(in >> (e / size) & 1ull)) rank[j] = ORDER_MASKED;
    }
  }
  // lane k keeps the k-th expert
  int id = 0;
  double weight = 0.0, total = 0.0;
  for (int k = 0; k < a.top; ++k) {
    long long best = ORDER_NONE;
#pragma unroll
    for (int j = 0; j < PER; ++j) best = rank[j] > best ? rank[j] : best;
    const long long top = wave_largest(best);
    const int owner = __builtin_ctzll(__ballot(best == top));
    int at = 0;
    double s = 0.0;
    bool found = false;
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (!found && rank[j] == top) { found = true; at = j; s = score[j]; if (lane == owner) rank[j] = ORDER_NONE; }
    const int e = owner * PER + __shfl(at, owner);
    s = top == ORDER_MASKED ? 0.0 : __shfl(s, owner);
    total += s;
    if (lane == k) { id = e; weight = s; }
  }
  if (lane < a.top) {
    if (a.renormalize) weight = total == 0.0 ? 0.0 : weight / total;
    ((HTR_GLOBAL int*)a.ids)[token * a.top + lane] = id;
    ((HTR_GLOBAL float*)a.weights)[token * a.top + lane] = (float)(weight * a.scale);
  }
}

// ---- with float32 ranks.  Lanes in runs of `parts` = 2^parts_log2 to a group (without groups: all 64); element i of lane p of group g is expert g size + p + i parts.
// The threshold between the chosen and the others is found by halving the span of ranks (as integers): a comparison and a count of lanes to each element, until exactly
// `top` lie above it, which takes about ten steps; the largest one by one takes a wave's maximum for each.  Whatever lies next to the threshold is a candidate, too, and
// candidates too close to each other are ordered by their ranks in 64 bits, groups likewise.
struct Candidate { uint32_t after, key; float l, b; };      // after: ~expert; with the key in front, a number for each candidate in descending order
__device__ __forceinline__ void two_largest(uint32_t& first, uint32_t& second, uint32_t f, uint32_t s) {      // of both
  second = max(max(second, s), min(first, f));
  first = max(first, f);
}
template <int H> __device__ __forceinline__ void two_largest(uint32_t& first, uint32_t& second) {                // with lane ^ H
  two_largest(first, second, __float_as_uint(lane_xor_dpp<H>(__uint_as_float(first))), __float_as_uint(lane_xor_dpp<H>(__uint_as_float(second))));
}
template <int PER> struct Route {
  const RouteArgs& a;
  const int lane, parts_log2, parts, g, p, e0;
  const bool biased, scored;      // scored: some ranks are no logits
  float l[PER], b[PER], most;     // a token's; most: the largest logit (softmax)
  bool odd_bias;                  // one that float32 sums are not for
  __device__ __forceinline__ Route(const RouteArgs& a, int lane)
      : a(a), lane(lane), parts_log2(a.parts_log2), parts(1 << a.parts_log2), g(lane >> a.parts_log2), p(lane & ((1 << a.parts_log2) - 1)), e0(g * a.size + p),
        biased(a.bias != nullptr), scored(a.bias != nullptr || (a.groups > 1 && a.group_best > 1)), odd_bias(false) {
#pragma unroll
    for (int i = 0; i < PER; ++i) b[i] = 0.f;
    if (biased) {
#pragma unroll
      for (int i = 0; i < PER; ++i) b[i] = ((const HTR_GLOBAL float*)a.bias)[at(i)];
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        b[i] = in(i) ? b[i] : 0.f;
        odd_bias |= (magnitude(b[i]) >= 0x5D800000u) & (b[i] != -INFINITY);      // 2^60
      }
    }
  }
  __device__ __forceinline__ bool in(int i) const { return (g < a.groups) & (p + i * parts < a.size); }
  __device__ __forceinline__ uint32_t at(int i) const { return (uint32_t)min(e0 + i * parts, a.experts - 1); }      // where it may be loaded from
  // All loads at once, none behind a condition of its lane
  __device__ __forceinline__ void load(long long token, float (&to)[PER]) const {
    if (a.dtype == HTR_F32) {
      const HTR_GLOBAL float* row = (const HTR_GLOBAL float*)a.logits + token * a.stride;
#pragma unroll
      for (int i = 0; i < PER; ++i) to[i] = row[at(i)];
    } else {
      const HTR_GLOBAL uint16_t* row = (const HTR_GLOBAL uint16_t*)a.logits + token * a.stride;
      uint32_t raw[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) raw[i] = row[at(i)];
      if (a.dtype == HTR_BF16) {
#pragma unroll
        for (int i = 0; i < PER; ++i) to[i] = __uint_as_float(raw[i] << 16);
      } else {
#pragma unroll
        for (int i = 0; i < PER; ++i) to[i] = f16_bits_to_float((uint16_t)raw[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) to[i] = in(i) ? to[i] : -INFINITY;
  }
  __device__ __forceinline__ double all64() const {      // the softmax's sum
    double total = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) total += l[i] == -INFINITY ? 0.0 : exp64((double)l[i] - (double)most);
    return wave_sum(total);
  }

  // The token's candidates: their number, at least `top`; 0 where ranks are no finite numbers, or there are more than 64
  __device__ __forceinline__ int select(Candidate* place) {
    const int top = a.top;
    bool odd = odd_bias;
    most = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; ++i) { odd |= !(l[i] < INFINITY); most = fmaxf(most, l[i]); }
    if (__ballot(odd)) return 0;
    if (!a.sigmoid) most = value_of_key(wave_max(key_of(most)));
    float score[PER];
    uint32_t key[PER];      // of the ranks
    if (scored) {
      if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < PER; ++i) score[i] = __builtin_amdgcn_rcpf(1.f + __expf(-l[i]));
      } else {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) { score[i] = __expf(l[i] - most); sum += score[i]; }
        sum = 1.f / wave_sum(sum);
#pragma unroll
        for (int i = 0; i < PER; ++i) score[i] *= sum;
      }
    }
    if (biased) {
#pragma unroll
      for (int i = 0; i < PER; ++i) key[i] = key_of_sum(l[i] == -INFINITY ? l[i] : score[i] + b[i]);      // a bias of -inf masks, too; scores are no -0
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) key[i] = key_of(l[i]);
    }
    // float32 ranks, and differences of two, are off by less: a score by 2 PER + 32 steps of 2^-24 at most (the exponential and its argument 6, the sum PER + 5, its
    // inverse and the product 3), the sum with the bias by one more of its own
    const float slack = (2 * PER + 32) * 0x1p-24f;
    bool out = g >= a.groups;
    if (a.groups > 1) {
      // a lane's two largest, then those of the group's lanes
      uint32_t k1 = KEY_MASKED, k2 = KEY_MASKED;
      const bool two = a.group_best > 1 && a.size > 1;
      if (biased || a.group_best == 1) {
#pragma unroll
        for (int i = 0; i < PER; ++i) two_largest(k1, k2, key[i], KEY_MASKED);
      } else {
#pragma unroll
        for (int i = 0; i < PER; ++i) two_largest(k1, k2, key[i] == KEY_MASKED ? KEY_MASKED : key_of(score[i]), KEY_MASKED);
      }
      if (parts > 1) two_largest<1>(k1, k2);
      if (parts > 2) two_largest<2>(k1, k2);
      if (parts > 4) two_largest<4>(k1, k2);
      if (parts > 8) two_largest<8>(k1, k2);
      if (parts > 16) {
        const u2s x = __builtin_amdgcn_permlane16_swap(k1, k1, false, false), y = __builtin_amdgcn_permlane16_swap(k2, k2, false, false);
        k1 = x.x; k2 = y.x;
        two_largest(k1, k2, x.y, y.y);
      }
      const float first = value_of_key(k1), second = value_of_key(k2);
      // each group's lanes compare it with as many others at once
      const unsigned long long own = ((1ull << parts) - 1) << (g << parts_log2);
      auto count_better = [&](auto mine, auto near, bool& close) {
        int better = 0;
        for (int k = 0; k < a.groups; k += parts) {
          const auto other = __shfl(mine, (k + p) << parts_log2);
          const bool there = k + p < a.groups;
          better += (int)__builtin_popcountll(__ballot(there & ((other > mine) | ((other == mine) & (k + p < g)))) & own);
          close |= there & (k + p != g) & !(other > mine + near) & !(other < mine - near);
        }
        return better;
      };
      const float mine = two && k2 != KEY_MASKED ? first + second : first;
      bool close = false, none = false;
      int better = count_better(mine, 2.f * slack * (1.f + fabsf(mine)), close);
      // groups so close that float32 does not tell which is better count where one of them may be in and another out
      if (scored && __ballot(close && g < a.groups && mine > -INFINITY && better <= a.top_groups && better >= a.top_groups - 1)) {
        const double over = a.sigmoid ? 1.0 : inverse64(all64());
        double first = -INFINITY, second = -INFINITY;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const double v = key[i] == KEY_MASKED ? -INFINITY : (a.sigmoid ? sigmoid64(l[i]) : exp64((double)l[i] - (double)most) * over) + (double)b[i];
          second = fmax(second, fmin(first, v));
          first = fmax(first, v);
        }
        for (int off = 1; off < parts; off <<= 1) {
          const double f = __shfl_xor(first, off), s = __shfl_xor(second, off);
          second = fmax(fmax(second, s), fmin(first, f));
          first = fmax(first, f);
        }
        better = count_better(two && second != -INFINITY ? first + second : first, 0.0, none);
      }
      out |= better >= a.top_groups;
    }
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      key[i] = out ? KEY_MASKED : key[i];
      key[i] = in(i) ? key[i] : 0u;
      largest = max(largest, key[i]);
    }
    largest = __builtin_amdgcn_readfirstlane(wave_max(largest));
    auto count = [&](uint32_t from) {
      int n = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) n += (int)__builtin_popcountll(__ballot(key[i] >= from));
      return n;
    };
    // at least `top` from lo on, fewer from hi on
    uint32_t hi = largest + 1, lo, step = 1u << 20;
    int n;
    for (;;) {
      lo = hi > step ? hi - step : 1u;
      n = count(lo);
      if (n >= top) break;
      hi = lo;
      step = min(step * 4, 1u << 28);
    }
    while (n != top && hi - lo > 1) {
      const uint32_t mid = lo + ((hi - lo) >> 1);
      const int m = count(mid);
      if (m >= top) { lo = mid; n = m; } else hi = mid;
    }
    bool taken[PER];
    if ((biased && lo > KEY_MASKED) || n == top) {
      if (biased && lo > KEY_MASKED) {
        const float t = value_of_key(lo);
        lo = __builtin_amdgcn_readfirstlane(key_of(t - slack * (1.f + fabsf(t))));
        n = count(lo);
        if (n > 64) return 0;
      }
#pragma unroll
      for (int i = 0; i < PER; ++i) taken[i] = key[i] >= lo;
    } else {
      // lo itself is the rank of several, of which the first by number are taken
      int ahead = 0;
      unsigned long long at[PER];
      const unsigned long long mine = (parts == 64 ? ~0ull : (1ull << parts) - 1) << (g << parts_log2), before = (1ull << (g << parts_log2)) - 1, lower = (1ull << lane) - 1;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        at[i] = __ballot(key[i] == lo);
        ahead += (int)__builtin_popcountll(__ballot(key[i] > lo)) + (int)__builtin_popcountll(at[i] & before);
      }
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int here = ahead + (int)__builtin_popcountll(at[i] & mine & lower);
        ahead += (int)__builtin_popcountll(at[i] & mine);
        taken[i] = key[i] > lo || (key[i] == lo && here < top);
      }
      n = top;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const unsigned long long lanes = __ballot(taken[i]);
      if (taken[i])
        place[__builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0))] = Candidate{~(uint32_t)(e0 + i * parts), key[i], l[i], b[i]};
      place += (int)__builtin_popcountll(lanes);
    }
    return n;
  }

  // Of n candidates, one to a lane, the chosen in order with their weights
  __device__ __forceinline__ void finish(Candidate* place, long long token, int n) const {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int top = a.top;
    const Candidate c = lane < n ? place[lane] : Candidate{0u, KEY_MASKED, -INFINITY, 0.f};
    const bool none = c.key == KEY_MASKED;
    const uint32_t e = ~c.after;
    auto number = [](const Candidate& c) { return (unsigned long long)c.key << 32 | c.after; };
    const unsigned long long mine = number(c);
    int order = 0;
    for (int j = 0; j < n; ++j) order += number(place[j]) > mine;
    bool close = false;
    if (biased) {
      // each one's rank to its place, where the one before it looks
      const float v = value_of_key(c.key);
      if (lane < n) place[order].l = v;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      close = (order + 1 < n) & (fabsf(v - place[min(order + 1, 63)].l) <= (2 * PER + 32) * 0x1p-24f * (1.f + fabsf(v)));
    }
    // scores of the candidates; of the softmax over the sum of all only where that does not cancel
    double w = a.sigmoid ? sigmoid64(c.l) : exp64((double)c.l - (double)most);
    w = none ? 0.0 : w;
    if (!a.sigmoid && most > -INFINITY && (!a.renormalize || biased)) w *= inverse64(all64());
    if (__ballot(close & !none)) {
      const long long rank = none ? ORDER_MASKED : order_of(w + (double)c.b);
      order = 0;
      for (int j = 0; j < n; ++j) {
        const long long other = __shfl(rank, j);
        order += (other > rank) | ((other == rank) & (place[j].after > c.after));
      }
    }
    const bool chosen = lane < n && order < top;
    if (a.renormalize) {
      double all = chosen ? w : 0.0;
      if (n > 16) {
        all = wave_sum(all);
      } else {      // in the first 16 lanes, which have them all
        all += dpp_mov64<0xB1>(all); all += dpp_mov64<0x4E>(all); all += dpp_mov64<0x141>(all); all += dpp_mov64<0x140>(all);
      }
      w = all > 0x1p-1000 ? w * inverse64(all) : all == 0.0 ? 0.0 : w / all;
    }
    if (chosen) {
      ((HTR_GLOBAL int*)a.ids + token * top)[order] = (int)e;
      ((HTR_GLOBAL float*)a.weights + token * top)[order] = (float)(w * a.scale);
    }
  }
};

template <int PER>
__global__ __launch_bounds__(ROUTE_WAVES * 64) void k_route(const RouteArgs a) {
  __shared__ Candidate candidates[ROUTE_WAVES][64];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long token = (long long)blockIdx.x * ROUTE_WAVES + wv;
  if (token >= a.tokens) return;
  Route<PER> r(a, lane);
  r.load(token, r.l);
  const int n = r.select(candidates[wv]);
  if (n == 0) route_exact<(PER < 16 ? PER : 16)>(a, token, lane);
  else r.finish(candidates[wv], token, n);
}
