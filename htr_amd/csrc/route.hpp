// Part of unpacked.hip, included inside its anonymous namespace: a router's logits to each token's experts and their weights.
//
//   s_e = softmax_e(l) or 1 / (1 + exp(-l_e));   r_e = s_e + b_e, without a bias l_e, of which s_e is a growing function
//   groups: the sum of a group's `group_best` largest s_e + b_e ranks it; experts of the best `top_groups` groups compete (one best, no bias: by l_e)
//   the `top` largest r_e in descending order, ties to the lowest number;  weights s_e, over their sum if `renormalize`, times `scale`
//
// A logit or bias of -inf masks its expert: it comes behind every other, with weight 0; a token of which every expert is masked has weights 0.  NaN ranks first.
// Scores and ranks are 64 bits: experts' ranks lie within 2^-24 of each other in one token of some thousand, and an expert taken for its neighbour is another result.
constexpr int ROUTE_MOST = 1024, ROUTE_WAVES = 4;

struct RouteArgs {
  const void* logits;                 // [tokens][experts], `stride` elements from token to token
  const float* bias;                  // [experts] or NULL
  int* ids;                           // [tokens][top]
  float* weights;
  long long stride, tokens;
  int dtype, experts, top, sigmoid, groups, top_groups, group_best, renormalize;
  double scale;
};

// ranks as integers of the same order: -0 as 0, NaN (of either sign) above all
__device__ __forceinline__ long long order_of(double v) {
  if (!(v == v)) return 0x7FFFFFFFFFFFFFFFll;
  const long long u = __builtin_bit_cast(long long, v + 0.0);
  return u < 0 ? u ^ 0x7FFFFFFFFFFFFFFFll : u;
}
constexpr long long ORDER_MASKED = (long long)0x800FFFFFFFFFFFFFull;      // order_of(-inf)
constexpr long long ORDER_NONE = (long long)0x8000000000000000ull;        // no expert, or one that is taken
template <typename V> __device__ __forceinline__ V wave_largest(V v) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) { const V w = __shfl_xor(v, off); v = w > v ? w : v; }
  return v;
}

// One wave to a token, PER consecutive experts to a lane
template <int PER>
__global__ __launch_bounds__(ROUTE_WAVES * 64) void k_route(const RouteArgs a) {
  const int lane = threadIdx.x & 63;
  const long long token = (long long)blockIdx.x * ROUTE_WAVES + (threadIdx.x >> 6);
  if (token >= a.tokens) return;
  double l[PER], score[PER], most = -INFINITY;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = lane * PER + j;
    l[j] = e < a.experts ? (double)load_elem_g(a.logits, a.dtype, (size_t)(token * a.stride) + e) : -INFINITY;
    most = fmax(most, l[j]);
  }
  if (a.sigmoid) {
#pragma unroll
    for (int j = 0; j < PER; ++j) score[j] = 1.0 / (1.0 + exp(-l[j]));
  } else {
    most = wave_largest(most);
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j) { score[j] = l[j] == -INFINITY ? 0.0 : exp(l[j] - most); sum += score[j]; }
    sum = wave_sum(sum);
#pragma unroll
    for (int j = 0; j < PER; ++j) score[j] = sum == 0.0 ? 0.0 : score[j] / sum;
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
    const int size = a.experts / a.groups;
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
        sum += __shfl(value, e / PER);
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
