// Part of unpacked.hip, included inside its anonymous namespace: what lies around the two products of a routed-expert layer on stacked matrices.
//
//   k_expert_order    pairs (token, slot) sorted by expert, in their own order within one: ends of the experts, token of each position, position of
//                     each pair
//   product           silu(gate) * up of every pair, in the activations' type or in e4m3 (few pairs: gate and up in float32, then k_gated)
//   product           down, float32
//   k_weighted_sum    y_t = sum_j w_tj out(t, j), j ascending
//
// The hidden values are rounded between the products, to the type of the matrices: that is what the second product's instructions take.  In float32 they would
// need two 16-bit parts each, twice the instructions and the bytes; the packed layer (htr_moe_experts) rounds them as well.  In bfloat16 a layer's result is off by
// 2.3e-3 in the 2-norm, of which 1.7e-3 are its own last rounding.

// One workgroup for each expert counts the pairs of smaller experts and its own, then places its own: no atomics, no order but the pairs'.  A wave takes a run of
// consecutive pairs, 64 at a time.  A pair whose expert is out of range has position -1.  24576 pairs, 64 experts: 16 us (34 with a run to each thread).
constexpr int ORDER_WAVES = 16;
__global__ __launch_bounds__(ORDER_WAVES * 64) void k_expert_order(const void* __restrict__ ids, int ids64, int pairs, int top, int experts,
                                                                   int* __restrict__ ends, int* __restrict__ token, int* __restrict__ pos_of) {
  __shared__ int s_less[ORDER_WAVES], s_same[ORDER_WAVES];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), e = blockIdx.x;
  const int per = (pairs + ORDER_WAVES * 64 - 1) / (ORDER_WAVES * 64) * 64, p0 = min(pairs, wv * per), p1 = min(pairs, p0 + per);
  // AHEAD loads on their way at once: -1 for an expert out of range, or no pair
  constexpr int AHEAD = 8;
  auto load = [&](int q, int (&v)[AHEAD]) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int p = min(q + 64 * k + lane, pairs - 1);
      const long long id = ids64 ? ((const HTR_GLOBAL long long*)ids)[p] : (long long)((const HTR_GLOBAL int*)ids)[p];
      v[k] = id < 0 || id >= experts || q + 64 * k + lane >= p1 ? -1 : (int)id;
    }
  };
  int less = 0, same = 0;
  for (int q = p0; q < p1; q += 64 * AHEAD) {
    int v[AHEAD];
    load(q, v);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      less += (int)__builtin_popcountll(__ballot(v[k] >= 0 && v[k] < e));
      same += (int)__builtin_popcountll(__ballot(v[k] == e));
      if (e == 0 && v[k] < 0 && q + 64 * k + lane < p1) pos_of[q + 64 * k + lane] = -1;
    }
  }
  if (lane == 0) { s_less[wv] = less; s_same[wv] = same; }
  __syncthreads();
  int at = 0, total = 0;
  for (int k = 0; k < ORDER_WAVES; ++k) {
    at += s_less[k] + (k < wv ? s_same[k] : 0);
    total += s_less[k] + s_same[k];
  }
  if (threadIdx.x == 0) ends[e] = total;
  if (same == 0) return;
  for (int q = p0; q < p1; q += 64 * AHEAD) {
    int v[AHEAD];
    load(q, v);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const unsigned long long mine = __ballot(v[k] == e);
      if (mine >> lane & 1ull) {
        const int p = q + 64 * k + lane, pos = at + (int)__builtin_popcountll(mine & ((1ull << lane) - 1ull));
        token[pos] = p / top;
        pos_of[p] = pos;
      }
      at += (int)__builtin_popcountll(mine);
    }
  }
}

// silu(gate) * up, eight columns to a thread
template <int OUT>      // HTR_BF16, HTR_F16 or P_F8
__global__ __launch_bounds__(256) void k_gated(const float* __restrict__ h, const int* __restrict__ ends, int experts, int F, void* __restrict__ y,
                                               float* __restrict__ scales) {
  const int pos = blockIdx.x;
  if (pos >= ends[experts - 1]) return;
  for (int c = 8 * threadIdx.x; c < F; c += 8 * 256) {
    Eight<HTR_F32> g, u;
    g.load(h, (size_t)pos * 2 * F + c);
    u.load(h, (size_t)pos * 2 * F + F + c);
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = silu(g.get(k)) * u.get(k);
    if constexpr (OUT == P_F8) {
      float scale;
      *(HTR_GLOBAL u2*)((HTR_GLOBAL uint8_t*)y + (size_t)pos * F + c) = quantize8(f, scale);
      if ((threadIdx.x & 15) == 0) ((HTR_GLOBAL float*)scales)[(size_t)pos * (F >> 7) + (c >> 7)] = scale;
    } else {
      Eight<OUT> v;
      v.set(f);
      v.store(y, (size_t)pos * F + c);
    }
  }
}

template <int T>
__global__ __launch_bounds__(256) void k_weighted_sum(const float* __restrict__ out, const int* __restrict__ pos_of, const float* __restrict__ wt, int top,
                                                      int H, void* __restrict__ y) {
  const int t = blockIdx.x, c = 8 * (blockIdx.y * 256 + threadIdx.x);
  if (c >= H) return;
  float s[8] = {};
  for (int j = 0; j < top; ++j) {
    const int p = pos_of[(size_t)t * top + j];                   // uniform
    const float w = p < 0 ? __builtin_nanf("") : wt[(size_t)t * top + j];
    Eight<HTR_F32> v;
    v.load(out, (size_t)(p < 0 ? 0 : p) * H + c);
#pragma unroll
    for (int k = 0; k < 8; ++k) s[k] += v.get(k) * w;
  }
  Eight<T> v;
  v.set(s);
  v.store(y, (size_t)t * H + c);
}
