// Part of unpacked.hip, included inside its anonymous namespace: what lies around the two products of a routed-expert layer on stacked matrices.
//
//   k_expert_order    pairs (token, slot) sorted by expert, in their own order within one: ends of the experts, token of each position, position of
//                     each pair
//   product           silu(gate) * up of every pair, in the activations' type or in e4m3 (few pairs: gate and up in float32, then k_gated); for int8 in float32, which
//                     k_round_rows rounds by row (few pairs: gate and up, then both by k_round_rows)
//   product           down, float32
//   k_weighted_sum    y_t = sum_j w_tj out(t, j), j ascending
//
// The hidden values are rounded between the products, to the type of the matrices: that is what the second product's instructions take.  In float32 they would
// need two 16-bit parts each, twice the instructions and the bytes; the packed layer (htr_moe_experts) rounds them as well.  In bfloat16 a layer's result is off by
// 2.3e-3 in the 2-norm, of which 1.7e-3 are its own last rounding.

// One workgroup for each expert counts the pairs of smaller experts and its own, then places its own: no atomics, no order but the pairs'.  A wave takes a run of
// consecutive pairs, 64 at a time, and keeps up to KEEP of them to a lane between the two.  A pair whose expert is out of range has position -1.  24576 pairs,
// 64 experts: 11 us (16 with eight loads on their way at a time, read again for the second pass, and tokens by integer division).
constexpr int ORDER_WAVES = 16;
__device__ __forceinline__ void expert_order(const void* __restrict__ ids, int ids64, int pairs, int top, int experts, int* __restrict__ ends, int* __restrict__ token,
                                             int* __restrict__ pos_of, int e) {
  __shared__ int s_less[ORDER_WAVES], s_same[ORDER_WAVES];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = (pairs + ORDER_WAVES * 64 - 1) / (ORDER_WAVES * 64) * 64, p0 = min(pairs, wv * per), p1 = min(pairs, p0 + per);
  // -1 for an expert out of range, or no pair
  constexpr int AHEAD = 8, KEEP = 4;
  auto load = [&](int q, int (&v)[AHEAD]) {
    long long id[AHEAD];
    if (ids64) {
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) id[k] = ((const HTR_GLOBAL long long*)ids)[min(q + 64 * k + lane, pairs - 1)];
    } else {
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) id[k] = ((const HTR_GLOBAL int*)ids)[min(q + 64 * k + lane, pairs - 1)];
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) v[k] = (((unsigned long long)id[k] >= (unsigned long long)experts) | (q + 64 * k + lane >= p1)) ? -1 : (int)id[k];
  };
  int less = 0, same = 0;
  auto count = [&](int q, const int (&v)[AHEAD]) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      less += (int)__builtin_popcountll(__ballot((uint32_t)v[k] < (uint32_t)e));      // -1 is none
      same += (int)__builtin_popcountll(__ballot(v[k] == e));
    }
    if (e == 0) {
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) if (v[k] < 0 && q + 64 * k + lane < p1) pos_of[q + 64 * k + lane] = -1;
    }
  };
  int at = 0;
  const double each = 1.0 / top;
  auto put = [&](int q, const int (&v)[AHEAD]) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const unsigned long long mine = __ballot(v[k] == e);
      if (v[k] == e) {
        const int p = q + 64 * k + lane, pos = __builtin_amdgcn_mbcnt_hi((uint32_t)(mine >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mine, at));
        token[pos] = (int)__builtin_fma((double)p, each, 0.5 * each);      // p / top: half a pair away from the next whole number, where 64 bits are off by 2^-22 of one
        pos_of[p] = pos;
      }
      at += (int)__builtin_popcountll(mine);
    }
  };
  int kept[KEEP][AHEAD];
#pragma unroll
  for (int j = 0; j < KEEP; ++j) if (p0 + j * 64 * AHEAD < p1) load(p0 + j * 64 * AHEAD, kept[j]);
#pragma unroll
  for (int j = 0; j < KEEP; ++j) if (p0 + j * 64 * AHEAD < p1) count(p0 + j * 64 * AHEAD, kept[j]);
  for (int q = p0 + KEEP * 64 * AHEAD; q < p1; q += 64 * AHEAD) {
    int v[AHEAD];
    load(q, v);
    count(q, v);
  }
  if (lane == 0) { s_less[wv] = less; s_same[wv] = same; }
  __syncthreads();
  int total = 0;
  for (int k = 0; k < ORDER_WAVES; ++k) {
    at += s_less[k] + (k < wv ? s_same[k] : 0);
    total += s_less[k] + s_same[k];
  }
  if (threadIdx.x == 0) ends[e] = total;
  if (same == 0) return;
#pragma unroll
  for (int j = 0; j < KEEP; ++j) if (p0 + j * 64 * AHEAD < p1) put(p0 + j * 64 * AHEAD, kept[j]);
  for (int q = p0 + KEEP * 64 * AHEAD; q < p1; q += 64 * AHEAD) {
    int v[AHEAD];
    load(q, v);
    put(q, v);
  }
}
__global__ __launch_bounds__(ORDER_WAVES * 64) void k_expert_order(const void* __restrict__ ids, int ids64, int pairs, int top, int experts, int* __restrict__ ends,
                                                                   int* __restrict__ token, int* __restrict__ pos_of) {
  expert_order(ids, ids64, pairs, top, experts, ends, token, pos_of, blockIdx.x);
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
