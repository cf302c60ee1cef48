// Part of unpacked.hip, included inside its anonymous namespace: what lies around the two products of a routed-expert layer on stacked matrices.
//
//   k_expert_order    pairs (token, slot) sorted by expert, in their own order within one: ends of the experts, token of each position, position of
//                     each pair
//   product           gate and up of every pair, float32
//   k_gated           silu(gate) * up, to the activations' type or to e4m3
//   product           down, float32
//   k_weighted_sum    y_t = sum_j w_tj out(t, j), j ascending

// One workgroup for each expert counts the pairs of smaller experts and its own, then places its own: no atomics, no order but the pairs'.  A
// thread takes a run of consecutive pairs.  A pair whose expert is out of range has position -1.
constexpr int ORDER_THREADS = 1024;
__global__ __launch_bounds__(ORDER_THREADS) void k_expert_order(const void* __restrict__ ids, int ids64, int pairs, int top, int experts,
                                                                int* __restrict__ ends, int* __restrict__ token, int* __restrict__ pos_of) {
  __shared__ int s_less[16], s_same[16];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, e = blockIdx.x;
  const int per = (pairs + ORDER_THREADS - 1) / ORDER_THREADS, p0 = min(pairs, tid * per), p1 = min(pairs, p0 + per);
  auto id_of = [&](int p) { return ids64 ? ((const HTR_GLOBAL long long*)ids)[p] : (long long)((const HTR_GLOBAL int*)ids)[p]; };
  int less = 0, same = 0;
  for (int p = p0; p < p1; ++p) {
    const long long v = id_of(p);
    less += v >= 0 && v < e;
    same += v == e;
    if (e == 0 && (v < 0 || v >= experts)) pos_of[p] = -1;
  }
  int incl = same;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) { const int u = __shfl_up(incl, off); if (lane >= off) incl += u; }
#pragma unroll
  for (int off = 32; off; off >>= 1) less += __shfl_xor(less, off);
  if (lane == 63) { s_less[wv] = less; s_same[wv] = incl; }
  __syncthreads();
  int at = incl - same, total = 0;
  for (int k = 0; k < ORDER_THREADS / 64; ++k) {
    at += s_less[k] + (k < wv ? s_same[k] : 0);
    total += s_less[k] + s_same[k];
  }
  if (tid == 0) ends[e] = total;
  for (int p = p0; same > 0 && p < p1; ++p)
    if (id_of(p) == e) { token[at] = p / top; pos_of[p] = at++; }
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
    for (int k = 0; k < 8; ++k) f[k] = g.get(k) / (1.f + expf(-g.get(k))) * u.get(k);
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
