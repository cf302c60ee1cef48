// Part of unpacked.hip, included inside its anonymous namespace: rows in 8-bit integers with one scale each.
//
//   s = float32(max(max_c |y_c|, 2^-100) / 127),   q_c = y_c / s to the nearest integer, halves away from zero;   a row with an infinity or NaN: s = NaN, q = 0
//
// of rows as they are, of normed ones (y as in norm.hpp, not rounded before) and of silu(gate) up.  A step is 1/127 of a row's largest value, so a quotient next to
// a half decides by as much as one outlier may be worth of the small ones: quotients are formed in 64 bits, and with halves away from zero they need no division.
// y / s is y f with f = (1 / s)(1 + 2^-50): what is a half of an integer, exactly, lies beyond it then, and everything else is 2^-32 of itself or more away from one
// (numerator and denominator have 24 bits).  Added to 1.5 2^52, one fused operation leaves the integer in the low bits.
// Bound: HBM, rows read once and kept in registers between the two passes: 24576 rows of 1408 float32 29 us (6.0 TB/s), the norm with a residual of 333 rows of 4096 in f16
// 5.7 us, of one 2.6.

constexpr int I8_MOST = 32768;              // columns of a row in registers: 1024 threads by four runs of eight

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }      // ordered as the values are, NaN behind infinity
__device__ __forceinline__ unsigned long long magnitude(double v) { return __builtin_bit_cast(unsigned long long, v) & 0x7FFFFFFFFFFFFFFFull; }
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  auto by = [](uint32_t v, uint32_t w) { return v > w ? v : w; };
  v = by(v, __float_as_uint(dpp_mov<0xB1>(__uint_as_float(v)))); v = by(v, __float_as_uint(dpp_mov<0x4E>(__uint_as_float(v))));
  v = by(v, __float_as_uint(dpp_mov<0x141>(__uint_as_float(v)))); v = by(v, __float_as_uint(dpp_mov<0x140>(__uint_as_float(v))));
  u2s r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = by(r.x, r.y);
  r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return by(r.x, r.y);
}
__device__ __forceinline__ unsigned long long wave_max(unsigned long long v) {
  const uint32_t hi = wave_max((uint32_t)(v >> 32)), lo = wave_max((uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
  return (unsigned long long)hi << 32 | lo;
}
// largest over the workgroup, the same in every thread; `lds` is not in use by a wave that may be late
template <typename V> __device__ __forceinline__ V block_max(V v, V* lds) {
  v = wave_max(v);
  const int waves = (blockDim.x + 63) >> 6;
  if (waves == 1) return v;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  for (int k = 0; k < waves; ++k) v = lds[k] > v ? lds[k] : v;
  return v;
}

// A row's scale, and what a value is multiplied with; largest: of the row's magnitudes
struct RowScale {
  float s;
  double f;
  bool ok;
  __device__ __forceinline__ RowScale(double largest, double factor) {      // values are multiplied with `factor` first
    const double amax = largest * factor;
    s = (float)(fmax(amax, 0x1p-100) / 127.0);
    ok = amax < INFINITY && s < INFINITY;      // neither for NaN
    f = ok ? factor / (double)s * (1.0 + 0x1p-50) : 0.0;
    if (!ok) s = __builtin_nanf("");
  }
  __device__ __forceinline__ uint32_t round(double v) const {
    return ok ? (uint32_t)__builtin_bit_cast(unsigned long long, __builtin_fma(v, f, 0x1.8p52)) & 0xFFu : 0u;
  }
};
template <typename V> __device__ __forceinline__ u2 round8(const RowScale& s, const V (&v)[8]) {
  u2 q;
#pragma unroll
  for (int h = 0; h < 2; ++h) q[h] = s.round(v[4 * h]) | s.round(v[4 * h + 1]) << 8 | s.round(v[4 * h + 2]) << 16 | s.round(v[4 * h + 3]) << 24;
  return q;
}

// Rows as they are (G = false, x [rows][n] of T, `stride` elements apart), or silu(gate) up of float32 rows [gate | up] of n columns each (G = true).
// NV runs of eight columns to a thread; NV = 0: rows too long for that are read twice.  Rows from `from` on; last: rows from last[0] on are left, NULL: none.
template <int T, int NV, bool G>
__global__ __launch_bounds__(1024) void k_round_rows(const void* __restrict__ x, long long stride, long long from, int n, const int* __restrict__ last,
                                                     uint8_t* __restrict__ q, float* __restrict__ scales) {
  __shared__ uint32_t s_max[16];
  const long long row = from + blockIdx.x;
  if (last != nullptr && row >= last[0]) return;
  auto get = [&](int c, float (&f)[8]) {
    Eight<T> v;
    v.load_any(x, (size_t)(row * stride) + c);
    if constexpr (G) {
      Eight<T> u;
      u.load_any(x, (size_t)(row * stride) + n + c);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = silu(v.get(k)) * u.get(k);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = v.get(k);
    }
  };
  const int step = 8 * blockDim.x;
  float f[NV ? NV : 1][8];
  uint32_t m = 0;
  auto look = [&](const float (&f)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) m = max(m, magnitude(f[k]));
  };
  if constexpr (NV == 0) {
    for (int c = 8 * threadIdx.x; c < n; c += step) { get(c, f[0]); look(f[0]); }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) if (8 * (int)threadIdx.x + i * step < n) get(8 * threadIdx.x + i * step, f[i]);
#pragma unroll
    for (int i = 0; i < NV; ++i) if (8 * (int)threadIdx.x + i * step < n) look(f[i]);
  }
  const RowScale s((double)__uint_as_float(block_max(m, s_max)), 1.0);
  auto put = [&](int c, const float (&f)[8]) { *(HTR_GLOBAL u2*)((HTR_GLOBAL uint8_t*)q + (size_t)(row * n) + c) = round8(s, f); };
  if (threadIdx.x == 0) ((HTR_GLOBAL float*)scales)[row] = s.s;
  if constexpr (NV == 0) {
    for (int c = 8 * threadIdx.x; c < n; c += step) { get(c, f[0]); put(c, f[0]); }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) if (8 * (int)threadIdx.x + i * step < n) put(8 * threadIdx.x + i * step, f[i]);
  }
}

// A routed layer's beginning: pairs sorted by expert in the first `experts` workgroups, the tokens' rows rounded in the others, a wave to each.  Neither waits for the other:
// 4096 tokens of 2048, top 6 of 64: 12 us in one launch, 11 and 8 in two.
template <int T>
__global__ __launch_bounds__(ORDER_WAVES * 64) void k_order_and_round(const void* __restrict__ ids, int ids64, int pairs, int top, int experts, int* __restrict__ ends,
                                                                      int* __restrict__ token, int* __restrict__ pos_of, const void* __restrict__ x, int tokens, int n,
                                                                      uint8_t* __restrict__ q, float* __restrict__ scales) {
  if ((int)blockIdx.x < experts) {
    expert_order(ids, ids64, pairs, top, experts, ends, token, pos_of, blockIdx.x);
    return;
  }
  const int lane = threadIdx.x & 63;
  const size_t row = (size_t)(blockIdx.x - experts) * ORDER_WAVES + (threadIdx.x >> 6);
  if (row >= (size_t)tokens) return;
  constexpr int RUNS = 8;                     // of 512 columns, in registers; longer rows are read again
  Eight<T> v[RUNS];
  auto load = [&](int c) {
#pragma unroll
    for (int i = 0; i < RUNS; ++i) if (c + 512 * i < n) v[i].load_any(x, row * n + c + 512 * i);
  };
  uint32_t m = 0;
  for (int c = 8 * lane; c < n; c += 512 * RUNS) {
    load(c);
#pragma unroll
    for (int i = 0; i < RUNS; ++i)
      if (c + 512 * i < n) {
#pragma unroll
        for (int k = 0; k < 8; ++k) m = max(m, magnitude(v[i].get(k)));
      }
  }
  const RowScale s((double)__uint_as_float(wave_max(m)), 1.0);
  if (lane == 0) ((HTR_GLOBAL float*)scales)[row] = s.s;
  for (int c = 8 * lane; c < n; c += 512 * RUNS) {
    if (n > 512 * RUNS) load(c);
#pragma unroll
    for (int i = 0; i < RUNS; ++i)
      if (c + 512 * i < n) {
        float f[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = v[i].get(k);
        *(HTR_GLOBAL u2*)((HTR_GLOBAL uint8_t*)q + row * n + c + 512 * i) = round8(s, f);
      }
  }
}

// The norm of norm.hpp, rounded to int8.  NV as above.  The largest |t w| goes with the sum of squares; products of 16-bit values are exact in float32 where they do
// not leave it, others are formed in 64 bits.
template <int T, int NV, bool RES>
__global__ __launch_bounds__(1024) void k_rms_norm_int8(const NormArgs a) {
  __shared__ double s_sum[16];
  __shared__ uint32_t s_max[16];
  __shared__ unsigned long long s_wide[16];
  const long long row = blockIdx.x;
  const int n = a.n, step = 8 * blockDim.x;
  Eight<T> t[NV ? NV : 1], w[NV ? NV : 1];
  double sq = 0.0;
  uint32_t m = 0;
  auto first = [&](int c, Eight<T>& t, Eight<T>& w, bool loaded) {
    if (!loaded) {
      t.load_any(a.x, (size_t)(row * a.x_stride) + c);
      w.load_any(a.weight, c);
    }
    if constexpr (RES) {
      Eight<T> r;
      float f[8];
      r.load_any(a.residual, (size_t)(row * a.residual_stride) + c);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = t.get(k) + r.get(k);
      t.set(f);
      t.store_any(a.sum, (size_t)(row * n) + c);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const double v = t.get(k);
      sq += v * v;
      if constexpr (T != HTR_F32) m = max(m, magnitude(t.get(k) * w.get(k)));
    }
  };
  auto again = [&](int c, Eight<T>& t, Eight<T>& w) {
    if constexpr (RES) t.load_any(a.sum, (size_t)(row * n) + c); else t.load_any(a.x, (size_t)(row * a.x_stride) + c);
    w.load_any(a.weight, c);
  };
  auto each = [&](auto work) {      // what was read, or read again
    if constexpr (NV == 0) {
      for (int c = 8 * threadIdx.x; c < n; c += step) { again(c, t[0], w[0]); work(c, t[0], w[0]); }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) { const int c = 8 * threadIdx.x + i * step; if (c < n) work(c, t[i], w[i]); }
    }
  };
  if constexpr (NV == 0) {
    for (int c = 8 * threadIdx.x; c < n; c += step) first(c, t[0], w[0], false);
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * threadIdx.x + i * step;
      if (c < n) { t[i].load_any(a.x, (size_t)(row * a.x_stride) + c); w[i].load_any(a.weight, c); }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) { const int c = 8 * threadIdx.x + i * step; if (c < n) first(c, t[i], w[i], true); }
  }
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = m;
  const double r = 1.0 / sqrt(block_sum(sq, s_sum) / n + a.eps);
  for (int k = 0; k < (int)((blockDim.x + 63) >> 6); ++k) m = max(m, s_max[k]);
  auto put = [&](int c, u2 q) { *(HTR_GLOBAL u2_any*)((HTR_GLOBAL uint8_t*)a.y + (size_t)(row * n) + c) = q; };
  float scale;
  if (T != HTR_F32 && m >= 0x17800000u && m < 0x7F800000u) {      // 2^-80: what is lost of products below 2^-126 is no half of a step
    const RowScale s((double)__uint_as_float(m), r);
    scale = s.s;
    each([&](int c, const Eight<T>& t, const Eight<T>& w) {
      float p[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) p[k] = t.get(k) * w.get(k);
      put(c, round8(s, p));
    });
  } else {
    unsigned long long wide = 0;
    each([&](int, const Eight<T>& t, const Eight<T>& w) {
#pragma unroll
      for (int k = 0; k < 8; ++k) { const unsigned long long v = magnitude((double)t.get(k) * (double)w.get(k)); wide = v > wide ? v : wide; }
    });
    const RowScale s(__builtin_bit_cast(double, block_max(wide, s_wide)), r);
    scale = s.s;
    each([&](int c, const Eight<T>& t, const Eight<T>& w) {
      double p[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) p[k] = (double)t.get(k) * (double)w.get(k);
      put(c, round8(s, p));
    });
  }
  if (threadIdx.x == 0) ((HTR_GLOBAL float*)a.scales)[row] = scale;
}
