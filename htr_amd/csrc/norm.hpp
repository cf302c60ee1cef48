// Part of unpacked.hip, included inside its anonymous namespace: root-mean-square norm with the residual's addition, and rows in e4m3 with a
// scale for each 128 columns.
//
//   t = round(x + r),   y_c = t_c w_c / sqrt(mean_c t_c^2 + eps)
//   e4m3: s_b = the least power of two from max_b |y| / 448 up,   q_c = e4m3(y_c / s_b)      for each block b of 128 columns
//
// Scales are powers of two: the division is then exact, and the values of a 16-bit row reach e4m3 in one rounding.  With amax / 448 as the scale,
// x / s falls on ties of e4m3 for one block in seven (448 = 7 2^6), where the rounding of s itself decides: results then differ by
// several thousandths between machines, and by 2 % behind a second quantization.  A power of two costs no precision but at the lower
// end, where values below 2^-15 of the block's largest lose a bit more.
// Bound: HBM (x, r and w read once, t and y or q and s written once).  A workgroup takes one row and keeps it in registers between the two passes.
// 8192 rows of 4096 in bf16 to e4m3: 25 us (4.0 TB/s), with a residual 40 us (5.9 TB/s; a copy of large arrays reaches 5.1, a read alone 7.3); one row 3.3 us.

// ---- e4m3
// the scale of a block whose largest finite magnitude is `amax`: amax = f 2^e with f in [1/2, 1), 448 = 0.875 2^9.  A block of zeros (or of
// values below 2^-100) counts as 2^-100, so that neither the scale nor its inverse leaves float32.
__device__ __forceinline__ int e4m3_exponent(double amax) {
  amax = fmax(amax, 0x1p-100);
  const unsigned long long u = __builtin_bit_cast(unsigned long long, amax);
  const int e = (int)(u >> 52) - 1022;                                // frexp's exponent
  return e - 9 + ((u & 0xFFFFFFFFFFFFFull) > 0xC000000000000ull);     // mantissa beyond 1.75
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }      // -126 <= e <= 127
// what e4m3 has no value for becomes NaN there, and takes no part in the scale
__device__ __forceinline__ float finite_or_nan(float v) { return fabsf(v) < INFINITY ? v : __builtin_nanf(""); }
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}
// largest of 16 neighbouring lanes, in all of them
__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, dpp_mov<0xB1>(v)); v = fmaxf(v, dpp_mov<0x4E>(v));
  v = fmaxf(v, dpp_mov<0x141>(v)); return fmaxf(v, dpp_mov<0x140>(v));
}
__device__ __forceinline__ double max16(double v) {
#pragma unroll
  for (int off = 1; off < 16; off <<= 1) v = fmax(v, __shfl_xor(v, off));
  return v;
}

// ---- two floats to 16 bits each, rounded to nearest
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) { return __builtin_bit_cast(uint32_t, b2{(__bf16)a, (__bf16)b}); }
__device__ __forceinline__ uint32_t pack_f16(float a, float b) { return __builtin_bit_cast(uint32_t, h2{(_Float16)a, (_Float16)b}); }

// ---- eight consecutive elements, on a 16-byte boundary or (ANY) wherever an element may be: the memory unit takes 16 bytes from any address
typedef uint32_t u4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef float f4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u2_any __attribute__((ext_vector_type(2), aligned(1)));
template <int T> struct Eight;      // T: HTR_BF16, HTR_F16 or HTR_F32
template <> struct Eight<HTR_BF16> {
  u4 v;
  __device__ __forceinline__ void load(const void* p, size_t i) { v = *(const HTR_GLOBAL u4*)((const HTR_GLOBAL uint16_t*)p + i); }
  __device__ __forceinline__ void store(void* p, size_t i) const { *(HTR_GLOBAL u4*)((HTR_GLOBAL uint16_t*)p + i) = v; }
  __device__ __forceinline__ void load_any(const void* p, size_t i) { v = *(const HTR_GLOBAL u4_any*)((const HTR_GLOBAL uint16_t*)p + i); }
  __device__ __forceinline__ void store_any(void* p, size_t i) const { *(HTR_GLOBAL u4_any*)((HTR_GLOBAL uint16_t*)p + i) = v; }
  // the first `count`, zeros behind
  __device__ __forceinline__ void load_first(const void* p, size_t i, int count) {
    v = u4{0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < 7; ++k) if (k < count) v[k >> 1] |= (uint32_t)((const HTR_GLOBAL uint16_t*)p)[i + k] << 16 * (k & 1);
  }
  __device__ __forceinline__ void store_first(void* p, size_t i, int count) const {
#pragma unroll
    for (int k = 0; k < 7; ++k) if (k < count) ((HTR_GLOBAL uint16_t*)p)[i + k] = (uint16_t)(v[k >> 1] >> 16 * (k & 1));
  }
  __device__ __forceinline__ float get(int k) const { return __uint_as_float(k & 1 ? v[k >> 1] & 0xFFFF0000u : v[k >> 1] << 16); }
  __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = pack_bf16(f[2 * k], f[2 * k + 1]);
  }
};
template <> struct Eight<HTR_F16> {
  u4 v;
  __device__ __forceinline__ void load(const void* p, size_t i) { v = *(const HTR_GLOBAL u4*)((const HTR_GLOBAL uint16_t*)p + i); }
  __device__ __forceinline__ void store(void* p, size_t i) const { *(HTR_GLOBAL u4*)((HTR_GLOBAL uint16_t*)p + i) = v; }
  __device__ __forceinline__ void load_any(const void* p, size_t i) { v = *(const HTR_GLOBAL u4_any*)((const HTR_GLOBAL uint16_t*)p + i); }
  __device__ __forceinline__ void store_any(void* p, size_t i) const { *(HTR_GLOBAL u4_any*)((HTR_GLOBAL uint16_t*)p + i) = v; }
  // the first `count`, zeros behind
  __device__ __forceinline__ void load_first(const void* p, size_t i, int count) {
    v = u4{0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < 7; ++k) if (k < count) v[k >> 1] |= (uint32_t)((const HTR_GLOBAL uint16_t*)p)[i + k] << 16 * (k & 1);
  }
  __device__ __forceinline__ void store_first(void* p, size_t i, int count) const {
#pragma unroll
    for (int k = 0; k < 7; ++k) if (k < count) ((HTR_GLOBAL uint16_t*)p)[i + k] = (uint16_t)(v[k >> 1] >> 16 * (k & 1));
  }
  __device__ __forceinline__ float get(int k) const { return f16_bits_to_float((uint16_t)(k & 1 ? v[k >> 1] >> 16 : v[k >> 1])); }
  __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = pack_f16(f[2 * k], f[2 * k + 1]);
  }
};
template <> struct Eight<HTR_F32> {
  f4 v[2];
  __device__ __forceinline__ void load(const void* p, size_t i) {
    v[0] = *(const HTR_GLOBAL f4*)((const HTR_GLOBAL float*)p + i); v[1] = *(const HTR_GLOBAL f4*)((const HTR_GLOBAL float*)p + i + 4);
  }
  __device__ __forceinline__ void store(void* p, size_t i) const {
    *(HTR_GLOBAL f4*)((HTR_GLOBAL float*)p + i) = v[0]; *(HTR_GLOBAL f4*)((HTR_GLOBAL float*)p + i + 4) = v[1];
  }
  __device__ __forceinline__ void load_any(const void* p, size_t i) {
    v[0] = *(const HTR_GLOBAL f4_any*)((const HTR_GLOBAL float*)p + i); v[1] = *(const HTR_GLOBAL f4_any*)((const HTR_GLOBAL float*)p + i + 4);
  }
  __device__ __forceinline__ void store_any(void* p, size_t i) const {
    *(HTR_GLOBAL f4_any*)((HTR_GLOBAL float*)p + i) = v[0]; *(HTR_GLOBAL f4_any*)((HTR_GLOBAL float*)p + i + 4) = v[1];
  }
  __device__ __forceinline__ void load_first(const void* p, size_t i, int count) {
    v[0] = v[1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 7; ++k) if (k < count) v[k >> 2][k & 3] = ((const HTR_GLOBAL float*)p)[i + k];
  }
  __device__ __forceinline__ void store_first(void* p, size_t i, int count) const {
#pragma unroll
    for (int k = 0; k < 7; ++k) if (k < count) ((HTR_GLOBAL float*)p)[i + k] = v[k >> 2][k & 3];
  }
  __device__ __forceinline__ float get(int k) const { return v[k >> 2][k & 3]; }
  __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k >> 2][k & 3] = f[k];
  }
};

// Eight products (t w) r of a row, 16 neighbouring lanes holding a block of 128: their e4m3 values and the block's scale, in float32 to one rounding.
// t w = p + l without an error (l = 0 for 16-bit types, whose products have 22 bits at most); the factor r of the row, 64 bits, over the scale is u + v;
// then p u + (p v + l u).  The scale is the right one also where the block's largest value lies next to 448 times a power of two: there, and where
// parts that count may fall off either end of float32, the block is formed in 64 bits.
template <int T>
__device__ __forceinline__ u2 quantize8(const Eight<T>& t, const Eight<T>& w, double r, float& scale) {
  float p[8], l[8], m = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    p[k] = t.get(k) * w.get(k);
    if constexpr (T == HTR_F32) l[k] = __builtin_fmaf(t.get(k), w.get(k), -p[k]);
    m = fmaxf(m, fabsf(p[k]));
  }
  m = max16(m);                                     // the same in all 16 lanes, and what follows from it
  int e = e4m3_exponent((double)m * r);
  bool exact = m >= 0x1p-80f && m < INFINITY && e > -100 && e < 100;
  if constexpr (T == HTR_F32) exact = exact && e == e4m3_exponent((double)m * r * (1.0 + 0x1p-22)) && e == e4m3_exponent((double)m * r * (1.0 - 0x1p-22));
  float y[8];
  if (exact) {
    const double f = r * __builtin_bit_cast(double, (unsigned long long)(1023 - e) << 52);
    const float u = (float)f, v = (float)(f - u);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if constexpr (T == HTR_F32) y[k] = __builtin_fmaf(p[k], u, __builtin_fmaf(l[k], u, p[k] * v));
      else y[k] = __builtin_fmaf(p[k], u, p[k] * v);
    }
  } else {
    double d[8], amax = 0.0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      d[k] = (double)finite_or_nan(t.get(k)) * (double)w.get(k) * r;
      if (fabs(d[k]) > (double)__FLT_MAX__) d[k] = __builtin_nan("");
      amax = fmax(amax, fabs(d[k]));
    }
    e = min(e4m3_exponent(max16(amax)), 120);       // beyond: larger than float32 can hold
    const double inv = __builtin_bit_cast(double, (unsigned long long)(1023 - e) << 52);
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = (float)(d[k] * inv);
  }
  scale = exp2i(e);
  return u2{pack_e4m3(y[0], y[1], y[2], y[3]), pack_e4m3(y[4], y[5], y[6], y[7])};
}
// The same for eight values in float32 as they are
__device__ __forceinline__ u2 quantize8(const float (&v)[8], float& scale) {
  float f[8], m = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) { f[k] = finite_or_nan(v[k]); m = fmaxf(m, fabsf(f[k])); }
  const int e = e4m3_exponent((double)max16(m));
  const float inv = exp2i(-e);
  scale = exp2i(e);
  u2 q;
#pragma unroll
  for (int h = 0; h < 2; ++h) q[h] = pack_e4m3(f[4 * h] * inv, f[4 * h + 1] * inv, f[4 * h + 2] * inv, f[4 * h + 3] * inv);
  return q;
}

struct NormArgs {
  const void *x, *residual, *weight;
  void *y, *sum;                    // y: of x's type, or e4m3; sum: t, where there is a residual
  float* scales;                    // e4m3: [rows][n / 128]
  long long x_stride, residual_stride;      // elements between rows
  long long rows;
  int n;
  double eps;
};

// sum of a wave, the same in every lane: within 16 lanes by DPP, across them by swaps of rows of lanes (a shuffle through LDS takes several times as long)
template <int CTRL> __device__ __forceinline__ double dpp_mov64(double v) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const uint32_t lo = __float_as_uint(dpp_mov<CTRL>(__uint_as_float((uint32_t)u))), hi = __float_as_uint(dpp_mov<CTRL>(__uint_as_float((uint32_t)(u >> 32))));
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum(double v) {
  v += dpp_mov64<0xB1>(v); v += dpp_mov64<0x4E>(v); v += dpp_mov64<0x141>(v); v += dpp_mov64<0x140>(v);
  auto both = [](double v, auto swap) {
    const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
    const u2s lo = swap((uint32_t)u), hi = swap((uint32_t)(u >> 32));
    return __builtin_bit_cast(double, (unsigned long long)hi.x << 32 | lo.x) + __builtin_bit_cast(double, (unsigned long long)hi.y << 32 | lo.y);
  };
  v = both(v, [](uint32_t x) { return __builtin_amdgcn_permlane16_swap(x, x, false, false); });
  return both(v, [](uint32_t x) { return __builtin_amdgcn_permlane32_swap(x, x, false, false); });
}
// sum over the workgroup, the same in every thread
__device__ __forceinline__ double block_sum(double v, double* lds) {
  v = wave_sum(v);
  const int waves = (blockDim.x + 63) >> 6;
  if (waves == 1) return v;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
  for (int k = 0; k < waves; ++k) s += lds[k];
  return s;
}

// NV runs of eight columns to a thread; n <= 8 NV threads.  Every row on a 16-byte boundary and n a multiple of 8, or (ANY) neither: the last run of a
// row may then be a part of one.  Runs from any address cost little next to loads of single elements: 8000 rows of 1001 bf16 columns with their
// residual 19 us (element by element 54; 13 at the rate of a copy).
// The squares are summed in 64 bits: a row's mean of many of them keeps what float32 holds, for two instructions to an element
// that the memory hides.
template <int T, int NV, bool RES, bool QUANT, bool ANY>
__global__ __launch_bounds__(1024) void k_rms_norm(const NormArgs a) {
  __shared__ double s_sum[16];
  const long long row = blockIdx.x;
  const int n = a.n;
  auto load = [&](Eight<T>& e, const void* p, size_t row_at, int c) {
    if constexpr (!ANY) e.load(p, row_at + c);
    else if (c + 8 <= n) e.load_any(p, row_at + c);
    else e.load_first(p, row_at + c, n - c);
  };
  auto store = [&](const Eight<T>& e, void* p, int c) {
    const size_t i = (size_t)(row * n) + c;
    if constexpr (!ANY) e.store(p, i);
    else if (c + 8 <= n) e.store_any(p, i);
    else e.store_first(p, i, n - c);
  };
  Eight<T> t[NV], w[NV];
  double sq = 0.0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = 8 * (threadIdx.x + i * blockDim.x);
    if (c < n) {
      load(t[i], a.x, (size_t)(row * a.x_stride), c);
      load(w[i], a.weight, 0, c);
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = 8 * (threadIdx.x + i * blockDim.x);
    if (c >= n) continue;
    if constexpr (RES) {
      Eight<T> r;
      float f[8];
      load(r, a.residual, (size_t)(row * a.residual_stride), c);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = t[i].get(k) + r.get(k);
      t[i].set(f);
      store(t[i], a.sum, c);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) { const double v = t[i].get(k); sq += v * v; }
  }
  const double mean = block_sum(sq, s_sum) / n + a.eps;
  const double r = 1.0 / sqrt(mean);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = 8 * (threadIdx.x + i * blockDim.x);
    if constexpr (QUANT) {
      // n is a multiple of 128 and blockDim.x of 64: 16 neighbouring lanes are inside or outside together
      if (c >= n) continue;
      float scale;
      const u2 q = quantize8<T>(t[i], w[i], r, scale);
      *(HTR_GLOBAL u2_any*)((HTR_GLOBAL uint8_t*)a.y + (size_t)(row * n) + c) = q;
      if ((threadIdx.x & 15) == 0) ((HTR_GLOBAL float*)a.scales)[(size_t)row * (n >> 7) + (c >> 7)] = scale;
    } else {
      if (c >= n) continue;
      float f[8];
      if (r > 0x1p-100 && r < 0x1p100) {
        const float rf = (float)r;
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = t[i].get(k) * rf * w[i].get(k);
      } else {      // the factor may have no float32, t r has
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = (float)(t[i].get(k) * r) * w[i].get(k);
      }
      Eight<T> y;
      y.set(f);
      store(y, a.y, c);
    }
  }
}

// Rows of more than 32768 columns: read twice, the second time from the cache; with a residual the sums as they were written.  2000 rows of 40960 in bf16 to e4m3
// with a residual 125 us, 4.6 TB/s of bytes read or written once (loads of single elements 530); without one 75 us, 3.3 TB/s, the second reading apart.
template <int T, bool RES, bool QUANT>
__global__ __launch_bounds__(1024) void k_rms_norm_long(const NormArgs a) {
  __shared__ double s_sum[16];
  const long long row = blockIdx.x;
  const int n = a.n;
  auto load = [&](Eight<T>& e, const void* p, size_t row_at, int c) {
    if (c + 8 <= n) e.load_any(p, row_at + c); else e.load_first(p, row_at + c, n - c);
  };
  auto store = [&](const Eight<T>& e, void* p, int c) {
    const size_t i = (size_t)(row * n) + c;
    if (c + 8 <= n) e.store_any(p, i); else e.store_first(p, i, n - c);
  };
  double sq = 0.0;
  for (int c = 8 * threadIdx.x; c < n; c += 8 * 1024) {
    Eight<T> t;
    load(t, a.x, (size_t)(row * a.x_stride), c);
    if constexpr (RES) {
      Eight<T> r;
      float f[8];
      load(r, a.residual, (size_t)(row * a.residual_stride), c);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = t.get(k) + r.get(k);
      t.set(f);
      store(t, a.sum, c);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) { const double v = t.get(k); sq += v * v; }
  }
  const double r = 1.0 / sqrt(block_sum(sq, s_sum) / n + a.eps);
  for (int c = 8 * threadIdx.x; c < n; c += 8 * 1024) {
    Eight<T> t, w;
    if constexpr (RES) load(t, a.sum, (size_t)(row * n), c); else load(t, a.x, (size_t)(row * a.x_stride), c);
    load(w, a.weight, 0, c);
    if constexpr (QUANT) {
      float scale;
      *(HTR_GLOBAL u2_any*)((HTR_GLOBAL uint8_t*)a.y + (size_t)(row * n) + c) = quantize8<T>(t, w, r, scale);
      if ((threadIdx.x & 15) == 0) ((HTR_GLOBAL float*)a.scales)[(size_t)row * (n >> 7) + (c >> 7)] = scale;
    } else {
      float f[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = (float)(t.get(k) * r) * w.get(k);
      Eight<T> y;
      y.set(f);
      store(y, a.y, c);
    }
  }
}

// Rows to e4m3 as they are: 16 lanes to a block of 128 columns
template <int T>
__global__ __launch_bounds__(256) void k_quantize(const void* __restrict__ x, long long stride, long long blocks, int per_row, uint8_t* __restrict__ q,
                                                  float* __restrict__ scales) {
  const long long b = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
  if (b >= blocks) return;
  const long long row = b / per_row;
  const int c = (int)(b - row * per_row) * 128 + 8 * (threadIdx.x & 15);
  Eight<T> v;
  v.load(x, (size_t)(row * stride) + c);
  float f[8], scale;
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = v.get(k);
  *(HTR_GLOBAL u2*)((HTR_GLOBAL uint8_t*)q + (size_t)row * per_row * 128 + c) = quantize8(f, scale);
  if ((threadIdx.x & 15) == 0) ((HTR_GLOBAL float*)scales)[b] = scale;
}
