// Part of unpacked.hip, included inside its anonymous namespace: products of rows with matrices that are not HTR-W1, one matrix or one for each expert.
//
//   y[r][i] = sum_k x[r][k] w_e[i][k],  e the expert of row r;  e4m3: the sum over each block of 128 columns times xs[r][k / 128] ws_e[i / 128][k / 128];
//   int8: the sum, exact in 32 bits, times xs[r] ws_e[i]
//
// Everything is cut into slabs of 128 bytes of a row: 128 e4m3 values, one v_mfma_f32_16x16x128_f8f6f4 whose result is scaled into the sum, 128
// integers, two v_mfma_i32_16x16x64_i8, or 64 16-bit values, two v_mfma_f32_16x16x32.  A lane feeds bytes 16 g .. and 64 + 16 g .. of its row (g = lane / 16): another order of the
// columns than the instructions' own, the same for both operands.  Matrix rows are MFMA rows (D: rows 4 g + i, four to a lane), activation
// rows are MFMA columns (lane % 16), so that a lane holds consecutive outputs of one row.
enum { P_F8 = 3, P_I8 = 4 };             // beside HTR_BF16, HTR_F16: the operands' type
template <int T> constexpr int bytes_of = T == P_F8 || T == P_I8 ? 1 : 2;
typedef int i4 __attribute__((ext_vector_type(4)));
template <int T> struct SumOf { typedef f4 type; typedef float one; };      // what products are summed in
template <> struct SumOf<P_I8> { typedef i4 type; typedef int one; };
typedef int i8v __attribute__((ext_vector_type(8)));

struct ProductArgs {
  const void* x;                         // [.][n]; also rows that the product rounds itself: 16 bits with e4m3 matrices (takes_16bit_rows), floating ones with an int8 one (rounds_rows)
  const float* xs;                       // e4m3 rows: [.][n / 128]; int8: [.]
  const void* w;                         // [experts][m][n]
  const float* ws;                       // e4m3: [experts][ceil(m / 128)][n / 128]; int8: [experts][m]
  const void* bias;                      // [m] in y's type or NULL
  void* y;                               // [rows][m]
  const int* ends;                       // [experts]: expert e has rows ends[e - 1] .. ends[e] - 1; NULL: one expert, all rows
  const int* gather;                     // row r of the product is row gather[r] of x; NULL: r
  int rows, m, n, experts, y_dtype, x_type;
  float* ys;                             // k_product_tile<GATED> with y in e4m3: its scales, [rows][m / 256]
  bool wide;                             // e4m3, few 16-bit rows: float32 sums, for a result that is rounded to e4m3 next
};

// Rows first .. first + count - 1 of expert e are tile number t of tiles of `height` rows, expert by expert; e = experts: rows behind the last
// expert's; e = -1: no such tile.  Ends are taken as what they may be: at least the one before, at least 0, at most `rows`.
struct Span { int e, first, count; };
// running maximum and sum of a wave's values, none below 0, by DPP: four steps within 16 lanes, then the last lane of 16 and of 32 to those behind
template <int CTRL, int ROWS = 0xF> __device__ __forceinline__ int dpp_or(int old, int v) { return __builtin_amdgcn_update_dpp(old, v, CTRL, ROWS, 0xF, false); }
__device__ __forceinline__ int scan_max(int v) {
  v = max(v, dpp_or<0x111>(0, v)); v = max(v, dpp_or<0x112>(0, v)); v = max(v, dpp_or<0x114>(0, v)); v = max(v, dpp_or<0x118>(0, v));
  v = max(v, dpp_or<0x142, 0xA>(0, v)); return max(v, dpp_or<0x143, 0xC>(0, v));
}
__device__ __forceinline__ int scan_sum(int v) {
  v += dpp_or<0x111>(0, v); v += dpp_or<0x112>(0, v); v += dpp_or<0x114>(0, v); v += dpp_or<0x118>(0, v);
  v += dpp_or<0x142, 0xA>(0, v); return v + dpp_or<0x143, 0xC>(0, v);
}
// 64 experts from `base` on, one to a lane: where its rows begin and end, its tiles, and those up to its last; end0, tiles0: of the experts before
struct Experts { int start, end, tiles, sum; };
__device__ __forceinline__ Experts experts_from(const ProductArgs& a, int height, int base, int end0, int tiles0) {
  const int e = base + (int)(threadIdx.x & 63);
  Experts x;
  x.end = max(scan_max(e < a.experts ? max(0, min(a.ends[e], a.rows)) : 0), end0);
  x.start = dpp_or<0x138>(end0, x.end);      // the lane before
  x.tiles = (x.end - x.start + height - 1) / height;
  x.sum = scan_sum(x.tiles) + tiles0;
  return x;
}
__device__ __forceinline__ Span find_span(const ProductArgs& a, int height, int t) {
  if (a.ends == nullptr) {
    const int first = t * height;
    return first < a.rows ? Span{0, first, min(height, a.rows - first)} : Span{-1, 0, 0};
  }
  int end0 = 0, tiles0 = 0;
  for (int base = 0; base < a.experts; base += 64) {
    const Experts x = experts_from(a, height, base, end0, tiles0);
    const unsigned long long in = __ballot(x.sum > t);
    if (in) {
      const int l = __builtin_ctzll(in);
      const int skip = (t - (__builtin_amdgcn_readlane(x.sum, l) - __builtin_amdgcn_readlane(x.tiles, l))) * height;
      const int first = __builtin_amdgcn_readlane(x.start, l) + skip;
      return Span{base + l, first, min(height, __builtin_amdgcn_readlane(x.end, l) - first)};
    }
    end0 = __builtin_amdgcn_readlane(x.end, 63);
    tiles0 = __builtin_amdgcn_readlane(x.sum, 63);
  }
  // t - tiles0 tiles behind the last expert's; the grid is a bound, so this may lie beyond 32 bits of rows
  const long long first = end0 + (long long)(t - tiles0) * height;
  return first < a.rows ? Span{a.experts, (int)first, min(height, a.rows - (int)first)} : Span{-1, 0, 0};
}
// tiles that find_span knows, those of rows behind the last expert's among them
__device__ __forceinline__ int count_spans(const ProductArgs& a, int height) {
  int end0 = 0, tiles0 = 0;
  for (int base = 0; a.ends != nullptr && base < a.experts; base += 64) {
    const Experts x = experts_from(a, height, base, end0, tiles0);
    end0 = __builtin_amdgcn_readlane(x.end, 63);
    tiles0 = __builtin_amdgcn_readlane(x.sum, 63);
  }
  return tiles0 + (a.rows - end0 + height - 1) / height;
}
// tiles that find_span knows at most: experts with rows leave one short tile each, and so do the rows behind them
inline long long span_bound(long long rows, int experts, bool grouped, int height) {
  const long long full = (rows + height - 1) / height;
  return !grouped ? full : rows / height + (rows < experts + 1 ? rows : experts + 1);
}

// rows behind the last expert's: zeros
__device__ __forceinline__ void zero_rows(const ProductArgs& a, const Span& s, int m0, int width) {
  const int w = min(width, a.m - m0);
  for (int i = threadIdx.x; i < s.count * w; i += blockDim.x)
    store_elem_g(a.y, a.y_dtype, (size_t)(s.first + i / w) * a.m + m0 + i % w, 0.f);
}

// Sums: an e4m3 instruction adds the products of eight consecutive columns first, to 2^-13 of the largest by its operands' exponents (none counts as less than that
// of 2^-6), and only these sums in float32 (measured, with one eight and with all; the older instruction for 32 columns does the same).  Eight products are off by
// 2^-10 of that largest at most, and a result in float32 by 1.5e-5 in the 2-norm (normal values), where a product in float32 is off by 1e-7: a hundredth of what
// rounding it to bfloat16 takes (1.7e-3), less than a thousandth of what the operands' own rounding to e4m3 does.  A choice for the rate: what holds float32
// throughout takes 16-bit operands at half of it (8192 rows on 14336x4096 462 us in e4m3, 744 in 16 bits).  Few rows, which wait for memory, take the same
// instruction, so that a block's products come to the same sum in every kernel.
// Where a result is rounded to e4m3 next, 1.5e-5 is enough to put one value in some thousand on the other side of a tie, a step of 6 to 12 % of it.  Gate and up of
// an expert layer therefore take float32 sums (WIDE) where the matrix unit has the time, with few rows and in tiles of up to 64: 16-bit instructions on the
// same values in f16, which holds every e4m3 value, two of them by one conversion.  A layer's result in float16 is off by 2e-4 then, where it was by 1.3e-3 (some tokens
// 5e-3); 16 tokens of 64 experts of 2048/1408 103 us and 102, 256 of 8 of 4096/2048 83 and 79.  Larger tiles are bound by the unit's power, which 16-bit
// instructions take twice of (4096 tokens 482 us and 393, 425 and 319), and stay with the e4m3 one.
__device__ __forceinline__ f4 mfma_f8(const u4& a0, const u4& a1, const u4& b0, const u4& b1) {
  const i8v a = {(int)a0.x, (int)a0.y, (int)a0.z, (int)a0.w, (int)a1.x, (int)a1.y, (int)a1.z, (int)a1.w};
  const i8v b = {(int)b0.x, (int)b0.y, (int)b0.z, (int)b0.w, (int)b1.x, (int)b1.y, (int)b1.z, (int)b1.w};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}
// 32 e4m3 values of a lane in f16, in their order
struct Wide { h8 v[4]; };
__device__ __forceinline__ h8 widen(uint32_t lo, uint32_t hi) {
  const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
  const h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
  return h8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
__device__ __forceinline__ Wide widen(const u4 (&q)[2]) { return Wide{{widen(q[0].x, q[0].y), widen(q[0].z, q[0].w), widen(q[1].x, q[1].y), widen(q[1].z, q[1].w)}}; }
template <int T> __device__ __forceinline__ typename SumOf<T>::type mfma_16(const u4& a, const u4& b, const typename SumOf<T>::type& c) {
  if constexpr (T == P_I8) return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i4, a), __builtin_bit_cast(i4, b), c, 0, 0, 0);
  else if constexpr (T == HTR_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

__device__ __forceinline__ float silu(float g) { return g / (1.f + __expf(-g)); }

// ------------------------------------------------------------------------------------------------ few rows
// A workgroup owns 16 R rows of a matrix and up to 16 TT rows of x; its waves take the slabs in turn, straight from memory into registers
// (every byte of the matrix is used by one wave once: LDS would only be a detour), and add up through LDS.
// Bound: HBM, the matrix read once: 96 rows of 64 experts of 2816x2048 in e4m3 52 us, 5.4 TB/s (a kernel that only reads reaches 7.3); one row on 1024x4096 5.0 us, the
// latency of two loads and the sum.
// X: the type of x; 16-bit rows with an e4m3 matrix are rounded on the way, by every workgroup for itself: about 110 instructions to a slab, beside
// its 2 KB or more of the matrix, against a launch ahead of this one.  WIDE: e4m3 products in float32 sums.
// TAIL: rows end inside their last slab, at a multiple of 16 bytes.  Others have no test of where a row ends (us in bf16, with it and without: 12 rows of 3 experts of 4096x1408
// 11.9 and 9.4, of 1024x4096 9.5 and 8.8, 4 rows on 4096x4096 10.1 and 9.2; 12 of 3 of 4096x8192 46.7 and 47.3, of 54 sizes the only one that was slower).  With a tail, whole
// slabs in a form of their own cost 16 rows in 16 bits more than the test does (1 row on 4096x7600, both forms and one: 17.4 and 16.8; 8 of 8 experts of 1024x4104 17.7 and
// 17.4, 12 of 3 of 4096x4104 27.3 and 27.9), and 32, or int8, less (128 of 4 of 512x4104 15.6 and 17.4; in int8 48 rows on 2048x4112 8.4 and 9.4, 48 of 8 of 1024x24592
// 58.7 and 60.5).
template <int T, int X, int R, int TT, int STREAM_WAVES, bool WIDE, bool TAIL>
__global__ __launch_bounds__(STREAM_WAVES * 64) void k_product_stream(const ProductArgs a) {
  constexpr int P = R + TT <= 3 && !(X != T && STREAM_WAVES > 8) ? 4 : 2;      // slabs in flight
  constexpr bool ROUNDS = X != T;
  static_assert(((!ROUNDS && !WIDE) || T == P_F8) && !(TAIL && T == P_F8), "");
  typedef typename SumOf<T>::type Sum;
  typedef typename SumOf<T>::one One;
  __shared__ One red[STREAM_WAVES][R * TT * 256];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
  const int m0 = blockIdx.x * 16 * R;
  const Span s = find_span(a, 16 * TT, blockIdx.y);
  if (s.e < 0) return;
  if (s.e == a.experts) { zero_rows(a, s, m0, 16 * R); return; }
  const size_t row_bytes = (size_t)a.n * bytes_of<T>;
  const int slabs = (int)((row_bytes + 127) >> 7);
  const HTR_GLOBAL uint8_t *wp[R], *xp[TT];
  const HTR_GLOBAL float* sp[TT];
#pragma unroll
  for (int i = 0; i < R; ++i)      // rows beyond the matrix: its last one, whose results are not stored
    wp[i] = (const HTR_GLOBAL uint8_t*)a.w + ((size_t)s.e * a.m + min(m0 + 16 * i + c, a.m - 1)) * row_bytes + 16 * g;
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    int r = s.first + min(16 * t + c, s.count - 1);
    if (a.gather != nullptr) r = a.gather[r];
    xp[t] = (const HTR_GLOBAL uint8_t*)a.x + (size_t)r * (ROUNDS ? 2 * row_bytes : row_bytes) + (ROUNDS ? 32 : 16) * g;
    sp[t] = (const HTR_GLOBAL float*)a.xs + (size_t)r * (a.n >> 7);
  }
  const HTR_GLOBAL float* wsp = (const HTR_GLOBAL float*)a.ws + ((size_t)s.e * ((a.m + 127) >> 7) + (m0 >> 7)) * (a.n >> 7);
  // int8: the scales of what this thread stores, asked for ahead of everything else
  constexpr int STORES = (R * TT * 256 + STREAM_WAVES * 64 - 1) / (STREAM_WAVES * 64);
  float row_scale[T == P_I8 ? STORES : 1], matrix_scale[T == P_I8 ? STORES : 1];
  if constexpr (T == P_I8) {
#pragma unroll
    for (int k = 0; k < STORES; ++k) {
      const int idx = min((int)threadIdx.x + k * STREAM_WAVES * 64, R * TT * 256 - 1);
      int r = s.first + min(idx / (16 * R), s.count - 1);
      if (a.gather != nullptr) r = a.gather[r];
      row_scale[k] = ((const HTR_GLOBAL float*)a.xs)[r];
      matrix_scale[k] = ((const HTR_GLOBAL float*)a.ws)[(size_t)s.e * a.m + min(m0 + idx % (16 * R), a.m - 1)];
    }
  }
  Sum acc[R][TT];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[i][t] = Sum{0, 0, 0, 0};
  u4 A[P][R][2], B[P][TT][2];
  Eight<X == P_F8 || X == P_I8 ? HTR_BF16 : X> raw[ROUNDS ? P : 1][TT][4];  // 16 elements of either half of the slab
  float sx[P][TT], sw[P];
  const u4 zero = {0u, 0u, 0u, 0u};
  auto load_slab = [&](int p, int slab, auto whole) {
    const size_t off = (size_t)slab << 7;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool in = decltype(whole)::value || off + 64 * h + 16 * g < row_bytes;
#pragma unroll
      for (int i = 0; i < R; ++i) { A[p][i][h] = zero; if (in) A[p][i][h] = __builtin_nontemporal_load((const HTR_GLOBAL u4*)(wp[i] + off + 64 * h)); }
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        if constexpr (ROUNDS) {
#pragma unroll
          for (int k = 0; k < 2; ++k) raw[p][t][2 * h + k].v = *(const HTR_GLOBAL u4*)(xp[t] + 2 * off + 128 * h + 16 * k);
        } else {
          B[p][t][h] = zero;
          if (in) B[p][t][h] = *(const HTR_GLOBAL u4*)(xp[t] + off + 64 * h);
        }
      }
    }
    if constexpr (T == P_F8) {
      sw[p] = wsp[slab];
#pragma unroll
      for (int t = 0; t < TT; ++t) if constexpr (!ROUNDS) sx[p][t] = sp[t][slab];
    }
  };
  auto load = [&](int p, int slab) {
    if constexpr (!TAIL) load_slab(p, slab, std::true_type());
    else if constexpr (TT == 1 && T != P_I8) load_slab(p, slab, std::false_type());
    else if (((size_t)slab << 7) + 128 <= row_bytes) load_slab(p, slab, std::true_type());
    else load_slab(p, slab, std::false_type());
  };
  // a row's 128 columns lie in the four lanes c, c + 16, c + 32, c + 48
  auto round_x = [&](int p, int t) {
    float f[32], m = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) { f[k] = finite_or_nan(raw[p][t][k >> 3].get(k & 7)); m = fmaxf(m, fabsf(f[k])); }
    u2s r = __builtin_amdgcn_permlane16_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    m = fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    m = fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
    const int e = e4m3_exponent((double)m);
    const float inv = exp2i(-e);
    sx[p][t] = exp2i(e);
#pragma unroll
    for (int k = 0; k < 8; ++k) B[p][t][k >> 2][k & 3] = pack_e4m3(f[4 * k] * inv, f[4 * k + 1] * inv, f[4 * k + 2] * inv, f[4 * k + 3] * inv);
  };
#pragma unroll
  for (int p = 0; p < P; ++p) if (wv + p * STREAM_WAVES < slabs) load(p, wv + p * STREAM_WAVES);
  for (int s0 = wv; s0 < slabs; s0 += P * STREAM_WAVES) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int slab = s0 + p * STREAM_WAVES;
      if (slab < slabs) {
        if constexpr (ROUNDS) {
#pragma unroll
          for (int t = 0; t < TT; ++t) round_x(p, t);
        }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
          for (int t = 0; t < TT; ++t) {
            if constexpr (WIDE) {
              const Wide a = widen(A[p][i]), b = widen(B[p][t]);
              f4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int k = 0; k < 4; ++k) part = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[k], b.v[k], part, 0, 0, 0);
              acc[i][t] += part * (sx[p][t] * sw[p]);
            } else if constexpr (T == P_F8) {
              acc[i][t] += mfma_f8(A[p][i][0], A[p][i][1], B[p][t][0], B[p][t][1]) * (sx[p][t] * sw[p]);
            } else {
              acc[i][t] = mfma_16<T>(A[p][i][0], B[p][t][0], acc[i][t]);
              acc[i][t] = mfma_16<T>(A[p][i][1], B[p][t][1], acc[i][t]);
            }
          }
        if (slab + P * STREAM_WAVES < slabs) load(p, slab + P * STREAM_WAVES);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int t = 0; t < TT; ++t) *(Sum*)&red[wv][(i * TT + t) * 256 + lane * 4] = acc[i][t];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < STORES; ++k) {
    const int idx = threadIdx.x + k * STREAM_WAVES * 64;
    if (R * TT * 256 % (STREAM_WAVES * 64) != 0 && idx >= R * TT * 256) break;
    const int i = idx % (16 * R), t = idx / (16 * R);            // matrix row, row of x
    const int at = ((i >> 4) * TT + (t >> 4)) * 256 + (((i & 15) >> 2) * 16 + (t & 15)) * 4 + (i & 3);
    One sum = 0;
#pragma unroll
    for (int w = 0; w < STREAM_WAVES; ++w) sum += red[w][at];
    if (t < s.count && m0 + i < a.m) {
      float v = (float)sum;
      if constexpr (T == P_I8) v = v * row_scale[k] * matrix_scale[k];
      if (a.bias != nullptr) v += load_elem_g(a.bias, a.y_dtype, m0 + i);
      store_elem_g(a.y, a.y_dtype, (size_t)(s.first + t) * a.m + m0 + i, v);
    }
  }
}

// ------------------------------------------------------------------------------------------------ many rows
// Bound: the matrix unit (its power) for thousands of rows, LDS loads' latency below, HBM where every expert has few.  8192 rows on 14336x4096 in e4m3 418 us, 2.3 PFLOP/s
// (the library with one scale 2.9); 24576 rows of 64 experts of 2048x1408 in 16 bits 187 us.  A slab of a 256x256 tile takes 1.6 us in 16 bits and 1.8 in e4m3.
// A workgroup of WM x WN waves takes tiles of TM = 16 AT WM rows of a matrix by TN = 16 BT WN rows of x, one after the other, their slabs one stream: slabs go
// from memory straight to LDS, a ring of NS stages.  While one slab is multiplied from registers, the next one is read, and the one NS behind is asked for;
// a tile's last products run while the next tile's first slabs arrive, and its results go out during the next one's products.
// LDS rows are 128 bytes in eight chunks of 16; chunk c of row r lies at place c ^ swizzle(r).  A 16-byte read serves 16 lanes at a time: lanes 0-3, 12-15,
// 20-23, 24-27, then 4-11, 16-19, 28-31, and the same of the upper half (measured: which pairs of lanes slow each other down on one bank), that is
// four fours of rows; two rows lie side by side in the banks, and the swizzles put the fours on different pairs of places.
// Row number 4 q + j of a wave's MFMA tiles 2 h and 2 h + 1 are its rows 32 h + 8 q + j and + 4: a lane then holds eight consecutive outputs, and four
// lanes 64 bytes of a row in 16 bits.
// GATED: the matrix is gate over up, m / 2 rows each; a tile takes TM / 2 of either, 32 by 32 in turn, so that a lane holds gate and up of eight consecutive
// hidden columns; y [rows][m / 2] is silu(gate) up, in 16 bits, in float32 (int8: a row's scale is not known before its last column, and values rounded to 16 bits before would
// fall on another integer here and there, 0.8 % of the result's norm) or in e4m3 (then TM / 2 = 128 columns share a scale); rows behind the last expert's are left.
// int8: the sums stay in the matrix unit's registers over all slabs, and the scales meet them at a tile's end, from LDS: 8192 rows on 14336x4096 392 to 412 us (2.33 to 2.45
// POP/s, the library's 8192^3 product 2.36), 465 with scales loaded where they are used; 24576 rows of 64 experts of 2048x1408 110; 333 rows on 6144x4096 22.
__device__ __forceinline__ int swizzle_w(int r) { return ((r >> 1) & 1) | ((r >> 3 & 3) << 1); }
__device__ __forceinline__ int swizzle_x(int r) { return (r >> 1) & 7; }
constexpr int TILE_XCDS = 8, TOGETHER = 8;

// eight consecutive outputs of a row, from i on, as far as the row goes
template <int Y> __device__ __forceinline__ void store8(const ProductArgs& a, float (&f)[8], size_t at, int i) {
  if (a.bias != nullptr) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] += load_elem_g(a.bias, Y, min(i + k, a.m - 1));
  }
  if ((a.m & 7) == 0) {
    Eight<Y> v;
    v.set(f);
    v.store(a.y, at);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) if (i + k < a.m) store_elem_g(a.y, Y, at + k, f[k]);
  }
}

// floats of a tile's scales in int8, whole loads of a wave
constexpr int scales_of_tile(int tm, int tn) { return (tm + tn + 63) / 64 * 64; }

template <int T, int WM, int WN, int AT, int BT, int NS, bool GATED>
__global__ __launch_bounds__(WM * WN * 64, 2) void k_product_tile(const ProductArgs a, int mtiles) {
  constexpr int WAVES = WM * WN, TM = 16 * AT * WM, TN = 16 * BT * WN;
  constexpr int XW = (TN + 63) / 64;                             // waves that load rows' scales
  constexpr int SCALES = T == P_F8 ? XW * 256 + 256 : 0, STAGE = (TM + TN) * 128 + SCALES;    // e4m3: the rows' scales, then the matrix's
  constexpr int LW = TM / 8 / WAVES, LX = TN / 8 / WAVES, L = LW + LX;        // 1 KB loads of a wave to a stage
  constexpr int RA = T == P_F8 || AT < 4 || (T == P_I8 && AT > 4) ? 2 : 4;      // MFMA tiles of the matrix in registers
  constexpr int BARRIER = AT - RA + 1;                           // the tile of products before which the next slab has landed
  constexpr bool WIDE = GATED && T == P_F8 && BT <= 2;           // float32 sums of what is rounded to e4m3 next
  static_assert(T != P_F8 || XW < WAVES, "a wave for the matrix's scales");
  static_assert(AT % 2 == 0 && TM % (8 * WAVES) == 0 && TN % (8 * WAVES) == 0 && AT % RA == 0, "whole loads, registers in turn");
  static_assert(!GATED || (AT % 4 == 0 && (T != P_F8 || TM == 256)), "32 gates and 32 ups to a wave; whole blocks of 128");
  constexpr int TILE_SCALES = T == P_I8 ? scales_of_tile(TM, TN) : 0;      // int8: two tiles' scales behind the ring, the matrix's, then the rows'
  extern __shared__ __align__(16) uint8_t lds[];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
  const int wm = wv / WN, wn = wv % WN;
  const size_t row_bytes = (size_t)a.n * bytes_of<T>;
  const int slabs = (int)((row_bytes + 127) >> 7);
  // Workgroups go to the eight XCDs in turn: neighbouring tiles to one XCD, one for each of its workgroups as far as there are tiles, TOGETHER tiles of x by a few
  // of the matrix, whose rows its L2 serves to several of them; the next run to the next XCD.  The launch knows a bound of the tiles only: without
  // counting them whole XCDs would come to nothing.
  const int ttiles = count_spans(a, TN), total = mtiles * ttiles;
  const int run = min((int)gridDim.x, (total + TILE_XCDS - 1) / TILE_XCDS * TILE_XCDS) / TILE_XCDS, nth = blockIdx.x / TILE_XCDS;
  int id = nth < run ? (int)(blockIdx.x % TILE_XCDS) * run + nth : total;

  // The tile in hand, and the next one that has products, if there is one; rows behind the last expert's become zeros on the way
  struct Tile { Span s; int m0; };
  Tile mine, then;
  auto find = [&](Tile& t) {
    for (; id < total; id += gridDim.x) {
      const int strip = id / (mtiles * TOGETHER), t0 = strip * TOGETHER, high = min(TOGETHER, ttiles - t0);
      const int rest = id - strip * mtiles * TOGETHER;
      t.m0 = rest / high * TM;
      t.s = find_span(a, TN, t0 + rest % high);
      if (t.s.e == a.experts) { if constexpr (!GATED) zero_rows(a, t.s, t.m0, TM); }
      else if (t.s.e >= 0) return true;
    }
    return false;
  };
  if (!find(mine)) return;
  // Where a lane's loads of a tile start: 32-bit distances from the tile's first row of either operand (from x where rows are gathered), so that a load takes
  // one register of address
  struct Source {
    const HTR_GLOBAL uint8_t *w, *x;
    const HTR_GLOBAL float* scales;
    uint32_t off[L], scale;
  };
  auto row_of = [&](int j) { return ((j < LW ? j : j - LW) * WAVES + wv) * 8 + (lane >> 3); };
  auto chunk_of = [&](int j) { return (lane & 7) ^ (j < LW ? swizzle_w(row_of(j)) : swizzle_x(row_of(j))); };
  auto source = [&](const Tile& t, Source& to) {
    to.w = (const HTR_GLOBAL uint8_t*)a.w + ((size_t)t.s.e * a.m + (GATED ? 0 : t.m0)) * row_bytes;
    to.x = (const HTR_GLOBAL uint8_t*)a.x + (a.gather != nullptr ? 0 : (size_t)t.s.first * row_bytes);
#pragma unroll
    for (int j = 0; j < L; ++j) {
      int r = row_of(j);
      if (GATED && j < LW) {
        r = min((t.m0 >> 1) + (r >> 6 << 5) + (r & 31), (a.m >> 1) - 1) + (r & 32 ? a.m >> 1 : 0);
      } else if (j < LW) {
        r = min(r, a.m - 1 - t.m0);      // beyond the matrix, or the expert's rows: the last row, whose results are not stored
      } else {
        r = min(r, t.s.count - 1);
        if (a.gather != nullptr) r = a.gather[t.s.first + r];
      }
      to.off[j] = (uint32_t)r * (uint32_t)row_bytes + 16 * chunk_of(j);
    }
    // A slab's scales come with it, through LDS: as loads into registers they would make the wave wait for all the loads issued after them.  Waves
    // 0 .. XW - 1 take 64 rows' each, the others the matrix's (one for each 128 rows; all the same, since a branch costs registers all over the loop).
    if constexpr (T == P_F8) {
      if (wv < XW) {
        int r = min(wv * 64 + lane, t.s.count - 1);
        if (a.gather != nullptr) r = a.gather[t.s.first + r];
        to.scales = (const HTR_GLOBAL float*)a.xs + (a.gather != nullptr ? 0 : (size_t)t.s.first * (a.n >> 7));
        to.scale = (uint32_t)r * (uint32_t)(a.n >> 7);
      } else {
        const int blocks = (a.m + 127) >> 7;
        const int block = t.m0 >> (GATED ? 8 : 7);      // GATED: the gates' in the first place, the ups' in the second
        to.scales = (const HTR_GLOBAL float*)a.ws + ((size_t)t.s.e * blocks + block) * (a.n >> 7);
        to.scale = (uint32_t)(GATED ? (lane & 1) * (blocks >> 1) : min(lane, blocks - 1 - block)) * (uint32_t)(a.n >> 7);
      }
    }
  };
  Source src, src2;
  source(mine, src);
  // Other than e4m3 rows may end inside the last slab, at a multiple of 16 bytes: chunks from there on are loaded as the slab's first, and zeroed in LDS
  const int tail = (int)(row_bytes & 127) >> 4;
  auto place = [&](int j, int stage) { return stage * STAGE + (j < LW ? (j * WAVES + wv) * 1024 : TM * 128 + ((j - LW) * WAVES + wv) * 1024); };
  auto issue = [&](Source& src, int slab, int stage, int from, int to) {
#pragma unroll
    for (int j = from; j < to; ++j) {
      asm volatile("" : "+v"(src.off[j]));                         // or the compiler keeps 64-bit addresses
      uint32_t off = src.off[j];
      if (T != P_F8 && tail != 0 && slab == slabs - 1) { const int ch = chunk_of(j); off -= ch >= tail ? 16 * ch : 0; }      // it holds 16 ch
      const HTR_GLOBAL uint8_t* p = (j < LW ? src.w : src.x) + ((size_t)slab << 7) + off;
      __builtin_amdgcn_global_load_lds((const HTR_GLOBAL void*)p, (__attribute__((address_space(3))) void*)(lds + place(j, stage)), 16, 0, 0);
    }
  };
  auto issue_scales = [&](const Source& src, int slab, int stage) {
    if constexpr (T == P_F8)
      __builtin_amdgcn_global_load_lds((const HTR_GLOBAL void*)(src.scales + slab + src.scale),
                                       (__attribute__((address_space(3))) void*)(lds + stage * STAGE + (TM + TN) * 128 + min(wv, XW) * 256), 4, 0, 0);
  };
  // int8: a tile's scales, asked for NS - 1 slabs or more ahead of its first product, so that `landed` has waited for them long before its last.  One load more than it counts makes it
  // wait longer, never shorter.
  auto issue_tile_scales = [&](const Tile& t, int which) {
    if constexpr (T == P_I8) {
#pragma unroll
      for (int k = 0; k < TILE_SCALES; k += WAVES * 64) {
        if (k + wv * 64 >= TILE_SCALES) break;
        const int j = k + wv * 64 + lane;
        const HTR_GLOBAL float* p = (const HTR_GLOBAL float*)a.ws + (size_t)t.s.e * a.m;
        if (j >= TM) {
          int r = t.s.first + min(j - TM, t.s.count - 1);
          if (a.gather != nullptr) r = a.gather[r];
          p = (const HTR_GLOBAL float*)a.xs + r;
        } else if (GATED) {
          const int half = TM / 2, F = a.m >> 1;
          p += min((t.m0 >> 1) + (j < half ? j : j - half), F - 1) + (j < half ? 0 : F);
        } else {
          p += min(t.m0 + j, a.m - 1);
        }
        __builtin_amdgcn_global_load_lds((const HTR_GLOBAL void*)p, (__attribute__((address_space(3))) void*)(lds + NS * STAGE + (which * TILE_SCALES + k + wv * 64) * 4), 4, 0, 0);
      }
    }
  };
  // The stage is there for every wave, and every wave has read all of the one before.  `behind`: later loads of this wave, which may still be on their way (they
  // arrive in order; results being stored in between only make the wait longer); `last`: the stage holds its tile's last slab
  auto landed = [&](int stage, bool last, auto behind) {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(decltype(behind)::value) : "memory");
    if (T != P_F8 && tail != 0 && last) {
#pragma unroll
      for (int j = 0; j < L; ++j) if (chunk_of(j) >= tail) *(u4*)(lds + place(j, stage) + 16 * lane) = u4{0u, 0u, 0u, 0u};
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  // where a lane reads its first chunk of each tile of either operand; the second lies at place ^ 4
  int ra[AT], rb[BT];
#pragma unroll
  for (int i = 0; i < AT; ++i) {
    const int r = wm * 16 * AT + 32 * (i >> 1) + 8 * (c >> 2) + 4 * (i & 1) + (c & 3);
    ra[i] = r * 128 + 16 * (g ^ swizzle_w(r));
  }
#pragma unroll
  for (int t = 0; t < BT; ++t) {
    const int r = wn * 16 * BT + 16 * t + c;
    rb[t] = TM * 128 + r * 128 + 16 * (g ^ swizzle_x(r));
  }
  u4 A[RA][2], B[BT][2];
  float sx[BT], sw[GATED ? 2 : 1];
  auto read_a = [&](int i, int stage) {
    const uint8_t* base = lds + stage * STAGE;
    A[i % RA][0] = *(const u4*)(base + ra[i]); A[i % RA][1] = *(const u4*)(base + (ra[i] ^ 64));
  };
  auto read_b = [&](int t, int stage) {
    const uint8_t* base = lds + stage * STAGE;
    B[t][0] = *(const u4*)(base + rb[t]); B[t][1] = *(const u4*)(base + (rb[t] ^ 64));
  };
  auto read_scales = [&](int stage) {
    const float* base = (const float*)(lds + stage * STAGE + (TM + TN) * 128);
#pragma unroll
    for (int t = 0; t < BT; ++t) sx[t] = base[wn * 16 * BT + 16 * t + c];
    if constexpr (GATED) { sw[0] = base[XW * 64]; sw[1] = base[XW * 64 + 1]; } else sw[0] = base[XW * 64 + ((wm * 16 * AT) >> 7)];
  };
  typedef typename SumOf<T>::type Sum;
  Sum acc[AT][BT];
#pragma unroll
  for (int i = 0; i < AT; ++i)
#pragma unroll
    for (int t = 0; t < BT; ++t) acc[i][t] = Sum{0, 0, 0, 0};
  int stage = 0;                                                 // of the slab in registers
  auto after = [](int st, int by) { const int to = st + by; return to >= NS ? to - NS : to; };
  constexpr int PIECES = AT < 4 ? AT : 4;                        // MFMA tiles over which the loads of a slab are spread
  auto issue_piece = [&](Source& from, int slab, int to, int piece) {
    if (piece < PIECES) issue(from, slab, to, piece * L / PIECES, (piece + 1) * L / PIECES);
  };
  // The products of the slab in registers, while the operands of the next one are read.  Every wave has read all of this slab RA - 1 MFMA tiles ahead of
  // its last product; there lies the barrier, behind which the slab NS after this one, `ask`, is asked for, into this one's stage: a few loads with each
  // MFMA tile, the first of the next call's among them (`asked`); all at once they would keep the wave from its products for as long as they take to issue
  auto multiply = [&](int asked, Source& from, int ask, Source& from2, bool last_lands) {
    float sc[GATED ? 2 : 1][BT];
    f4 part[3];
    const int next = after(stage, 1), prev = after(stage, NS - 1);
    if constexpr (T == P_F8) {
#pragma unroll
      for (int t = 0; t < BT; ++t) {
        sc[0][t] = sx[t] * sw[0];
        if constexpr (GATED) sc[1][t] = sx[t] * sw[1];
      }
    }
    Wide wide[WIDE ? BT : 1];                                     // the slab's rows of x in f16
    if constexpr (WIDE) {
#pragma unroll
      for (int t = 0; t < BT; ++t) wide[t] = widen(B[t]);
    }
    f4 sums[2][WIDE ? BT : 1];
    auto add_sums = [&](int i) {
      if constexpr (WIDE) {
#pragma unroll
        for (int t = 0; t < BT; ++t) acc[i][t] += sums[i & 1][t] * sc[GATED ? i >> 1 & 1 : 0][t];
      }
    };
#pragma unroll
    for (int i = 0; i < AT; ++i) {
      if (i == 0) __builtin_amdgcn_s_setprio(1);                 // a wave with products ahead of one that waits or loads: 1 to 2 %
      if (i == BARRIER) {
        __builtin_amdgcn_s_setprio(0);
        landed(next, last_lands, std::integral_constant<int, (NS - 2) * (L + (T == P_F8))>());
        issue_scales(from2, ask, stage);
        if constexpr (T == P_F8) read_scales(next);
      }
      if (i < BARRIER) issue_piece(from, asked, prev, i + AT - BARRIER); else issue_piece(from2, ask, stage, i - BARRIER);
      if (i + RA - 1 < AT) read_a(i + RA - 1, stage); else read_a(i + RA - 1 - AT, next);
      if constexpr (WIDE) {
        const Wide a = widen(A[i % RA]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int t = 0; t < BT; ++t) sums[i & 1][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[k], wide[t].v[k], k == 0 ? f4{0.f, 0.f, 0.f, 0.f} : sums[i & 1][t], 0, 0, 0);
        if (i > 0) add_sums(i - 1);
      }
#pragma unroll
      for (int t = 0; t < BT; ++t) {
        if constexpr (WIDE) {
        } else if constexpr (T == P_F8) {
          // the sums two products behind the matrix unit
          const int k = i * BT + t, l = k - 2;
          part[k % 3] = mfma_f8(A[i % RA][0], A[i % RA][1], B[t][0], B[t][1]);
          if (l >= 0) acc[l / BT][l % BT] += part[l % 3] * sc[GATED ? l / BT >> 1 & 1 : 0][l % BT];
        } else {
          acc[i][t] = mfma_16<T>(A[i % RA][0], B[t][0], acc[i][t]);
          acc[i][t] = mfma_16<T>(A[i % RA][1], B[t][1], acc[i][t]);
        }
        if (i == AT - 1) read_b(t, next);
      }
      if constexpr (WIDE) {
        // conversions, and the sums of the tile before, between the products
#pragma unroll
        for (int t = 0; t < 4 * BT; ++t) { __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); __builtin_amdgcn_sched_group_barrier(0x002, 3, 0); }
      } else if constexpr (T == P_F8) {
        // a product, then the four sums of the one two before it: left to itself the compiler waits for results just asked for
#pragma unroll
        for (int t = 0; t < BT; ++t) { __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); __builtin_amdgcn_sched_group_barrier(0x002, 4, 0); }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (WIDE) {
      add_sums(AT - 1);
    } else if constexpr (T == P_F8) {
#pragma unroll
      for (int l = AT * BT - 2; l < AT * BT; ++l) acc[l / BT][l % BT] += part[l % 3] * sc[GATED ? l / BT >> 1 & 1 : 0][l % BT];
    }
    stage = next;
  };
  issue_tile_scales(mine, 0);
  int which = 0;                                                 // int8: the half of the scales' place that the tile in hand has
  // slabs behind the last one: the last one again, for nothing
#pragma unroll
  for (int st = 0; st < NS - 1; ++st) {
    issue_scales(src, min(st, slabs - 1), st);
    issue(src, min(st, slabs - 1), st, 0, L);
  }
  int asked = min(NS - 1, slabs - 1);
  issue_scales(src, asked, NS - 1);
#pragma unroll
  for (int piece = 0; piece < AT - BARRIER; ++piece) issue_piece(src, asked, NS - 1, piece);
  landed(0, slabs == 1, std::integral_constant<int, (NS - 2) * (L + (T == P_F8))>());
#pragma unroll
  for (int i = 0; i < RA - 1; ++i) read_a(i, 0);
#pragma unroll
  for (int t = 0; t < BT; ++t) read_b(t, 0);
  if constexpr (T == P_F8) read_scales(0);
  bool more = false;
  src2 = src;
  for (int slab = 0;;) {
    // the last NS slabs of a tile ask for the next one's first; where there is no next tile, for their own tile's again, for nothing
    if (slab + NS == slabs) {
      id += gridDim.x;
      more = find(then);
      if (more) {
        source(then, src2);
        // with as many slabs as stages no barrier has passed since the tile before was stored: a wave may still read that half of the scales' place
        if (T == P_I8 && slab == 0) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        issue_tile_scales(then, which ^ 1);
      }
    }
    const int ask = slab + NS < slabs ? slab + NS : slabs >= NS ? slab + NS - slabs : slabs - 1;
    multiply(asked, src, ask, src2, slab + 2 == slabs);
    asked = ask;
    src = src2;
    if (++slab < slabs) continue;
    slab = 0;
    // int8: the scales of the lane's rows of x, and of eight consecutive rows of the matrix
    const float* tile_scales = (const float*)(lds + NS * STAGE) + which * TILE_SCALES;
    auto row_scale = [&](int t) { return tile_scales[TM + wn * 16 * BT + 16 * t + c]; };
    auto matrix_scales = [&](int i, float (&w)[8]) {
      const f4 lo = *(const f4*)(tile_scales + i), hi = *(const f4*)(tile_scales + i + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) { w[k] = lo[k]; w[4 + k] = hi[k]; }
    };
    if constexpr (GATED && T == P_I8) {
      const int F = a.m >> 1, i0 = (mine.m0 >> 1) + wm * 8 * AT + 8 * g;      // hidden columns; first of the lane's
      float rs[BT];
#pragma unroll
      for (int t = 0; t < BT; ++t) rs[t] = row_scale(t);
#pragma unroll
      for (int h = 0; h < AT / 4; ++h) {
        float gate[8], up[8];
        matrix_scales(wm * 8 * AT + 8 * g + 32 * h, gate);
        matrix_scales(TM / 2 + wm * 8 * AT + 8 * g + 32 * h, up);
#pragma unroll
        for (int t = 0; t < BT; ++t) {
          float f[8];
#pragma unroll
          for (int k = 0; k < 8; ++k)
            f[k] = silu((float)acc[4 * h + (k >> 2)][t][k & 3] * rs[t] * gate[k]) * ((float)acc[4 * h + 2 + (k >> 2)][t][k & 3] * rs[t] * up[k]);
          const int r = wn * 16 * BT + 16 * t + c;
          if (r < mine.s.count && i0 + 32 * h < F) { Eight<HTR_F32> v; v.set(f); v.store(a.y, (size_t)(mine.s.first + r) * F + i0 + 32 * h); }
        }
      }
    } else if constexpr (GATED) {
      const int F = a.m >> 1, i0 = (mine.m0 >> 1) + wm * 8 * AT + 8 * g;      // hidden columns; first of the lane's
      float amax[BT];
#pragma unroll
      for (int t = 0; t < BT; ++t) {
        amax[t] = 0.f;
#pragma unroll
        for (int h = 0; h < AT / 4; ++h)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            float v = silu(acc[4 * h + (k >> 2)][t][k & 3]) * acc[4 * h + 2 + (k >> 2)][t][k & 3];
            if constexpr (T == P_F8) { v = finite_or_nan(v); amax[t] = fmaxf(amax[t], fabsf(v)); }
            acc[4 * h + (k >> 2)][t][k & 3] = v;
          }
      }
      if constexpr (T == P_F8) {
        // the waves' largest of each row; the last reads of the place lie a barrier of the main loop back
        float* place = (float*)(lds + NS * STAGE);
#pragma unroll
        for (int t = 0; t < BT; ++t) {
          amax[t] = fmaxf(amax[t], __shfl_xor(amax[t], 16));
          amax[t] = fmaxf(amax[t], __shfl_xor(amax[t], 32));
          if (g == 0) place[wm * TN + wn * 16 * BT + 16 * t + c] = amax[t];
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
        for (int t = 0; t < BT; ++t) {
          const int r = wn * 16 * BT + 16 * t + c;
          float m = place[r];
#pragma unroll
          for (int k = 1; k < WM; ++k) m = fmaxf(m, place[k * TN + r]);
          const int e = e4m3_exponent((double)m);
          const float inv = exp2i(-e);
          if (r >= mine.s.count) continue;
          const size_t row = (size_t)(mine.s.first + r);
          if (wm == 0 && g == 0) ((HTR_GLOBAL float*)a.ys)[row * (F >> 7) + (mine.m0 >> 8)] = exp2i(e);
#pragma unroll
          for (int h = 0; h < AT / 4; ++h) {
            const f4 lo = acc[4 * h][t] * inv, hi = acc[4 * h + 1][t] * inv;
            *(HTR_GLOBAL u2*)((HTR_GLOBAL uint8_t*)a.y + row * F + i0 + 32 * h) = u2{pack_e4m3(lo.x, lo.y, lo.z, lo.w), pack_e4m3(hi.x, hi.y, hi.z, hi.w)};
          }
        }
      } else {
#pragma unroll
        for (int t = 0; t < BT; ++t) {
          const int r = wn * 16 * BT + 16 * t + c;
#pragma unroll
          for (int h = 0; h < AT / 4; ++h) {
            float f[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = acc[4 * h + (k >> 2)][t][k & 3];
            if (r < mine.s.count && i0 + 32 * h < F) { Eight<T> v; v.set(f); v.store(a.y, (size_t)(mine.s.first + r) * F + i0 + 32 * h); }
          }
        }
      }
    } else {
      const int i0 = mine.m0 + wm * 16 * AT + 8 * g;               // first of the lane's outputs
      auto put = [&](auto type) {
        constexpr int Y = decltype(type)::value;
        auto each = [&](int t, int h, auto scaled) {
          const int r = wn * 16 * BT + 16 * t + c;
          float f[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) f[k] = scaled((float)acc[2 * h + (k >> 2)][t][k & 3], k);
          if (r < mine.s.count && i0 + 32 * h < a.m) store8<Y>(a, f, (size_t)(mine.s.first + r) * a.m + i0 + 32 * h, i0 + 32 * h);
        };
        if constexpr (T == P_I8) {
          float ws[8], rs[BT];
#pragma unroll
          for (int t = 0; t < BT; ++t) rs[t] = row_scale(t);
#pragma unroll
          for (int h = 0; h < AT / 2; ++h) {
            matrix_scales(wm * 16 * AT + 8 * g + 32 * h, ws);
#pragma unroll
            for (int t = 0; t < BT; ++t) each(t, h, [&](float v, int k) { return v * rs[t] * ws[k]; });
          }
        } else {
#pragma unroll
          for (int t = 0; t < BT; ++t)
#pragma unroll
            for (int h = 0; h < AT / 2; ++h) each(t, h, [](float v, int) { return v; });
        }
      };
      if (a.y_dtype == HTR_BF16) put(std::integral_constant<int, HTR_BF16>());
      else if (a.y_dtype == HTR_F16) put(std::integral_constant<int, HTR_F16>());
      else put(std::integral_constant<int, HTR_F32>());
    }
#pragma unroll
    for (int i = 0; i < AT; ++i)
#pragma unroll
      for (int t = 0; t < BT; ++t) acc[i][t] = Sum{0, 0, 0, 0};
    if (!more) break;
    mine = then;
    which ^= 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // loads for nothing: they write to LDS
}
