// Part of unpacked.hip, included inside its anonymous namespace: products of rows with matrices that are not HTR-W1, one matrix or one for each expert.
//
//   y[r][i] = sum_k x[r][k] w_e[i][k],  e the expert of row r;  e4m3: the sum over each block of 128 columns times xs[r][k / 128] ws_e[i / 128][k / 128]
//
// Everything is cut into slabs of 128 bytes of a row: 128 e4m3 values, one v_mfma_f32_16x16x128_f8f6f4 whose result is scaled into the sum, or
// 64 16-bit ones, two v_mfma_f32_16x16x32.  A lane feeds bytes 16 g .. and 64 + 16 g .. of its row (g = lane / 16): another order of the
// columns than the instructions' own, the same for both operands.  Matrix rows are MFMA rows (D: rows 4 g + i, four to a lane), activation
// rows are MFMA columns (lane % 16), so that a lane holds consecutive outputs of one row.
enum { P_F8 = 3 };                       // beside HTR_BF16, HTR_F16: the operands' type
template <int T> constexpr int bytes_of = T == P_F8 ? 1 : 2;
typedef int i8v __attribute__((ext_vector_type(8)));

struct ProductArgs {
  const void* x;                         // [.][n]
  const float* xs;                       // e4m3: [.][n / 128]
  const void* w;                         // [experts][m][n]
  const float* ws;                       // e4m3: [experts][ceil(m / 128)][n / 128]
  const void* bias;                      // [m] in y's type or NULL
  void* y;                               // [rows][m]
  const int* ends;                       // [experts]: expert e has rows ends[e - 1] .. ends[e] - 1; NULL: one expert, all rows
  const int* gather;                     // row r of the product is row gather[r] of x; NULL: r
  int rows, m, n, experts, y_dtype;
};

// Rows first .. first + count - 1 of expert e are tile number t of tiles of `height` rows, expert by expert; e = experts: rows behind the last
// expert's; e = -1: no such tile.  Ends are taken as what they may be: at least the one before, at least 0, at most `rows`.
struct Span { int e, first, count; };
__device__ __forceinline__ Span find_span(const ProductArgs& a, int height, int t) {
  if (a.ends == nullptr) {
    const int first = t * height;
    return first < a.rows ? Span{0, first, min(height, a.rows - first)} : Span{-1, 0, 0};
  }
  const int lane = threadIdx.x & 63;
  int end0 = 0, tiles0 = 0;
  for (int base = 0; base < a.experts; base += 64) {
    int end = base + lane < a.experts ? min(a.ends[base + lane], a.rows) : 0;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) { const int u = __shfl_up(end, off); if (lane >= off) end = max(end, u); }
    end = max(end, end0);
    int start = __shfl_up(end, 1);
    if (lane == 0) start = end0;
    const int tiles = (end - start + height - 1) / height;
    int sum = tiles;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) { const int u = __shfl_up(sum, off); if (lane >= off) sum += u; }
    sum += tiles0;
    const unsigned long long in = __ballot(sum > t);
    if (in) {
      const int l = __builtin_ctzll(in);
      const int skip = (t - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(tiles, l))) * height;
      const int first = __builtin_amdgcn_readlane(start, l) + skip;
      return Span{base + l, first, min(height, __builtin_amdgcn_readlane(end, l) - first)};
    }
    end0 = __builtin_amdgcn_readlane(end, 63);
    tiles0 = __builtin_amdgcn_readlane(sum, 63);
  }
  // t - tiles0 tiles behind the last expert's; the grid is a bound, so this may lie beyond 32 bits of rows
  const long long first = end0 + (long long)(t - tiles0) * height;
  return first < a.rows ? Span{a.experts, (int)first, min(height, a.rows - (int)first)} : Span{-1, 0, 0};
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

__device__ __forceinline__ f4 mfma_f8(const u4& a0, const u4& a1, const u4& b0, const u4& b1) {
  const i8v a = {(int)a0.x, (int)a0.y, (int)a0.z, (int)a0.w, (int)a1.x, (int)a1.y, (int)a1.z, (int)a1.w};
  const i8v b = {(int)b0.x, (int)b0.y, (int)b0.z, (int)b0.w, (int)b1.x, (int)b1.y, (int)b1.z, (int)b1.w};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}
template <int T> __device__ __forceinline__ f4 mfma_16(const u4& a, const u4& b, const f4& c) {
  if constexpr (T == HTR_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// four consecutive outputs of a row, from i on, as far as the row goes
__device__ __forceinline__ void store4(const ProductArgs& a, f4 v, int row, int i) {
  const size_t at = (size_t)row * a.m + i;
  if (a.bias != nullptr) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] += load_elem_g(a.bias, a.y_dtype, min(i + k, a.m - 1));
  }
  if ((a.m & 3) == 0) {
    if (a.y_dtype == HTR_F32) *(HTR_GLOBAL f4*)((HTR_GLOBAL float*)a.y + at) = v;
    else *(HTR_GLOBAL u2*)((HTR_GLOBAL uint16_t*)a.y + at) = a.y_dtype == HTR_BF16 ? u2{pack_bf16(v.x, v.y), pack_bf16(v.z, v.w)} : u2{pack_f16(v.x, v.y), pack_f16(v.z, v.w)};
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) if (i + k < a.m) store_elem_g(a.y, a.y_dtype, at + k, v[k]);
  }
}

// ------------------------------------------------------------------------------------------------ few rows
// A workgroup owns 16 R rows of a matrix and up to 16 TT rows of x; its eight waves take the slabs in turn, straight from memory into registers
// (every byte of the matrix is used by one wave once: LDS would only be a detour), and add up through LDS.
// Bound: HBM, the matrix read once.
constexpr int STREAM_WAVES = 8;
template <int T, int R, int TT>
__global__ __launch_bounds__(STREAM_WAVES * 64) void k_product_stream(const ProductArgs a) {
  constexpr int P = R + TT <= 3 ? 4 : 2;                       // slabs in flight
  __shared__ float red[STREAM_WAVES][R * TT * 256];
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
    xp[t] = (const HTR_GLOBAL uint8_t*)a.x + (size_t)r * row_bytes + 16 * g;
    sp[t] = (const HTR_GLOBAL float*)a.xs + (size_t)r * (a.n >> 7);
  }
  const HTR_GLOBAL float* wsp = (const HTR_GLOBAL float*)a.ws + ((size_t)s.e * ((a.m + 127) >> 7) + (m0 >> 7)) * (a.n >> 7);
  f4 acc[R][TT];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[i][t] = f4{0.f, 0.f, 0.f, 0.f};
  u4 A[P][R][2], B[P][TT][2];
  float sx[P][TT], sw[P];
  const u4 zero = {0u, 0u, 0u, 0u};
  auto load = [&](int p, int slab) {
    const size_t off = (size_t)slab << 7;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // 16-bit rows may end inside the slab, at a multiple of 16 bytes
      const bool in = T == P_F8 || off + 64 * h + 16 * g < row_bytes;
#pragma unroll
      for (int i = 0; i < R; ++i) { A[p][i][h] = zero; if (in) A[p][i][h] = __builtin_nontemporal_load((const HTR_GLOBAL u4*)(wp[i] + off + 64 * h)); }
#pragma unroll
      for (int t = 0; t < TT; ++t) { B[p][t][h] = zero; if (in) B[p][t][h] = *(const HTR_GLOBAL u4*)(xp[t] + off + 64 * h); }
    }
    if constexpr (T == P_F8) {
      sw[p] = wsp[slab];
#pragma unroll
      for (int t = 0; t < TT; ++t) sx[p][t] = sp[t][slab];
    }
  };
#pragma unroll
  for (int p = 0; p < P; ++p) if (wv + p * STREAM_WAVES < slabs) load(p, wv + p * STREAM_WAVES);
  for (int s0 = wv; s0 < slabs; s0 += P * STREAM_WAVES) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int slab = s0 + p * STREAM_WAVES;
      if (slab < slabs) {
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
          for (int t = 0; t < TT; ++t) {
            if constexpr (T == P_F8) {
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
    for (int t = 0; t < TT; ++t) *(f4*)&red[wv][(i * TT + t) * 256 + lane * 4] = acc[i][t];
  __syncthreads();
  for (int idx = threadIdx.x; idx < R * TT * 256; idx += STREAM_WAVES * 64) {
    const int i = idx % (16 * R), t = idx / (16 * R);            // matrix row, row of x
    const int at = ((i >> 4) * TT + (t >> 4)) * 256 + (((i & 15) >> 2) * 16 + (t & 15)) * 4 + (i & 3);
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < STREAM_WAVES; ++k) v += red[k][at];
    if (t < s.count && m0 + i < a.m) {
      if (a.bias != nullptr) v += load_elem_g(a.bias, a.y_dtype, m0 + i);
      store_elem_g(a.y, a.y_dtype, (size_t)(s.first + t) * a.m + m0 + i, v);
    }
  }
}

// ------------------------------------------------------------------------------------------------ many rows
// A workgroup of WM x WN waves owns TM = 16 AT WM rows of a matrix and TN = 16 BT WN rows of x; slabs go from memory straight to LDS, two stages.
// LDS rows are 128 bytes in eight chunks of 16; chunk c of row r lies at place c ^ swizzle(r), so that the 16 lanes that read one chunk of
// 16 rows hit all banks, in halves of 8 lanes and whole.  Row number 4 q + j of a wave's MFMA tile i is its row 4 AT q + 4 i + j: a
// lane then holds 4 AT consecutive outputs.
__device__ const uint32_t k_zero_page[4] = {0u, 0u, 0u, 0u};
template <int AT> __device__ __forceinline__ int swizzle_w(int r) {
  const int q = r / (4 * AT), j = r & 3;
  return ((j ^ ((q >> 1) & 1)) | ((q & 1) << 2)) & 7;
}
__device__ __forceinline__ int swizzle_x(int r) { return (r ^ ((r >> 3) & 1)) & 7; }

template <int T, int WM, int WN, int AT, int BT>
__global__ __launch_bounds__(WM * WN * 64) void k_product_tile(const ProductArgs a, int mtiles, int ttiles, int together) {
  constexpr int WAVES = WM * WN, TM = 16 * AT * WM, TN = 16 * BT * WN, STAGE = (TM + TN) * 128;
  constexpr int LW = TM / 8 / WAVES, LX = TN / 8 / WAVES;        // 1 KB loads of a wave to a stage
  static_assert(TM % (8 * WAVES) == 0 && TN % (8 * WAVES) == 0, "whole loads");
  extern __shared__ __align__(16) uint8_t lds[];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
  const int wm = wv / WN, wn = wv % WN;
  // workgroups go to the eight XCDs in turn: each XCD gets a run of tiles, `together` tiles of x at a time over all of the matrix
  const int per = gridDim.x >> 3, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (id >= mtiles * ttiles) return;
  const int strip = id / (mtiles * together), t0 = strip * together, high = min(together, ttiles - t0);
  const int rest = id - strip * mtiles * together, mt = rest / high, tt = t0 + rest % high;
  const int m0 = mt * TM;
  const Span s = find_span(a, TN, tt);
  if (s.e < 0) return;
  if (s.e == a.experts) { zero_rows(a, s, m0, TM); return; }
  const size_t row_bytes = (size_t)a.n * bytes_of<T>;
  const int slabs = (int)((row_bytes + 127) >> 7);
  const HTR_GLOBAL uint8_t* src[LW + LX];
  uint32_t chunk_at[LW + LX];
#pragma unroll
  for (int j = 0; j < LW + LX; ++j) {
    const bool is_w = j < LW;
    const int r = ((is_w ? j : j - LW) * WAVES + wv) * 8 + (lane >> 3);
    const int ch = (lane & 7) ^ (is_w ? swizzle_w<AT>(r) : swizzle_x(r));
    chunk_at[j] = 16 * ch;
    if (is_w) {
      src[j] = (const HTR_GLOBAL uint8_t*)a.w + ((size_t)s.e * a.m + min(m0 + r, a.m - 1)) * row_bytes + 16 * ch;
    } else {
      int row = s.first + min(r, s.count - 1);
      if (a.gather != nullptr) row = a.gather[row];
      src[j] = (const HTR_GLOBAL uint8_t*)a.x + (size_t)row * row_bytes + 16 * ch;
    }
  }
  auto issue = [&](int slab, int stage) {
#pragma unroll
    for (int j = 0; j < LW + LX; ++j) {
      const HTR_GLOBAL uint8_t* p = src[j] + ((size_t)slab << 7);
      // 16-bit rows may end inside the last slab, at a multiple of 16 bytes: zeros there, in both operands
      if (T != P_F8 && ((size_t)slab << 7) + chunk_at[j] >= row_bytes) p = (const HTR_GLOBAL uint8_t*)k_zero_page;
      const int at = stage * STAGE + (j < LW ? (j * WAVES + wv) * 1024 : TM * 128 + ((j - LW) * WAVES + wv) * 1024);
      __builtin_amdgcn_global_load_lds((const HTR_GLOBAL void*)p, (__attribute__((address_space(3))) void*)(lds + at), 16, 0, 0);
    }
  };
  // where a lane reads its first chunk of tile 0 of either operand; the second lies at place ^ 4
  int ra[AT], rb[BT];
#pragma unroll
  for (int i = 0; i < AT; ++i) {
    const int r = wm * 16 * AT + (c >> 2) * 4 * AT + 4 * i + (c & 3);
    ra[i] = r * 128 + 16 * (g ^ swizzle_w<AT>(r));
  }
#pragma unroll
  for (int t = 0; t < BT; ++t) {
    const int r = wn * 16 * BT + 16 * t + c;
    rb[t] = TM * 128 + r * 128 + 16 * (g ^ swizzle_x(r));
  }
  const HTR_GLOBAL float* sp[BT];
  const HTR_GLOBAL float* wsp = (const HTR_GLOBAL float*)a.ws + ((size_t)s.e * ((a.m + 127) >> 7) + min((m0 + wm * 16 * AT) >> 7, (a.m - 1) >> 7)) * (a.n >> 7);
  float sx[BT], sw = 0.f;
  if constexpr (T == P_F8) {
#pragma unroll
    for (int t = 0; t < BT; ++t) {
      int row = s.first + min(wn * 16 * BT + 16 * t + c, s.count - 1);
      if (a.gather != nullptr) row = a.gather[row];
      sp[t] = (const HTR_GLOBAL float*)a.xs + (size_t)row * (a.n >> 7);
      sx[t] = sp[t][0];
    }
    sw = wsp[0];
  }
  f4 acc[AT][BT];
#pragma unroll
  for (int i = 0; i < AT; ++i)
#pragma unroll
    for (int t = 0; t < BT; ++t) acc[i][t] = f4{0.f, 0.f, 0.f, 0.f};
  issue(0, 0);
  for (int slab = 0; slab < slabs; ++slab) {
    const int stage = slab & 1;
    float sc[BT];
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();                     // this stage has landed for every wave, and nobody reads the other one any more
    if (slab + 1 < slabs) issue(slab + 1, stage ^ 1);
    if constexpr (T == P_F8) {
      const int next = min(slab + 1, slabs - 1);
#pragma unroll
      for (int t = 0; t < BT; ++t) { sc[t] = sx[t] * sw; sx[t] = sp[t][next]; }
      sw = wsp[next];
    }
    const uint8_t* base = lds + stage * STAGE;
    u4 B[BT][2];
#pragma unroll
    for (int t = 0; t < BT; ++t) { B[t][0] = *(const u4*)(base + rb[t]); B[t][1] = *(const u4*)(base + (rb[t] ^ 64)); }
#pragma unroll
    for (int i = 0; i < AT; ++i) {
      const u4 A0 = *(const u4*)(base + ra[i]), A1 = *(const u4*)(base + (ra[i] ^ 64));
#pragma unroll
      for (int t = 0; t < BT; ++t) {
        if constexpr (T == P_F8) {
          acc[i][t] += mfma_f8(A0, A1, B[t][0], B[t][1]) * sc[t];
        } else {
          acc[i][t] = mfma_16<T>(A0, B[t][0], acc[i][t]);
          acc[i][t] = mfma_16<T>(A1, B[t][1], acc[i][t]);
        }
      }
    }
  }
  // results: 16 rows of x at a time through the wave's own part of LDS, four consecutive outputs to a lane, so that a row's go out in whole lines
  __syncthreads();
  constexpr int PITCH = 16 * AT + 4, ACROSS = 4 * AT;            // floats of a row there, lanes to a row
  static_assert(WAVES * 16 * PITCH * 4 <= 2 * STAGE, "room");
  float* mine = (float*)lds + wv * 16 * PITCH;
  const int i0 = m0 + wm * 16 * AT + (lane % ACROSS) * 4;        // first of the lane's outputs
#pragma unroll
  for (int t = 0; t < BT; ++t) {
#pragma unroll
    for (int i = 0; i < AT; ++i) *(f4*)(mine + c * PITCH + g * ACROSS + 4 * i) = acc[i][t];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int r = lane / ACROSS; r < 16; r += 64 / ACROSS) {
      const f4 v = *(const f4*)(mine + r * PITCH + (lane % ACROSS) * 4);
      const int row = wn * 16 * BT + 16 * t + r;
      if (row < s.count && i0 < a.m) store4(a, v, s.first + row, i0);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}
