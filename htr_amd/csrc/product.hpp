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
// LDS rows are 128 bytes in eight chunks of 16; chunk c of row r lies at place c ^ swizzle(r).  A 16-byte read serves 16 lanes at a time: lanes 0-3, 12-15,
// 20-23, 24-27, then 4-11, 16-19, 28-31, and the same of the upper half (measured: which pairs of lanes slow each other down on one bank), that is
// four fours of rows; two rows lie side by side in the banks, and the swizzles put the fours on different pairs of places.
// Row number 4 q + j of a wave's MFMA tile i is its row 4 AT q + 4 i + j: a lane then holds 4 AT consecutive outputs.
template <int AT> __device__ __forceinline__ int swizzle_w(int r) { return ((r >> 1) & 1) | ((r / (4 * AT) & 3) << 1); }
__device__ __forceinline__ int swizzle_x(int r) { return (r >> 1) & 7; }

#ifndef SPREAD
#define SPREAD 4
#endif
#define SPREAD_AT(k) ((k) >= SPREAD ? L : (k) * L / SPREAD)
template <int T, int WM, int WN, int AT, int BT>
__global__ __launch_bounds__(WM * WN * 64) void k_product_tile(const ProductArgs a, int mtiles, int ttiles, int together) {
  constexpr int WAVES = WM * WN, TM = 16 * AT * WM, TN = 16 * BT * WN;
  constexpr int SCALES = T == P_F8 ? TN * 4 + 256 : 0, STAGE = (TM + TN) * 128 + SCALES;      // e4m3: the rows' scales, then the matrix's
  constexpr int LW = TM / 8 / WAVES, LX = TN / 8 / WAVES, L = LW + LX;        // 1 KB loads of a wave to a stage
  constexpr int RA = T == P_F8 ? 2 : 4;                          // tiles of the matrix in registers
  static_assert(T != P_F8 || TN / 64 < WAVES, "a wave for the matrix's scales");
  static_assert(TM % (8 * WAVES) == 0 && TN % (8 * WAVES) == 0 && AT % RA == 0, "whole loads, registers in turn");
  extern __shared__ __align__(16) uint8_t lds[];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
  const int wm = wv / WN, wn = wv % WN;
  // Workgroups go to the eight XCDs in turn: 32 neighbouring tiles to one XCD (a tile for each of its compute units, `together` tiles of x by a few of
  // the matrix, whose rows its L2 serves to several of them), the next 32 to the next.  Tiles without rows, which are the last, fall on all alike.
  const int id = ((blockIdx.x >> 8) << 8) + (blockIdx.x & 7) * 32 + ((blockIdx.x >> 3) & 31);
  if (id >= mtiles * ttiles) return;
  const int strip = id / (mtiles * together), t0 = strip * together, high = min(together, ttiles - t0);
  const int rest = id - strip * mtiles * together, mt = rest / high, tt = t0 + rest % high;
  const int m0 = mt * TM;
  const Span s = find_span(a, TN, tt);
  if (s.e < 0) return;
  if (s.e == a.experts) { zero_rows(a, s, m0, TM); return; }
  const size_t row_bytes = (size_t)a.n * bytes_of<T>;
  const int slabs = (int)((row_bytes + 127) >> 7);
  // what the lane loads: 32-bit distances from the tile's first row of either operand (from x where rows are gathered), so that a load takes one
  // register of address
  const HTR_GLOBAL uint8_t* wb = (const HTR_GLOBAL uint8_t*)a.w + ((size_t)s.e * a.m + m0) * row_bytes;
  const HTR_GLOBAL uint8_t* xb = (const HTR_GLOBAL uint8_t*)a.x + (a.gather != nullptr ? 0 : (size_t)s.first * row_bytes);
  uint32_t src[L];
  auto chunk_of = [&](int j) {
    const int r = ((j < LW ? j : j - LW) * WAVES + wv) * 8 + (lane >> 3);
    return (lane & 7) ^ (j < LW ? swizzle_w<AT>(r) : swizzle_x(r));
  };
#pragma unroll
  for (int j = 0; j < L; ++j) {
    int r = ((j < LW ? j : j - LW) * WAVES + wv) * 8 + (lane >> 3);
    if (j < LW) {
      r = min(r, a.m - 1 - m0);
    } else {
      r = min(r, s.count - 1);
      if (a.gather != nullptr) r = a.gather[s.first + r];
    }
    src[j] = (uint32_t)r * (uint32_t)row_bytes + 16 * chunk_of(j);
  }
  // 16-bit rows may end inside the last slab, at a multiple of 16 bytes: chunks from there on are loaded as the slab's first, and zeroed in LDS
  const int tail = (int)(row_bytes & 127) >> 4;
  auto place = [&](int j, int stage) { return stage * STAGE + (j < LW ? (j * WAVES + wv) * 1024 : TM * 128 + ((j - LW) * WAVES + wv) * 1024); };
  auto issue = [&](int slab, int stage, int from, int to) {      // behind the last slab it is loaded again, for nothing
    slab = min(slab, slabs - 1);
#pragma unroll
    for (int j = from; j < to; ++j) {
      asm volatile("" : "+v"(src[j]));                           // or the compiler keeps 64-bit addresses
      uint32_t off = src[j];
      if (T != P_F8 && tail != 0 && slab == slabs - 1) { const int ch = chunk_of(j); off -= ch >= tail ? 16 * ch : 0; }      // src holds 16 ch
      const HTR_GLOBAL uint8_t* p = (j < LW ? wb : xb) + ((size_t)slab << 7) + off;
      __builtin_amdgcn_global_load_lds((const HTR_GLOBAL void*)p, (__attribute__((address_space(3))) void*)(lds + place(j, stage)), 16, 0, 0);
    }
  };
  // where a lane reads its first chunk of each tile of either operand; the second lies at place ^ 4
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
  // A slab's scales come with it, through LDS: as loads into registers they would make the wave wait for all the loads issued after them.  Waves 0 .. TN / 64 - 1
  // take 64 rows' each, the others the matrix's (one for each 128 rows; all the same, since a branch here costs registers all over the loop).
  const HTR_GLOBAL float* sb = nullptr;
  uint32_t so = 0u;
  if constexpr (T == P_F8) {
    if (wv < TN / 64) {
      int r = min(wv * 64 + lane, s.count - 1);
      if (a.gather != nullptr) r = a.gather[s.first + r];
      sb = (const HTR_GLOBAL float*)a.xs + (a.gather != nullptr ? 0 : (size_t)s.first * (a.n >> 7));
      so = (uint32_t)r * (uint32_t)(a.n >> 7);
    } else {
      const int blocks = (a.m + 127) >> 7;
      sb = (const HTR_GLOBAL float*)a.ws + ((size_t)s.e * blocks + (m0 >> 7)) * (a.n >> 7);
      so = (uint32_t)min(lane, blocks - 1 - (m0 >> 7)) * (uint32_t)(a.n >> 7);
    }
  }
  auto issue_scales = [&](int slab, int stage) {
    if constexpr (T == P_F8)
      __builtin_amdgcn_global_load_lds((const HTR_GLOBAL void*)(sb + min(slab, slabs - 1) + so),
                                       (__attribute__((address_space(3))) void*)(lds + stage * STAGE + (TM + TN) * 128 + min(wv, TN / 64) * 256), 4, 0, 0);
  };
  f4 acc[AT][BT];
#pragma unroll
  for (int i = 0; i < AT; ++i)
#pragma unroll
    for (int t = 0; t < BT; ++t) acc[i][t] = f4{0.f, 0.f, 0.f, 0.f};
  issue_scales(0, 0);
  issue(0, 0, 0, L);
  issue_scales(1, 1);
  issue(1, 1, 0, SPREAD_AT(RA - 1));
  // the stage of `slab` is there for every wave; `behind`: loads of this wave that may still be on their way (they arrive in order)
  auto landed = [&](int slab, auto behind) {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(decltype(behind)::value) : "memory");
    if (T != P_F8 && tail != 0 && slab == slabs - 1) {
#pragma unroll
      for (int j = 0; j < L; ++j) if (chunk_of(j) >= tail) *(u4*)(lds + place(j, slab & 1) + 16 * lane) = u4{0u, 0u, 0u, 0u};
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  u4 A[RA][2], B[BT][2];
  float sx[BT], sw = 0.f;
  auto read_scales = [&](int slab) {
    const float* base = (const float*)(lds + (slab & 1) * STAGE + (TM + TN) * 128);
#pragma unroll
    for (int t = 0; t < BT; ++t) sx[t] = base[wn * 16 * BT + 16 * t + c];
    sw = base[TN + ((wm * 16 * AT) >> 7)];
  };
  auto read_a = [&](int i, int slab) {
    const uint8_t* base = lds + (slab & 1) * STAGE;
    A[i % RA][0] = *(const u4*)(base + ra[i]); A[i % RA][1] = *(const u4*)(base + (ra[i] ^ 64));
  };
  auto read_b = [&](int t, int slab) {
    const uint8_t* base = lds + (slab & 1) * STAGE;
    B[t][0] = *(const u4*)(base + rb[t]); B[t][1] = *(const u4*)(base + (rb[t] ^ 64));
  };
  // A slab's operands are in registers before its products begin: the barrier lies where every wave has read all of the slab before, RA - 1 tiles ahead
  // of its last product, so its stage can be loaded again at once, and the last tiles' products cover the first reads
  landed(0, std::integral_constant<int, SPREAD_AT(RA - 1)>());
#pragma unroll
  for (int i = 0; i < RA - 1; ++i) read_a(i, 0);
#pragma unroll
  for (int t = 0; t < BT; ++t) read_b(t, 0);
  if constexpr (T == P_F8) read_scales(0);
  for (int slab = 0; slab < slabs; ++slab) {
    float sc[BT];
    f4 part[3];
    if constexpr (T == P_F8) {
#pragma unroll
      for (int t = 0; t < BT; ++t) sc[t] = sx[t] * sw;
    }
#pragma unroll
    for (int i = 0; i < AT; ++i) {
      if (i == AT - RA + 1) {
        landed(slab + 1, std::integral_constant<int, 0>());
        issue_scales(slab + 2, slab & 1);
        if constexpr (T == P_F8) read_scales(slab + 1);
      }
      if (i >= AT - RA + 1) issue(slab + 2, slab & 1, SPREAD_AT(i - (AT - RA + 1)), SPREAD_AT(i - (AT - RA + 1) + 1));
      else issue(slab + 1, (slab + 1) & 1, SPREAD_AT(i + RA - 1), SPREAD_AT(i + RA));
      if (i + RA - 1 < AT) read_a(i + RA - 1, slab); else read_a(i + RA - 1 - AT, slab + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < BT; ++t) {
        if constexpr (T == P_F8) {
          // the sums two products behind the matrix unit
          const int k = i * BT + t, l = k - 2;
          part[k % 3] = mfma_f8(A[i % RA][0], A[i % RA][1], B[t][0], B[t][1]);
          if (l >= 0) acc[l / BT][l % BT] += part[l % 3] * sc[l % BT];
        } else {
          acc[i][t] = mfma_16<T>(A[i % RA][0], B[t][0], acc[i][t]);
          acc[i][t] = mfma_16<T>(A[i % RA][1], B[t][1], acc[i][t]);
        }
        if (i == AT - 1) read_b(t, slab + 1);
      }
      if constexpr (T == P_F8) {
        // a product, then the four sums of the one two before it: left to itself the compiler waits for results just asked for
#pragma unroll
        for (int t = 0; t < BT; ++t) { __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); __builtin_amdgcn_sched_group_barrier(0x002, 4, 0); }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (T == P_F8) {
#pragma unroll
      for (int l = AT * BT - 2; l < AT * BT; ++l) acc[l / BT][l % BT] += part[l % 3] * sc[l % BT];
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // the last loads again: they write to LDS
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
