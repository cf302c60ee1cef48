// Part of unpacked.hip, included inside its anonymous namespace: few rows of x times one matrix in int8, or each expert's few rows times its matrix.
//
//   y[t][i] = (sum_k qx[t][k] w_e[i][k]) sx[t] sw_e[i] (+ bias),   the rows in int8, or floating and rounded here as in int8.hpp
//
// Bound: HBM, the matrices read once.  A workgroup goes through a run of tiles, its loads STAGES ahead of the products, in registers and across the ends of tiles; the
// rows of x stay in LDS until the next expert's.  KW waves take steps of 256 bytes of 8 matrix rows in turn; a tile has 8 rows for each such team.  What the waves of a
// team have is added up through LDS, by some of them while the others go on.
// A v_mfma_i32_16x16x64_i8 multiplies 16 rows by 16 columns; here its rows are the two halves of 128 bytes of 8 matrix rows, its columns the same halves of 8 rows of x,
// and of the products those of equal halves count: half of the matrix unit's work is lost, of which there is plenty, but a load of a wave takes whole lines of memory,
// where 16 rows would take half of each of twice as many (8 rows on 152064x4096 101 us and 118; 28672x4096 by one row 20.2 and 25.1, by quarters of 256 bytes of 4 rows
// 21.4).
// Whatever is read behind a row's end meets zeros of x.
constexpr int ROWS_WAVES = 8, ROWS_AHEAD = 256, ROWS_SPANS = 64;
inline __host__ __device__ int rows_tile(int kw) { return 8 * (ROWS_WAVES / kw); }
// bytes of a row of x in LDS: whole steps of a team, and 16 that put neighbouring rows on different banks
inline __host__ __device__ int rows_pitch(int n, int kw) { return (n + kw * 256 - 1) / (kw * 256) * (kw * 256) + 16; }
// that, two tiles' partial sums, the rows' largest by wave, their scales, two runs of ROWS_AHEAD matrix rows' scales and biases, and the spans of a workgroup's run
inline size_t rows_lds(int rows, int columns, int n, int kw, bool grouped) {
  return (size_t)rows * rows_pitch(n, kw) + (2 * ROWS_WAVES * 8 * columns + ROWS_WAVES + 32 + 4 * ROWS_AHEAD + (grouped ? 4 * ROWS_SPANS : 0)) * 4;
}

// CT: runs of 8 rows of x to a span; floating ones, which are rounded here, come in one.  mtiles: tiles of a matrix; most: rows of a span that LDS has place for
template <int X, int CT, int KW, bool GROUPED>
__global__ __launch_bounds__(ROWS_WAVES * 64) void k_product_rows(const ProductArgs a, int mtiles, int most) {
  constexpr int TEAMS = ROWS_WAVES / KW, TR = 8 * TEAMS, PART = 64 * CT, STAGES = 4;      // matrix rows of a tile, sums of a wave, loads ahead (6 and 8: no faster)
  extern __shared__ __align__(16) uint8_t lds[];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
  const int n = a.n, pitch = rows_pitch(n, KW), steps = (pitch - 16) / (KW * 256);
  const int team = wv / KW, kw = wv % KW;
  uint8_t* xq = lds;
  int* red = (int*)(lds + most * pitch);
  uint32_t* largest = (uint32_t*)(red + 2 * ROWS_WAVES * PART);               // by wave
  float* scale = (float*)(largest + ROWS_WAVES);
  float* ahead = scale + 32;                                                  // [2][scales, biases][ROWS_AHEAD]
  int4* spans = (int4*)(ahead + 4 * ROWS_AHEAD);                         // {expert, first row, rows}

  // The workgroup's tiles, span by span, a matrix's from first to last: `left` of them from tile mt0 of its first span on
  const long long total = (long long)mtiles * (GROUPED ? count_spans(a, 8 * CT) : 1);
  // two workgroups of a compute unit (they come 256 apart) take neighbouring runs, so that a tile more or less evens out between them
  const int nth = gridDim.x == 512 ? (int)(blockIdx.x & 255) * 2 + (int)(blockIdx.x >> 8) : (int)blockIdx.x;
  const long long from = nth * total / gridDim.x, to = (nth + 1ll) * total / gridDim.x;
  if (from == to) return;
  const int span0 = GROUPED ? (int)(from / mtiles) : 0, mt0 = (int)(from - (long long)span0 * mtiles);
  int left = (int)(to - from);
  if constexpr (GROUPED) {
    const int last = (int)((to - 1) / mtiles);                                // at most ROWS_SPANS - 1 behind the first
    for (int k = wv; k <= last - span0; k += ROWS_WAVES) {
      const Span s = find_span(a, 8 * CT, span0 + k);
      if (lane == 0) spans[k] = int4{s.e, s.first, s.count, 0};
    }
    __syncthreads();
  }
  auto span_of = [&](int k) {
    if constexpr (!GROUPED) return Span{0, 0, a.rows};
    const int4 s = spans[k];
    return Span{__builtin_amdgcn_readfirstlane(s.x), __builtin_amdgcn_readfirstlane(s.y), __builtin_amdgcn_readfirstlane(s.z)};
  };

  // Loads: tile and step of the next one.  Lane c has row c / 2 of the tile; the lanes of a row cover 128 consecutive bytes of it with each of a step's two loads.
  // Behind the last step, and for rows without an expert, comes the first matrix's first line, for nothing: a load that may not be there would make the others wait.
  int load_left = left, load_mt = mt0, load_span = 0, load_step = 0;
  u4 A[STAGES][2];
  const HTR_GLOBAL uint8_t *base, *matrix;
  uint32_t row_off, lane_off;
  bool idle;
  auto to_matrix = [&] {
    const int e = span_of(load_span).e;
    idle = e == a.experts;
    matrix = (const HTR_GLOBAL uint8_t*)a.w + (size_t)(idle ? 0 : e) * a.m * n;
  };
  auto to_tile = [&] {
    const int m0 = min(load_mt * TR + 8 * team, a.m - 1);
    base = matrix + (idle ? (size_t)0 : (size_t)m0 * n);
    row_off = idle ? 0u : (uint32_t)min(c >> 1, a.m - 1 - m0) * (uint32_t)n;
    lane_off = idle ? 0u : (c & 1) * 64 + 16 * g;
  };
  auto load = [&](int p) {
    const uint32_t at = idle ? 0u : (uint32_t)(load_step * KW + kw) * 256;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      A[p][h] = __builtin_nontemporal_load((const HTR_GLOBAL u4*)(base + row_off + min(at + lane_off + (idle ? 0 : h * 128), (uint32_t)n - 16)));
    if (++load_step == steps) {
      load_step = 0;
      if (--load_left == 0) {
        idle = true;
        matrix = (const HTR_GLOBAL uint8_t*)a.w;
      } else if (load_left > 0 && ++load_mt == mtiles) {
        load_mt = 0;
        ++load_span;
        to_matrix();
      }
      to_tile();
    }
  };
  // A span's rows of x to LDS, zeros behind them.  A row to one, two, four or all eight waves, as many as there are for it; all loads of a run of LOADS are on their way at
  // once, and a wave's first ones ahead of the matrix's, which it would wait for otherwise.  Several waves to a row: one row for each of them, the last one again for those
  // without, so that all come to the barrier.
  constexpr int LOADS = X == P_I8 ? 4 : 8, UNIT = X == P_I8 ? 16 : 8;
  u4 q8[LOADS];
  Eight<X == P_I8 ? HTR_BF16 : X> v[LOADS];
  auto waves_of = [](int rows) { return rows == 1 ? 8 : rows == 2 ? 4 : rows <= 4 ? 2 : 1; };
  auto first_of = [&](int rows) { const int w = waves_of(rows); return w > 1 ? min(wv / w, rows - 1) : wv; };
  auto row_of = [&](const Span& s, int r) { return (size_t)(a.gather != nullptr ? a.gather[s.first + r] : s.first + r); };
  auto load_run = [&](size_t row, int k, int step) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      if constexpr (X == P_I8) q8[j] = k + j * step < n ? *(const HTR_GLOBAL u4*)((const HTR_GLOBAL uint8_t*)a.x + row * n + k + j * step) : u4{0u, 0u, 0u, 0u};
      else if (k + j * step < n) v[j].load_any(a.x, row * n + k + j * step);
    }
  };
  auto row_to_lds = [&](const Span& s, int r, bool loaded) {
    const int waves = waves_of(s.count), part = wv % waves, step = UNIT * 64 * waves, k0 = UNIT * (lane + 64 * part);
    const size_t row = row_of(s, r);
    if (!loaded) load_run(row, k0, step);
    if constexpr (X == P_I8) {
      if (lane == 0 && part == 0) scale[r] = ((const HTR_GLOBAL float*)a.xs)[row];
      for (int k = k0; k < pitch; k += LOADS * step) {
        if (k != k0) load_run(row, k, step);
#pragma unroll
        for (int j = 0; j < LOADS; ++j) if (k + j * step < pitch) *(u4*)(xq + r * pitch + k + j * step) = q8[j];
      }
    } else {
      uint32_t m = 0;
      for (int k = k0; k < n; k += LOADS * step) {
        if (k != k0) load_run(row, k, step);
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
          if (k + j * step < n) {
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, magnitude(v[j].get(i)));
          }
      }
      m = wave_max(m);
      if (waves > 1) {
        if (lane == 0) largest[wv] = m;
        __syncthreads();
        for (int w = 0; w < waves; ++w) m = max(m, largest[wv - part + w]);
      }
      const RowScale of_row((double)__uint_as_float(m), 1.0);
      if (lane == 0 && part == 0) scale[r] = of_row.s;
      for (int k = k0; k < pitch; k += LOADS * step) {
        if (n > LOADS * step && k < n) load_run(row, k, step);
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
          if (k + j * step >= pitch) continue;
          u2 q = {0u, 0u};
          if (k + j * step < n) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = v[j].get(i);
            q = round8(of_row, f);
          }
          *(u2*)(xq + r * pitch + k + j * step) = q;
        }
      }
    }
  };
  Span s = span_of(0);
  if (s.e < a.experts) load_run(row_of(s, min(first_of(s.count), s.count - 1)), UNIT * (lane + 64 * (wv % waves_of(s.count))), UNIT * 64 * waves_of(s.count));
  to_matrix();
  to_tile();
#pragma unroll
  for (int p = 0; p < STAGES; ++p) load(p);

  // a thread's outputs of a tile: row i of the matrix, rows t, t + ROWS of x
  constexpr int ROWS = ROWS_WAVES * 64 / TR, OUT = (8 * CT + ROWS - 1) / ROWS;
  const int i = threadIdx.x % TR, t0 = threadIdx.x / TR;
  const uint8_t* xp[CT];
  float xs[OUT];
  auto span_there = [&] {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < OUT; ++k) xs[k] = t0 + k * ROWS < s.count && s.e < a.experts ? scale[t0 + k * ROWS] : 0.f;
#pragma unroll
    for (int t = 0; t < CT; ++t) xp[t] = xq + min(8 * t + (c >> 1), s.count - 1) * pitch + (c & 1) * 64 + 16 * g;
  };
  auto to_span = [&](int k) {
    s = span_of(k);
    if (s.e < a.experts)
      for (int r = first_of(s.count); r < s.count; r += ROWS_WAVES) row_to_lds(s, r, false);
    span_there();
  };
  if (s.e < a.experts) {
    const int r0 = first_of(s.count);
    if (r0 < s.count) row_to_lds(s, r0, true);
    for (int r = r0 + ROWS_WAVES; r < s.count; r += ROWS_WAVES) row_to_lds(s, r, false);
  }
  span_there();
  int span = 0, mt = mt0;
  auto type_of = [&](auto store) {
    if (a.y_dtype == HTR_BF16) store(std::integral_constant<int, HTR_BF16>());
    else if (a.y_dtype == HTR_F16) store(std::integral_constant<int, HTR_F16>());
    else store(std::integral_constant<int, HTR_F32>());
  };
  i4 acc[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) acc[t] = i4{0, 0, 0, 0};
  int step = 0, half = 0;
  // Scales and biases of ROWS_AHEAD of the matrix's rows at once: as loads of every tile they would hold up the matrix's
  int done = 0, which = 1;                                                    // of the tiles since the last of these, and where they lie
  auto scales_from = [&] {
    which ^= 1;
    done = 0;
    float* to = ahead + which * 2 * ROWS_AHEAD;
    const int r = mt * TR + threadIdx.x;
    if (threadIdx.x >= ROWS_AHEAD || r >= a.m || s.e == a.experts) return;
    to[threadIdx.x] = ((const HTR_GLOBAL float*)a.ws)[(size_t)s.e * a.m + r];
    if (a.bias != nullptr) to[ROWS_AHEAD + threadIdx.x] = load_elem_g(a.bias, a.y_dtype, r);
  };
  scales_from();
  while (left > 0) {
#pragma unroll
    for (int p = 0; p < STAGES; ++p) {
      if (left == 0) break;
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        const uint8_t* xb = xp[t] + (step * KW + kw) * 256;
        acc[t] = mfma_16<P_I8>(A[p][0], *(const u4*)xb, acc[t]);
        acc[t] = mfma_16<P_I8>(A[p][1], *(const u4*)(xb + 128), acc[t]);
      }
      load(p);
      if (++step < steps) continue;
      // D: rows 4 g + k, column c, that is halves k % 2 of the team's rows 2 g + k / 2 by half c % 2 of row c / 2
      int* mine_red = red + (half * ROWS_WAVES + wv) * PART;
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        int v0 = c & 1 ? acc[t][1] : acc[t][0], v1 = c & 1 ? acc[t][3] : acc[t][2];
        v0 += __builtin_amdgcn_update_dpp(0, v0, 0xB1, 0xF, 0xF, false);
        v1 += __builtin_amdgcn_update_dpp(0, v1, 0xB1, 0xF, 0xF, false);
        mine_red[(8 * t + (c >> 1)) * 8 + 2 * g + (c & 1)] = c & 1 ? v1 : v0;
      }
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");      // loads stay on their way
      const int r = mt * TR + i;
#pragma unroll
      for (int k = 0; k < OUT; ++k) {
        const int t = t0 + k * ROWS;
        if (t >= s.count || r >= a.m) continue;
        const int* parts = red + (half * ROWS_WAVES + (i >> 3) * KW) * PART + t * 8 + (i & 7);
        int sum = 0;
#pragma unroll
        for (int w = 0; w < KW; ++w) sum += parts[w * PART];
        const float* of_row = ahead + which * 2 * ROWS_AHEAD + done * TR + i;
        float v = (float)sum * xs[k] * of_row[0];
        if (a.bias != nullptr) v += of_row[ROWS_AHEAD];
        if (GROUPED && s.e == a.experts) v = 0.f;                             // rows behind the last expert's
        type_of([&](auto type) { store_elem_g(a.y, decltype(type)::value, (size_t)(s.first + t) * a.m + r, v); });
      }
#pragma unroll
      for (int t = 0; t < CT; ++t) acc[t] = i4{0, 0, 0, 0};
      step = 0;
      half ^= 1;
      --left;
      ++done;
      if (++mt == mtiles) {
        mt = 0;
        if (GROUPED && left > 0) to_span(++span);                             // every wave is past the products of the one before
        done = ROWS_AHEAD / TR;
      }
      if (done == ROWS_AHEAD / TR && left > 0) scales_from();
    }
  }
}
