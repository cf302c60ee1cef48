// Part of unpacked.hip, included inside its anonymous namespace: up to 32 rows of x times one matrix in int8.
//
//   y[t][i] = (sum_k qx[t][k] w[i][k]) sx[t] sw[i] (+ bias),   the rows in int8, or floating and rounded here as in int8.hpp
//
// Bound: HBM, the matrix read once.  Workgroups go on from tile to tile of 8 matrix rows, their loads STAGES ahead of the products, in registers and across the
// ends of tiles; rows of x stay in LDS.  Waves take a tile's steps of 256 bytes in turn and add up through LDS, some of them while the others go on.
// A v_mfma_i32_16x16x64_i8 multiplies 16 rows by 16 columns; here its rows are the two halves of 128 bytes of 8 matrix rows, its columns the same halves of 8 rows of x,
// and of the products those of equal halves count: half of the matrix unit's work is lost, of which there is plenty, but a load of a wave takes whole lines of memory,
// where 16 rows would take half of each of twice as many (8 rows on 152064x4096 101 us and 118; 28672x4096 by one row 20.2 and 25.1, by quarters of 256 bytes of 4 rows
// 21.4).
// Whatever is read behind a row's end meets zeros of x.
struct RowsArgs {
  const void* x;                        // [rows][n] of x_type, consecutive
  const float* xs;                      // int8: [rows]
  const uint8_t* w;                     // [m][n]
  const float* ws;                      // [m]
  const void* bias;                     // [m] of y_dtype or NULL
  void* y;                              // [rows][m]
  int rows, m, n, x_type, y_dtype;
};
constexpr int ROWS_WAVES = 8, ROWS_TILE = 8, ROWS_STEP = ROWS_WAVES * 256, ROWS_AHEAD = 32;
// bytes of a row of x in LDS: whole steps of all waves, and 16 that put neighbouring rows on different banks
inline __host__ __device__ int rows_pitch(int n) { return (n + ROWS_STEP - 1) / ROWS_STEP * ROWS_STEP + 16; }
// that, two tiles' partial sums, the rows' largest by wave, their scales, and two runs of ROWS_AHEAD tiles' scales and biases
inline size_t rows_lds(int rows, int columns, int n) {
  return (size_t)rows * rows_pitch(n) + (2 * ROWS_WAVES * ROWS_TILE * columns + ROWS_WAVES + 32 + 4 * ROWS_AHEAD * ROWS_TILE) * 4;
}

// CT: runs of 8 rows of x; floating ones, which are rounded here, come in one
template <int X, int CT>
__global__ __launch_bounds__(ROWS_WAVES * 64) void k_product_rows(const RowsArgs a, int tiles) {
  constexpr int TR = ROWS_TILE, PART = TR * 8 * CT, STAGES = 4;      // matrix rows of a tile, sums of a wave's, loads ahead (6 and 8: no faster)
  extern __shared__ __align__(16) uint8_t lds[];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
  const int n = a.n, rows = a.rows, pitch = rows_pitch(n), steps = (pitch - 16) / ROWS_STEP;
  uint8_t* xq = lds;
  int* red = (int*)(lds + rows * pitch);
  uint32_t* largest = (uint32_t*)(red + 2 * ROWS_WAVES * PART);               // by wave
  float* scale = (float*)(largest + ROWS_WAVES);
  float* ahead = scale + 32;                                                  // [2][scales, biases][ROWS_AHEAD][TR]

  // Loads: tile and step of the next one.  Lane c has row c / 2 of the tile; the lanes of a row cover 128 consecutive bytes of it with each of a step's two loads.
  // Behind the last step comes the matrix's first line, for nothing: a load that may not be there would make the others wait.
  int load_tile = blockIdx.x, load_step = 0;
  u4 A[STAGES][2];
  const HTR_GLOBAL uint8_t* base;
  uint32_t row_off, lane_off = (c & 1) * 64 + 16 * g;
  auto to_tile = [&](int tile) {
    if (tile < tiles) {
      const int m0 = tile * TR;
      base = (const HTR_GLOBAL uint8_t*)a.w + (size_t)m0 * n;
      row_off = (uint32_t)min(c >> 1, a.m - 1 - m0) * (uint32_t)n;
    } else {
      base = (const HTR_GLOBAL uint8_t*)a.w;
      row_off = lane_off = 0;
    }
  };
  auto load = [&](int p) {
    const uint32_t at = load_tile < tiles ? (uint32_t)(load_step * ROWS_WAVES + wv) * 256 : 0u;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      A[p][h] = __builtin_nontemporal_load((const HTR_GLOBAL u4*)(base + row_off + min(at + lane_off + (load_tile < tiles ? h * 128 : 0), (uint32_t)n - 16)));
    if (++load_step == steps) {
      load_step = 0;
      if (load_tile < tiles) { load_tile += gridDim.x; to_tile(load_tile); }
    }
  };
  to_tile(load_tile);
#pragma unroll
  for (int p = 0; p < STAGES; ++p) load(p);

  // x to LDS, zeros behind its rows.  A row to one, two, four or all eight waves, as many as there are for it; all loads of a run of LOADS are on their way at once.
  const int per_row = rows == 1 ? 8 : rows == 2 ? 4 : rows <= 4 ? 2 : 1, part = wv % per_row;
  constexpr int LOADS = 8, UNIT = X == P_I8 ? 16 : 8;
  const int step_x = UNIT * 64 * per_row, k0 = UNIT * (lane + 64 * part);
  // several waves to a row: one row for each of them, the last one again for those without, so that all come to the barrier
  for (int r = per_row > 1 ? min(wv / per_row, rows - 1) : wv; r < rows; r += ROWS_WAVES) {
    if constexpr (X == P_I8) {
      for (int k = k0; k < pitch; k += LOADS * step_x) {
        u4 v[LOADS];
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
          v[j] = k + j * step_x < n ? *(const HTR_GLOBAL u4*)((const HTR_GLOBAL uint8_t*)a.x + (size_t)r * n + k + j * step_x) : u4{0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < LOADS; ++j) if (k + j * step_x < pitch) *(u4*)(xq + r * pitch + k + j * step_x) = v[j];
      }
      if (lane == 0 && part == 0) scale[r] = ((const HTR_GLOBAL float*)a.xs)[r];
    } else {
      Eight<X> v[LOADS];
      auto load_run = [&](int k) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) if (k + j * step_x < n) v[j].load_any(a.x, (size_t)r * n + k + j * step_x);
      };
      uint32_t m = 0;
      for (int k = k0; k < n; k += LOADS * step_x) {
        load_run(k);
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
          if (k + j * step_x < n) {
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, magnitude(v[j].get(i)));
          }
      }
      m = wave_max(m);
      if (per_row > 1) {
        if (lane == 0) largest[wv] = m;
        __syncthreads();
        for (int w = 0; w < per_row; ++w) m = max(m, largest[wv - part + w]);
      }
      const RowScale s((double)__uint_as_float(m), 1.0);
      if (lane == 0 && part == 0) scale[r] = s.s;
      for (int k = k0; k < pitch; k += LOADS * step_x) {
        if (n > LOADS * step_x && k < n) load_run(k);
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
          if (k + j * step_x >= pitch) continue;
          u2 q = {0u, 0u};
          if (k + j * step_x < n) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = v[j].get(i);
            q = round8(s, f);
          }
          *(u2*)(xq + r * pitch + k + j * step_x) = q;
        }
      }
    }
  }
  __syncthreads();

  // a thread's output of a tile: row i of the matrix, row t of x
  const int i = threadIdx.x % TR, t = threadIdx.x / TR;
  const bool mine = t < rows;
  const float xs = mine ? scale[t] : 0.f;
  const uint8_t* xp[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) xp[t] = xq + min(8 * t + (c >> 1), rows - 1) * pitch + (c & 1) * 64 + 16 * g;
  auto type_of = [&](auto store) {
    if (a.y_dtype == HTR_BF16) store(std::integral_constant<int, HTR_BF16>());
    else if (a.y_dtype == HTR_F16) store(std::integral_constant<int, HTR_F16>());
    else store(std::integral_constant<int, HTR_F32>());
  };
  i4 acc[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) acc[t] = i4{0, 0, 0, 0};
  int step = 0, tile = blockIdx.x, half = 0;
  // Scales and biases of ROWS_AHEAD of the workgroup's tiles at once: as loads of every tile they would hold up the matrix's
  auto scales_from = [&](int tile, int which) {
    float* to = ahead + which * 2 * ROWS_AHEAD * TR;
    const int k = threadIdx.x / TR;
    const long long r = (tile + (long long)k * gridDim.x) * TR + i;
    if (k >= ROWS_AHEAD || r >= a.m) return;
    to[threadIdx.x] = ((const HTR_GLOBAL float*)a.ws)[r];
    if (a.bias != nullptr) to[ROWS_AHEAD * TR + threadIdx.x] = load_elem_g(a.bias, a.y_dtype, r);
  };
  int nth = 0;                                                                // of the workgroup's tiles
  while (tile < tiles) {
#pragma unroll
    for (int p = 0; p < STAGES; ++p) {
      if (tile >= tiles) break;
      if (step == 0 && nth % ROWS_AHEAD == 0) scales_from(tile, nth / ROWS_AHEAD & 1);
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        const uint8_t* xb = xp[t] + (step * ROWS_WAVES + wv) * 256;
        acc[t] = mfma_16<P_I8>(A[p][0], *(const u4*)xb, acc[t]);
        acc[t] = mfma_16<P_I8>(A[p][1], *(const u4*)(xb + 128), acc[t]);
      }
      load(p);
      if (++step < steps) continue;
      // D: rows 4 g + k, column c, that is halves k % 2 of the tile's rows 2 g + k / 2 by half c % 2 of row c / 2
      int* mine_red = red + (half * ROWS_WAVES + wv) * PART;
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        int v0 = c & 1 ? acc[t][1] : acc[t][0], v1 = c & 1 ? acc[t][3] : acc[t][2];
        v0 += __builtin_amdgcn_update_dpp(0, v0, 0xB1, 0xF, 0xF, false);
        v1 += __builtin_amdgcn_update_dpp(0, v1, 0xB1, 0xF, 0xF, false);
        mine_red[(8 * t + (c >> 1)) * TR + 2 * g + (c & 1)] = c & 1 ? v1 : v0;
      }
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");      // loads stay on their way
      if (mine) {
        int sum = 0;
#pragma unroll
        for (int w = 0; w < ROWS_WAVES; ++w) sum += red[(half * ROWS_WAVES + w) * PART + threadIdx.x];
        const int r = tile * TR + i;
        if (r < a.m) {
          const float* of_tile = ahead + ((nth / ROWS_AHEAD & 1) * 2 * ROWS_AHEAD + nth % ROWS_AHEAD) * TR + i;
          float v = (float)sum * xs * of_tile[0];
          if (a.bias != nullptr) v += of_tile[ROWS_AHEAD * TR];
          type_of([&](auto type) { store_elem_g(a.y, decltype(type)::value, (size_t)t * a.m + r, v); });
        }
      }
#pragma unroll
      for (int t = 0; t < CT; ++t) acc[t] = i4{0, 0, 0, 0};
      step = 0;
      half ^= 1;
      tile += gridDim.x;
      ++nth;
    }
  }
}
