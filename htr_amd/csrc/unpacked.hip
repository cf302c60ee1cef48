// Kernels for MI355X (gfx950) around the packed linears, behind the same C ABI: the norm in front of them, and products with matrices that a
// checkpoint keeps in 16 bits, in e4m3 with block scales or in int8 with a scale for each channel, whole or by expert, and the router of experts.  Own translation unit: the packed kernels take two minutes to
// compile, these a few seconds.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>
#include <stdlib.h>
#include <math.h>
#include <atomic>
#include <type_traits>

#include "../../include/htr_gfx950.h"

// keeps the runtime's error for htr_last_hip_error (htr_gfx950.hip)
extern "C" __attribute__((visibility("hidden"))) int htr_note_hip_error(int e);

namespace {
#include "decode.hpp"
#include "norm.hpp"
#include "product.hpp"
#include "experts.hpp"
#include "int8.hpp"
#include "int8_rows.hpp"
#include "route.hpp"

#define TRY_HIP(EXPR) do { const hipError_t e_ = (EXPR); if (e_ != hipSuccess) return htr_note_hip_error((int)e_); } while (0)

// one launch with the runtime's own return value, as in plan.hpp
template <typename T> struct same { typedef T type; };
template <typename... K>
hipError_t launch(void (*kernel)(K...), dim3 grid, unsigned threads, size_t lds, hipStream_t st, typename same<K>::type... args) {
  void* argv[] = {(void*)&args...};
  return hipLaunchKernel((const void*)kernel, grid, dim3(threads), argv, lds, st);
}
// more dynamic LDS than the default 64 KB, once per device and kernel
template <auto Kernel> hipError_t allow_lds(size_t bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_acquire) & bit) return hipSuccess;
  e = hipFuncSetAttribute((const void*)Kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == hipSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

bool is_16bit(int dtype) { return dtype == HTR_BF16 || dtype == HTR_F16; }
bool is_dtype(int dtype) { return is_16bit(dtype) || dtype == HTR_F32; }
bool is_8bit(int type) { return type == HTR_E4M3 || type == HTR_I8; }
size_t element_bytes(int dtype) { return dtype == HTR_F32 ? 4 : is_8bit(dtype) ? 1 : 2; }
bool aligned(const void* p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

// ---- norm
template <int T, bool RES, bool QUANT, bool ANY>
hipError_t launch_norm(const NormArgs& a, hipStream_t st) {
  const int eights = (a.n + 7) / 8;
  const dim3 grid((unsigned)a.rows);
  // A row's loads are all in flight at once.  Few rows: one run of eight columns to a thread where that is a workgroup, two or four beyond (1 row of 4096 in
  // bf16 3.3 us, by two runs 4.0, by four 4.5).  Many: more runs, so that more workgroups share a compute unit and one's arithmetic hides behind the
  // others' loads (8192 rows of 4096 in bf16 to e4m3 29.4, 24.1 and 23.8 us; 13665 of 12800 by two and four 153 and 126); float32 rows have enough bytes to
  // load, and gain only where they go to e4m3 (8192 x 4096 35.8 and 33.3; with a residual 82.2 and 83.8).
  const bool many = a.rows >= 2048 && eights > 64;
  const int nv = eights <= 1024 ? (many && (T != HTR_F32 || (QUANT && !RES)) ? 2 : 1) : eights > 2048 || (many && (T != HTR_F32 || QUANT)) ? 4 : 2;
  const unsigned threads = ((eights + nv - 1) / nv + 63) / 64 * 64;
  switch (nv) {
    case 1: return launch(k_rms_norm<T, 1, RES, QUANT, ANY>, grid, threads, 0, st, a);
    case 2: return launch(k_rms_norm<T, 2, RES, QUANT, ANY>, grid, threads, 0, st, a);
    default: return launch(k_rms_norm<T, 4, RES, QUANT, ANY>, grid, threads, 0, st, a);
  }
}
template <int T, bool ANY> hipError_t launch_norm(const NormArgs& a, hipStream_t st) {
  const bool quant = a.scales != nullptr;
  if (a.residual) return quant ? launch_norm<T, true, true, ANY>(a, st) : launch_norm<T, true, false, ANY>(a, st);
  return quant ? launch_norm<T, false, true, ANY>(a, st) : launch_norm<T, false, false, ANY>(a, st);
}
template <int T> hipError_t launch_norm(const NormArgs& a, hipStream_t st) {
  if (a.n > 32768) {
    const dim3 grid((unsigned)a.rows);
    if (a.residual) return a.scales ? launch(k_rms_norm_long<T, true, true>, grid, 1024, 0, st, a) : launch(k_rms_norm_long<T, true, false>, grid, 1024, 0, st, a);
    return a.scales ? launch(k_rms_norm_long<T, false, true>, grid, 1024, 0, st, a) : launch(k_rms_norm_long<T, false, false>, grid, 1024, 0, st, a);
  }
  const bool vector = a.n % 8 == 0 && aligned(a.x, 16) && aligned(a.residual, 16) && aligned(a.weight, 16) && aligned(a.y, 16) && aligned(a.sum, 16) &&
                      a.x_stride % 8 == 0 && a.residual_stride % 8 == 0;
  return vector ? launch_norm<T, false>(a, st) : launch_norm<T, true>(a, st);
}

hipError_t launch_quantize(const void* x, int dtype, long long rows, int n, long long stride, void* q, float* scales, hipStream_t st) {
  const int per_row = n / 128;
  const long long blocks = rows * per_row;
  const dim3 grid((unsigned)((blocks + 15) / 16));
  if (dtype == HTR_BF16) return launch(k_quantize<HTR_BF16>, grid, 256, 0, st, x, stride, blocks, per_row, (uint8_t*)q, scales);
  if (dtype == HTR_F16) return launch(k_quantize<HTR_F16>, grid, 256, 0, st, x, stride, blocks, per_row, (uint8_t*)q, scales);
  return launch(k_quantize<HTR_F32>, grid, 256, 0, st, x, stride, blocks, per_row, (uint8_t*)q, scales);
}

// ---- rows to int8: one workgroup to a row, one, two or four runs of eight columns to a thread
template <typename F> hipError_t by_runs(int n, F take) {
  const int eights = n / 8, nv = eights <= 1024 ? 1 : eights <= 2048 ? 2 : 4;
  if (n > I8_MOST) return take(std::integral_constant<int, 0>(), 1024u);
  const unsigned threads = ((eights + nv - 1) / nv + 63) / 64 * 64;
  return nv == 1 ? take(std::integral_constant<int, 1>(), threads) : nv == 2 ? take(std::integral_constant<int, 2>(), threads) : take(std::integral_constant<int, 4>(), threads);
}
template <int T, bool G> hipError_t launch_round(const void* x, long long stride, long long rows, int n, const int* last, void* q, void* scales, hipStream_t st) {
  constexpr long long MOST = 1 << 21;      // a launch has fewer than 2^32 threads, up to 1024 of them to a row
  return by_runs(n, [&](auto nv, unsigned threads) {
    hipError_t e = hipSuccess;
    for (long long r = 0; r < rows && e == hipSuccess; r += MOST)
      e = launch(k_round_rows<T, decltype(nv)::value, G>, dim3((unsigned)(rows - r < MOST ? rows - r : MOST)), threads, 0, st, x, stride, r, n, last, (uint8_t*)q, (float*)scales);
    return e;
  });
}
hipError_t launch_round(const void* x, int dtype, long long stride, long long rows, int n, void* q, void* scales, hipStream_t st) {
  return dtype == HTR_BF16 ? launch_round<HTR_BF16, false>(x, stride, rows, n, nullptr, q, scales, st)
         : dtype == HTR_F16 ? launch_round<HTR_F16, false>(x, stride, rows, n, nullptr, q, scales, st)
                            : launch_round<HTR_F32, false>(x, stride, rows, n, nullptr, q, scales, st);
}
template <int T> hipError_t launch_norm_int8(const NormArgs& a, hipStream_t st) {
  return by_runs(a.n, [&](auto nv, unsigned threads) {
    return launch(a.residual ? k_rms_norm_int8<T, decltype(nv)::value, true> : k_rms_norm_int8<T, decltype(nv)::value, false>, dim3((unsigned)a.rows), threads, 0, st, a);
  });
}

// ---- products
// The kernels by their template arguments, for who launches them and for who asks which one is launched
template <int R_, int TT_, int WAVES_> struct Stream { static constexpr int R = R_, TT = TT_, WAVES = WAVES_; };
template <int WM_, int WN_, int AT_, int BT_, int NS_, bool GATED_ = false> struct Tiles {
  static constexpr int WM = WM_, WN = WN_, AT = AT_, BT = BT_, NS = NS_, TM = 16 * AT_ * WM_, TN = 16 * BT_ * WN_;
  static constexpr bool GATED = GATED_;
  template <int T> static constexpr size_t LDS = NS * ((TM + TN) * 128 + (T == P_F8 ? (TN + 63) / 64 * 256 + 256 : 0)) + (GATED && T == P_F8 ? WM * TN * 4 : 0) + (T == P_I8 ? 2 * 4 * scales_of_tile(TM, TN) : 0);
};
struct TileGrid { long long mtiles, tiles; unsigned workgroups; };      // tiles: a bound where rows are grouped
template <int T, typename K> TileGrid tile_grid(const ProductArgs& a) {
  constexpr size_t LDS = K::template LDS<T>;
  static_assert(LDS <= 160 * 1024, "a compute unit's LDS");
  TileGrid g;
  g.mtiles = (a.m + K::TM - 1) / K::TM;
  g.tiles = g.mtiles * span_bound(a.rows, a.experts, a.ends != nullptr, K::TN);
  // as many workgroups as run at once (an MI355X has 256 compute units), a multiple of the XCDs; rows of fewer slabs than stages have no stream to run on from
  // tile to tile
  const bool stream = (long long)a.n * bytes_of<T> > 128 * (K::NS - 1);
  const long long wgs = 256 * (160 * 1024 / LDS), up = (g.tiles + TILE_XCDS - 1) / TILE_XCDS * TILE_XCDS;
  g.workgroups = (unsigned)(stream && wgs < up ? wgs : up);
  return g;
}
template <int T, int R, int TT, int WAVES> hipError_t launch_kernel(Stream<R, TT, WAVES>, const ProductArgs& a, hipStream_t st) {
  const dim3 grid((a.m + 16 * R - 1) / (16 * R), (unsigned)span_bound(a.rows, a.experts, a.ends != nullptr, 16 * TT));
  if constexpr (T == P_F8 && TT == 1) {
    if (a.wide) return launch(a.x_type == HTR_BF16 ? k_product_stream<T, HTR_BF16, R, TT, WAVES, true, false> : k_product_stream<T, HTR_F16, R, TT, WAVES, true, false>, grid, WAVES * 64, 0, st, a);
    if (a.x_type == HTR_BF16) return launch(k_product_stream<T, HTR_BF16, R, TT, WAVES, false, false>, grid, WAVES * 64, 0, st, a);
    if (a.x_type == HTR_F16) return launch(k_product_stream<T, HTR_F16, R, TT, WAVES, false, false>, grid, WAVES * 64, 0, st, a);
  }
  if constexpr (T != P_F8) {
    if ((size_t)a.n * bytes_of<T> % 128 != 0) return launch(k_product_stream<T, T, R, TT, WAVES, false, true>, grid, WAVES * 64, 0, st, a);
  }
  return launch(k_product_stream<T, T, R, TT, WAVES, false, false>, grid, WAVES * 64, 0, st, a);
}
template <int T, int WM, int WN, int AT, int BT, int NS, bool GATED> hipError_t launch_kernel(Tiles<WM, WN, AT, BT, NS, GATED> k, const ProductArgs& a, hipStream_t st) {
  constexpr size_t LDS = decltype(k)::template LDS<T>;
  const TileGrid g = tile_grid<T, decltype(k)>(a);
  const hipError_t e = allow_lds<k_product_tile<T, WM, WN, AT, BT, NS, GATED>>(LDS);
  if (e != hipSuccess) return e;
  return launch(k_product_tile<T, WM, WN, AT, BT, NS, GATED>, dim3(g.workgroups), WM * WN * 64, LDS, st, a, (int)g.mtiles);
}
// what htr_product_plan says of a kernel: matrix rows and rows of x to a tile, waves and ring stages (0: no ring), workgroups, tiles
template <int T, int R, int TT, int WAVES> void describe_kernel(Stream<R, TT, WAVES>, const ProductArgs& a, int* out) {
  const long long tiles = (a.m + 16 * R - 1) / (16 * R) * span_bound(a.rows, a.experts, a.ends != nullptr, 16 * TT);
  const int v[6] = {16 * R, 16 * TT, WAVES, 0, (int)tiles, (int)tiles};
  memcpy(out, v, sizeof(v));
}
template <int T, int WM, int WN, int AT, int BT, int NS, bool GATED> void describe_kernel(Tiles<WM, WN, AT, BT, NS, GATED> k, const ProductArgs& a, int* out) {
  const TileGrid g = tile_grid<T, decltype(k)>(a);
  const int v[6] = {k.TM, k.TN, WM * WN, NS, (int)g.workgroups, (int)g.tiles};
  memcpy(out, v, sizeof(v));
}
// Which tiles for many rows: the ones whose rounds take the least time by what a slab of a tile takes (ns) with a tile to a few compute units, and with all
// at work, as many to each as fit.  Measured on 48 .. 8192 rows of 4096 .. 8192 columns, matrices from HBM.  A larger tile multiplies more for what it loads, a
// smaller one leaves fewer compute units idle: 256 rows on 4096x8192 in e4m3 99 us by 256x256, 50 by 128x128, 40 by 128x64, 29 by 64x64, 35 by 64x32; 512 rows
// 97, 50, 41, 47, 61; 4096 rows 126, 183, 200, 283, 385.
struct TileChoice { int tm, tn, at_once; float light, full; };
constexpr TileChoice TILES_8[] = {{256, 256, 1, 1440.f, 1900.f}, {256, 128, 1, 1050.f, 1100.f}, {128, 128, 1, 710.f, 760.f},
                                  {128, 64, 2, 570.f, 870.f},    {64, 64, 2, 395.f, 685.f},     {64, 32, 3, 285.f, 695.f}};
constexpr TileChoice TILES_16[] = {{256, 256, 1, 1380.f, 1700.f}, {256, 128, 1, 810.f, 1000.f}, {128, 128, 1, 580.f, 640.f},
                                   {128, 64, 2, 480.f, 735.f},    {64, 64, 2, 315.f, 510.f},    {64, 32, 3, 290.f, 450.f}};
// gate and up in one: 128 hidden columns to a tile.  Fitted to whole layers of 32 .. 4096 tokens, matrices from HBM, in 16 bits and e4m3: 8 experts (top 2) of 4096/2048,
// 64 (6) of 2048/1408, 16 (4) of 1024/512, 32 (4) and 128 (8) of 2048/768.  The way taken is within 5 % of the fastest in these 54, within 17 % on sizes apart from
// them (us by 256x256, x128, x64, x32: 1500 tokens of 64 experts in e4m3 263, 222, 289, 312, in 16 bits 403, 351, 374, 439; 256 tokens of 8 in 16 bits 161, 131,
// 128, 149; 1500 tokens of 32 in e4m3 95, 100, 123, 130).
constexpr TileChoice GATED_TILES[] = {{256, 256, 1, 1450.f, 2250.f}, {256, 128, 1, 950.f, 1250.f}, {256, 64, 1, 750.f, 950.f}, {256, 32, 1, 600.f, 700.f}};
template <int N> int best_tile(const TileChoice (&choices)[N], const ProductArgs& a, size_t row_bytes) {
  int best = 0;
  float least = 0.f;
  for (int k = 0; k < N; ++k) {
    const TileChoice& c = choices[k];
    const float mtiles = (float)((a.m + c.tm - 1) / c.tm), full = (float)a.rows / c.tn;
    const float experts = (float)(a.rows < a.experts ? a.rows : a.experts);
    // an expert's last tile is half full on average
    const float tiles = mtiles * (a.experts == 1 ? ceilf(full) : fmaxf(experts, full + 0.5f * experts));
    const float whole = floorf(tiles / (256.f * c.at_once)), rest = tiles - whole * 256.f * c.at_once;
    // the last round: the share of compute units at work, or where several tiles fit, tiles to one beyond the first; with half of them at one more, all wait
    const float beyond = fmaxf(rest / 256.f - 1.f, 0.f), some = beyond - floorf(beyond);
    const float share = c.at_once == 1 ? rest / 256.f : (floorf(beyond) + (some > 0.f ? fminf(1.f, (1.f + 4.f * some) / 3.f) : 0.f)) / (c.at_once - 1.f);
    const float ns = 4000.f + (float)((row_bytes + 127) >> 7) * (whole * c.full + (rest > 0.f ? c.light + share * (c.full - c.light) : 0.f));
    if (k == 0 || ns < least) { least = ns; best = k; }
  }
  return best;
}
// Few rows of a matrix are a matter of reading it.  k_product_stream has the most loads on their way where a matrix's rows alone make enough workgroups;
// k_product_tile goes on from tile to tile without a pause where there is more (e4m3, us):
//   one row: 1024x4096 5.0 (16 rows to a workgroup of 8 waves; 4 waves 6.4, tiles of 64x32 10.9), 4096x4096 5.9 (7.4, 12.0), 14336x4096 15.5 (17.2, 16.9),
//   28672x4096 25.7 (27.2, 29.5); 32 rows: 4096x4096 10.3 (tiles of 64x32 12.4, of 128x32 16.6), 28672x4096 64 (33, 31)
//   96 rows of 64 experts: 2816x2048 56 (64 rows to a workgroup of 4 waves; 16 rows to one of 8 86; tiles of 128x32 59), 2048x1408 34 (52; 35)
//   9 rows of 16 experts of 523x7600 in bf16: 28 us (64 rows to a workgroup of 4 waves 54, tiles of 64x32 37)
bool takes_16bit_rows(long long rows, int experts, bool grouped) {
  return grouped ? rows <= 4ll * experts && span_bound(rows, experts, true, 16) <= 65535 : rows <= 16;
}
// The kernel for a product, handed to `take`
template <int T, typename F> auto product_kernel(const ProductArgs& a, F take) {
  const int mean = (int)((a.rows + (long long)a.experts - 1) / a.experts);
  const bool grouped = a.ends != nullptr, few = takes_16bit_rows(a.rows, a.experts, grouped);
  if (few) {
    const long long tiles = grouped ? (a.rows < a.experts ? a.rows : a.experts) : 1, wgs = (a.m + 15) / 16 * tiles;
    const long long slabs = ((long long)a.n * bytes_of<T> + 127) / 128;
    // In 16 bits a ring is ahead where there are that many (92 sizes of 4 to 160 experts, up to 4 rows to one: 0.81 to 0.87 of the time on average, 1.03 at worst; us by
    // 64 rows to a workgroup of 4 waves, by tiles of 64x64: 96 rows of 64 experts of 2816x2048 146 and 127, 12 of 8 of 14336x4096 242 and 178, 72 of 48 of
    // 1536x2560 85 and 63, 48 of 24 of 3000x3000 122 and 80, 160 of 160 of 1024x1024 51 and 48).  Rows that all have one expert take less either way (256 rows of
    // 64 experts of 2816x2048 in e4m3 22 us, evenly 69).
    if (grouped && wgs >= 4 * 512) {
      if constexpr (T == P_F8 || T == P_I8) return take(Stream<4, 1, 4>{});
      return take(Tiles<2, 2, 2, 2, 4>{});
    }
    // Rows of fewer slabs than waves leave some idle (7 rows on 15657x384 in e4m3 5.5 us by 16 rows to a workgroup of 8 waves, 4.7 by 32 to one of 4), and rows
    // to be rounded are rounded by half as many (4 tokens over 8 of 16 experts of 1920/384 37 and 31); long rows of few workgroups need more waves to share them.
    // In int8 what comes here has rows too long for k_product_rows.
    if (T != P_I8 && wgs >= 512 && (slabs < 8 || (slabs <= 16 && T == P_F8 && a.x_type != HTR_E4M3))) {
      if constexpr (T != P_I8) return take(Stream<2, 1, 4>{});
    }
    if (wgs <= 256 && slabs >= 64) return take(Stream<1, 1, 16>{});
    return take(Stream<1, 1, 8>{});
  }
  // Matrices so small that each compute unit has a workgroup of 16 of their rows by 16 or 32 of x at most: many waves for each are faster than a ring for few.
  // Measured from HBM on 17 .. 384 rows of 256 .. 4096 matrix rows of 1024, 4096 and 8192 columns, 108 sizes in each type: the way taken was the fastest in all.
  // us by 16 rows, by 32, by tiles of 64x32: 64 rows on 1024x4096 in 16 bits 10.3, 14.7, 20.8, in e4m3 7.2, 9.8, 11.9; 48 rows on 2048x4096 19.5, 13.8, 21.0 and
  // 11.8, 9.9, 11.9; beyond the limits 192 rows on 1024x4096 26.1, 26.2, 20.7 and 16.1, 18.6, 11.8, 64 rows on 4096x4096 38, 30, 22 and 21.6, 19.4, 12.6.
  auto workgroups = [&](int height) {
    const float full = (float)a.rows / height, experts = (float)(a.rows < a.experts ? a.rows : a.experts);
    return (float)((a.m + 15) / 16) * (a.experts == 1 ? ceilf(full) : fmaxf(experts, full + 0.5f * experts));
  };
  const bool y_fits = span_bound(a.rows, a.experts, grouped, 16) <= 65535;      // the grid's second dimension
  if (y_fits && workgroups(16) <= 256.f) return take(Stream<1, 1, 8>{});
  if (y_fits && workgroups(32) <= 256.f) return take(Stream<1, 2, 8>{});
  if (!grouped) {
    if (mean <= 32) return a.m < 8192 ? take(Stream<1, 2, 8>{}) : a.m < 16384 ? take(Tiles<2, 2, 2, 1, 4>{}) : take(Tiles<4, 1, 2, 2, 4>{});
  } else if (mean <= 24) {
    // experts' rows are uneven: where 16 rows to a workgroup leave two to a compute unit they are still ahead of tiles of 128x32 (us, 192 rows of 8 experts of
    // 512x4096 in e4m3 12.1 and 16.8, in 16 bits 18.3 and 26.7; of 512x768 4.4 and 6.1, 5.9 and 8.4; 1056 rows of 48 of 72x3200 in 16 bits 20.1 and 19.4)
    return y_fits && workgroups(16) <= 512.f ? take(Stream<1, 1, 8>{}) : take(Tiles<4, 1, 2, 2, 4>{});
  }
  switch (T == P_F8 || T == P_I8 ? best_tile(TILES_8, a, (size_t)a.n) : best_tile(TILES_16, a, (size_t)a.n * 2)) {
    case 0: return take(Tiles<2, 4, 8, 4, 2>{});
    case 1: return take(Tiles<4, 2, 4, 4, 3>{});
    case 2: return take(Tiles<2, 2, 4, 4, 3>{});
    case 3: return take(Tiles<2, 2, 4, 2, 3>{});
    case 4: return take(Tiles<2, 2, 2, 2, 4>{});
    default: return take(Tiles<2, 2, 2, 1, 4>{});
  }
}
// In int8 the tables in e4m3 fit: the tile chosen takes as long as the best one on average and 1.15 times as long at most on 84 sizes of one
// matrix, 1.02 and 1.32 on 47 of experts.
// ---- few rows in int8
struct RowsGrid { int columns, kw, most, mtiles, workgroups; long long tiles; size_t lds; bool fits; };      // most: rows of a span; tiles: a bound where rows are grouped
RowsGrid rows_grid(const ProductArgs& a) {
  const bool grouped = a.ends != nullptr;
  RowsGrid g;
  // Experts' rows are uneven: spans of 16 or 32 read a matrix once that spans of 8 would read twice (us by 8, 16 and 32: 96 rows of 64 experts of 2816x2048 45.8, 46.0
  // and 60 by whole teams, 256 62.5, 57.5 and 63, 500 -, 67.9 and 65.4; 80 of 8 of 14336x4096 -, 93 and 77)
  g.columns = grouped ? (a.rows <= 6ll * a.experts ? 16 : 32) : a.rows <= 8 ? 8 : a.rows <= 16 ? 16 : 32;
  g.most = a.rows < g.columns ? a.rows : g.columns;
  // Waves to a team.  One matrix: all, so that few tiles come to as many workgroups (us by 8, 4 and 2: 1 row on 28672x4096 20.5, 21.7 and 22.3, 8 on 152064x4096 99.5, 100.3
  // and 98.4).  Experts have tiles enough; fewer waves to one mean fewer ends of tiles, more leave long rows to few (96 rows of 64 experts of 2816x2048 51.7, 47.1 and
  // 46.0, of 2048x1408 31.4, 28.9 and 26.9; 32 of 8 of 14336x4096 74.0, 73.3 and 76.3)
  g.kw = !grouped ? 8 : a.n > 2048 ? 4 : 2;
  g.mtiles = (a.m + rows_tile(g.kw) - 1) / rows_tile(g.kw);
  const long long spans = span_bound(a.rows, a.experts, grouped, g.columns);
  g.tiles = g.mtiles * spans;
  g.lds = rows_lds(g.most, g.columns, a.n, g.kw, grouped);
  // two workgroups to a compute unit where the rows of x are few to prepare (us by two and by one: 1 row on 6144x4096 7.7 and 8.0, 4 on 14336x4096 12.0 and 12.7,
  // 8 on 152064x4096 102 and 101, 32 on 28672x4096 30 and 25)
  int most = (a.rows <= 4 || grouped) && g.lds <= 80 * 1024 ? 512 : 256;
  g.workgroups = (int)(g.tiles < most ? g.tiles : most);
  g.fits = g.lds <= 160 * 1024 && spans / g.workgroups + 4 <= ROWS_SPANS;
  return g;
}
template <int X, int CT, int KW, bool GROUPED> hipError_t launch_rows(const ProductArgs& a, const RowsGrid& g, hipStream_t st) {
  const hipError_t e = allow_lds<k_product_rows<X, CT, KW, GROUPED>>(160 * 1024);
  return e != hipSuccess ? e : launch(k_product_rows<X, CT, KW, GROUPED>, dim3(g.workgroups), ROWS_WAVES * 64, g.lds, st, a, g.mtiles, g.most);
}
hipError_t launch_rows(const ProductArgs& a, hipStream_t st) {
  const RowsGrid g = rows_grid(a);
  if (a.ends != nullptr) {
    if (g.kw == 4) return g.columns == 16 ? launch_rows<P_I8, 2, 4, true>(a, g, st) : launch_rows<P_I8, 4, 4, true>(a, g, st);
    return g.columns == 16 ? launch_rows<P_I8, 2, 2, true>(a, g, st) : launch_rows<P_I8, 4, 2, true>(a, g, st);
  }
  if (a.x_type == HTR_BF16) return launch_rows<HTR_BF16, 1, 8, false>(a, g, st);
  if (a.x_type == HTR_F16) return launch_rows<HTR_F16, 1, 8, false>(a, g, st);
  if (a.x_type == HTR_F32) return launch_rows<HTR_F32, 1, 8, false>(a, g, st);
  return g.columns == 8    ? launch_rows<P_I8, 1, 8, false>(a, g, st)
         : g.columns == 16 ? launch_rows<P_I8, 2, 8, false>(a, g, st)
                           : launch_rows<P_I8, 4, 8, false>(a, g, st);
}
// Up to 32 rows of one matrix that LDS holds.  us by k_product_rows and by the faster of the kernels for more rows: 1 row on 1024x4096 4.9 and 5.3, on 6144x4096 7.7 and
// 10.1, 8 on 152064x4096 101 and 125, 16 on 14336x4096 14.0 and 15.8, 32 on 28672x4096 25 and 29, but 32 on 4096x4096 9.6 and 8.8 (the matrix's height is no part of the rule)
bool takes_rows(int64_t rows, int n) { return rows >= 1 && rows <= 32 && rows_lds((int)rows, 32, n, 8, false) <= 160 * 1024; }
// Up to 8 of them rounded on the way, by every workgroup for itself: 1 row on 6144x4096 9.5 us, 8 rows 11.3 (rounded ahead 7.7 and 8.5, and 4.5 for that launch), 16 rows
// on 14336x4096 19.2 (14.0 and 4.6)
bool rounds_rows(int64_t rows, int n) { return rows <= 8 && takes_rows(rows, n); }
// Up to 8 rows to an expert on average (us by k_product_rows and by the fastest of the others, 64 experts of 2816x2048: 96 rows 46 and 53, 256 57 and 69, 500 65 and 70,
// 800 73 and 69; 8 of 14336x4096: 48 rows 74 and 88; 64 of 2048x1408: 400 rows 36 and 37, 800 43 and 39)
bool few_int8(long long rows, int experts) { return rows <= 8ll * experts; }
// the kernel for few rows, for a product in int8
bool takes_rows(const ProductArgs& a) { return a.ends == nullptr ? takes_rows(a.rows, a.n) : few_int8(a.rows, a.experts) && rows_grid(a).fits; }
// silu(gate) up of rows by expert, where one launch is the better way (few rows to an expert: the matrices are read by k_product_stream, in int8 by k_product_rows, and
// k_gated or k_round_rows follows)
bool gates_in_one(long long rows, int experts, int type) { return type == HTR_I8 ? !few_int8(rows, experts) : !takes_16bit_rows(rows, experts, true); }
template <int T, typename F> auto gated_kernel(const ProductArgs& a, F take) {
  switch (best_tile(GATED_TILES, a, (size_t)a.n * bytes_of<T>)) {
    case 0: return take(Tiles<2, 4, 8, 4, 2, true>{});
    case 1: return take(Tiles<4, 2, 4, 4, 3, true>{});
    case 2: return take(Tiles<2, 2, 8, 2, 3, true>{});
    default: return take(Tiles<4, 1, 4, 2, 4, true>{});
  }
}
template <int T> hipError_t launch_product(const ProductArgs& a, bool gated, hipStream_t st) {
  auto take = [&](auto kernel) { return launch_kernel<T>(kernel, a, st); };
  return gated ? gated_kernel<T>(a, take) : product_kernel<T>(a, take);
}
hipError_t launch_product(const ProductArgs& a, int type, bool gated, hipStream_t st) {
  if (type == HTR_I8 && !gated && takes_rows(a)) return launch_rows(a, st);
  return type == HTR_E4M3 ? launch_product<P_F8>(a, gated, st) : type == HTR_I8 ? launch_product<P_I8>(a, gated, st) : type == HTR_BF16 ? launch_product<HTR_BF16>(a, gated, st) : launch_product<HTR_F16>(a, gated, st);
}
template <int T> void describe_product(const ProductArgs& a, bool gated, int* out) {
  auto take = [&](auto kernel) { describe_kernel<T>(kernel, a, out); };
  if (gated) gated_kernel<T>(a, take); else product_kernel<T>(a, take);
}
// columns: whole blocks of e4m3, rows on 16-byte boundaries
int unit_of(int type) { return type == HTR_E4M3 ? 128 : type == HTR_I8 ? 16 : 8; }
// what product_kernel takes: HTR_OK or the status to refuse with
int product_shape(long long rows, int m, int n, int experts, int type, bool grouped) {
  if (!is_8bit(type) && !is_16bit(type)) return HTR_ERR_DTYPE;
  if (rows < 0 || rows > (1ll << 31) - (1 << 20) || m < 1 || n < 1 || experts < 1 || experts > 65535 || n % unit_of(type)) return HTR_ERR_SIZE;
  if (type == HTR_I8 && n >= 1 << 17) return HTR_ERR_SIZE;        // 2^14 a product, sums below 2^31
  if (m > (1 << 26) || n > (1 << 22)) return HTR_ERR_SIZE;       // 256 rows of a tile by 32-bit distances; the launch's threads below 2^32
  // numbers of the smallest tiles, and workgroups where there is one to a tile (rows of fewer slabs than the deepest ring has stages)
  const long long tiles = span_bound(rows, experts, grouped, 32) * ((m + 63) / 64);
  return tiles > ((long long)n * (is_8bit(type) ? 1 : 2) > 128 * 3 ? (1ll << 31) - (1 << 16) : 1ll << 23) ? HTR_ERR_SIZE : HTR_OK;
}

// ---- a routed-expert layer: scratch laid out one after the other, every part on a 256-byte boundary
struct StackedScratch {
  size_t ends, token, pos_of, xq, xs, h, a, as, out, bytes;
  StackedScratch(long long tokens, int top, int experts, int hidden, int inter, int type) {
    size_t at = 0;
    auto take = [&](size_t n) { const size_t here = at; at += (n + 255) / 256 * 256; return here; };
    const size_t pairs = (size_t)tokens * top;
    const bool f8 = type == HTR_E4M3, i8 = type == HTR_I8, in_one = gates_in_one(pairs, experts, type);
    ends = take((size_t)experts * 4);
    token = take(pairs * 4);
    pos_of = take(pairs * 4);
    const bool ahead = i8 || (f8 && in_one);      // x is rounded by a launch of its own
    xq = take(ahead ? (size_t)tokens * hidden : 0);
    xs = take(i8 ? (size_t)tokens * 4 : ahead ? (size_t)tokens * (hidden / 128) * 4 : 0);
    h = take(!in_one ? pairs * 2 * inter * 4 : i8 ? pairs * inter * 4 : 0);
    a = take(pairs * inter * (f8 || i8 ? 1 : 2));
    as = take(i8 ? pairs * 4 : f8 ? pairs * (inter / 128) * 4 : 0);
    out = take(pairs * hidden * 4);
    bytes = at;
  }
};
hipError_t launch_route(RouteArgs a, hipStream_t st) {
  const dim3 grid((unsigned)((a.tokens + ROUTE_WAVES - 1) / ROUTE_WAVES));
  a.size = a.experts / a.groups;
  a.parts_log2 = 6;
  while ((64 >> a.parts_log2) < a.groups) --a.parts_log2;
  const int per = (a.size + (1 << a.parts_log2) - 1) >> a.parts_log2;      // below 2 ROUTE_MOST / 64
  auto take = [&](auto kernel) { return launch(kernel, grid, ROUTE_WAVES * 64, 0, st, a); };
  return per <= 1 ? take(k_route<1>) : per <= 2 ? take(k_route<2>) : per <= 4 ? take(k_route<4>) : per <= 8 ? take(k_route<8>) : per <= 16 ? take(k_route<16>) : take(k_route<32>);
}
int stacked_shape(long long tokens, int top, int experts, int hidden, int inter, int type) {
  if (tokens < 1 || top < 1 || experts < 1 || hidden < 1 || inter < 1 || top > 4096 || tokens >= (1 << 24) || inter > (1 << 28)) return HTR_ERR_SIZE;
  if (!is_8bit(type) && !is_16bit(type)) return HTR_ERR_DTYPE;
  if (hidden % 8 || inter % unit_of(type)) return HTR_ERR_SIZE;
  // loads go by 32-bit distances from x, from the gathered rows' scales and from an expert's matrices
  const unsigned long long size = is_8bit(type) ? 1 : 2, most = 1ull << 32;
  if (tokens * top > (1 << 30) || (unsigned long long)tokens * hidden * size >= most || 2ull * inter * hidden * size >= most) return HTR_ERR_SIZE;
  const int rc = product_shape(tokens * top, 2 * inter, hidden, experts, type, true);
  return rc != HTR_OK ? rc : product_shape(tokens * top, hidden, inter, experts, type, true);
}
}  // namespace

// ================================================================================================ C ABI
extern "C" {

int htr_rms_norm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, const void* weight, int64_t rows, int n, double eps,
                 int dtype, void* y, void* scales, void* sum, void* stream) {
  if (rows < 0 || rows > 0x7FFFFFFF || n < 1 || n > (1 << 30)) return HTR_ERR_SIZE;
  if (!is_dtype(dtype)) return HTR_ERR_DTYPE;
  if (rows == 0) return HTR_OK;
  if (!x || !weight || !y || (residual != nullptr) != (sum != nullptr)) return HTR_ERR_NULL;
  const size_t size = element_bytes(dtype);
  if (!aligned(x, size) || !aligned(residual, size) || !aligned(weight, size) || !aligned(sum, size) || !aligned(scales, 4) || (!scales && !aligned(y, size)))
    return HTR_ERR_ALIGN;
  if (scales && n % 128) return HTR_ERR_SIZE;
  hipStream_t st = (hipStream_t)stream;
  // a launch has fewer than 2^32 threads, up to 1024 of them to a row
  constexpr int64_t MOST = 1 << 21;
  for (int64_t r = 0; r < rows; r += MOST) {
    const int64_t count = rows - r < MOST ? rows - r : MOST;
    auto at = [&](const void* p, int64_t elements, size_t bytes) { return p ? (void*)((uint8_t*)p + elements * (int64_t)bytes) : nullptr; };
    const NormArgs a{at(x, r * x_stride, size), at(residual, r * residual_stride, size), weight, at(y, r * n, scales ? 1 : size), at(sum, r * n, size),
                     (float*)at(scales, r * (n / 128), 4), x_stride, residual_stride, count, n, eps};
    TRY_HIP(dtype == HTR_BF16 ? launch_norm<HTR_BF16>(a, st) : dtype == HTR_F16 ? launch_norm<HTR_F16>(a, st) : launch_norm<HTR_F32>(a, st));
  }
  return HTR_OK;
}

int htr_rms_norm_int8(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, const void* weight, int64_t rows, int n, double eps,
                      int dtype, void* y, void* scales, void* sum, void* stream) {
  if (rows < 0 || rows > 0x7FFFFFFF || n < 1 || n > (1 << 30) || n % 16) return HTR_ERR_SIZE;
  if (!is_dtype(dtype)) return HTR_ERR_DTYPE;
  if (rows == 0) return HTR_OK;
  if (!x || !weight || !y || !scales || (residual != nullptr) != (sum != nullptr)) return HTR_ERR_NULL;
  const size_t size = element_bytes(dtype);
  if (!aligned(x, size) || !aligned(residual, size) || !aligned(weight, size) || !aligned(sum, size) || !aligned(scales, 4)) return HTR_ERR_ALIGN;
  hipStream_t st = (hipStream_t)stream;
  constexpr int64_t MOST = 1 << 21;      // as in htr_rms_norm
  for (int64_t r = 0; r < rows; r += MOST) {
    const int64_t count = rows - r < MOST ? rows - r : MOST;
    auto at = [&](const void* p, int64_t elements, size_t bytes) { return p ? (void*)((uint8_t*)p + elements * (int64_t)bytes) : nullptr; };
    const NormArgs a{at(x, r * x_stride, size), at(residual, r * residual_stride, size), weight, at(y, r * n, 1), at(sum, r * n, size), (float*)scales + r,
                     x_stride, residual_stride, count, n, eps};
    TRY_HIP(dtype == HTR_BF16 ? launch_norm_int8<HTR_BF16>(a, st) : dtype == HTR_F16 ? launch_norm_int8<HTR_F16>(a, st) : launch_norm_int8<HTR_F32>(a, st));
  }
  return HTR_OK;
}

int htr_quantize_int8(const void* x, int64_t stride, int64_t rows, int n, int dtype, void* q, void* scales, void* stream) {
  if (rows < 0 || n < 1 || n % 16 || n > (1 << 30)) return HTR_ERR_SIZE;
  if (!is_dtype(dtype)) return HTR_ERR_DTYPE;
  if (rows == 0) return HTR_OK;
  if (!x || !q || !scales) return HTR_ERR_NULL;
  if (!aligned(x, element_bytes(dtype)) || !aligned(q, 8) || !aligned(scales, 4)) return HTR_ERR_ALIGN;
  TRY_HIP(launch_round(x, dtype, stride, rows, n, q, scales, (hipStream_t)stream));
  return HTR_OK;
}

int htr_quantize_e4m3(const void* x, int64_t stride, int64_t rows, int n, int dtype, void* q, void* scales, void* stream) {
  if (rows < 0 || n < 1 || n % 128 || n > (1 << 30)) return HTR_ERR_SIZE;
  if (!is_dtype(dtype)) return HTR_ERR_DTYPE;
  if (rows == 0) return HTR_OK;
  if (!x || !q || !scales) return HTR_ERR_NULL;
  if (!aligned(x, 16) || stride % 8 || !aligned(q, 8) || !aligned(scales, 4)) return HTR_ERR_ALIGN;
  const int64_t most = (1 << 27) / (n / 128);      // rows of 2^31 threads
  for (int64_t r = 0; r < rows; r += most)
    TRY_HIP(launch_quantize((const uint8_t*)x + r * stride * (int64_t)element_bytes(dtype), dtype, rows - r < most ? rows - r : most, n, stride, (uint8_t*)q + r * n,
                            (float*)scales + r * (n / 128), (hipStream_t)stream));
  return HTR_OK;
}

int htr_product_rounds_int8(int64_t rows, int n) { return rounds_rows(rows, n); }

int htr_product_rounds(int64_t rows, int experts, int grouped) { return rows > 0 && experts > 0 && takes_16bit_rows(rows, experts, grouped != 0); }

int htr_product_plan(int64_t rows, int m, int n, int experts, int grouped, int gated, int type, int x_type, int* out6) {
  if (!out6) return HTR_ERR_NULL;
  const int rc = product_shape(rows, m, n, experts, type, grouped != 0);
  if (rc != HTR_OK) return rc;
  if (x_type != type && !(type == HTR_E4M3 && is_16bit(x_type) && !gated && takes_16bit_rows(rows, experts, grouped != 0)) &&
      !(type == HTR_I8 && is_dtype(x_type) && !grouped && rounds_rows(rows, n)))
    return HTR_ERR_DTYPE;
  if (rows == 0 || (gated && (!grouped || m % (2 * unit_of(type)) || !gates_in_one(rows, experts, type))) || (!grouped && experts != 1)) return HTR_ERR_SIZE;
  const int some = 0;      // the choice asks whether there are ends, not what they hold
  ProductArgs a{};
  a.rows = (int)rows; a.m = m; a.n = n; a.experts = experts; a.x_type = x_type;
  a.ends = grouped ? &some : nullptr;
  if (type == HTR_I8 && !gated && takes_rows(a)) {
    const RowsGrid g = rows_grid(a);
    const int v[6] = {rows_tile(g.kw), g.columns, ROWS_WAVES, 0, g.workgroups, (int)g.tiles};
    memcpy(out6, v, sizeof(v));
    return HTR_OK;
  }
  if (type == HTR_E4M3) describe_product<P_F8>(a, gated != 0, out6);
  else if (type == HTR_I8) describe_product<P_I8>(a, gated != 0, out6);
  else if (type == HTR_BF16) describe_product<HTR_BF16>(a, gated != 0, out6);
  else describe_product<HTR_F16>(a, gated != 0, out6);
  return HTR_OK;
}

int htr_product(const void* x, int x_type, const void* x_scales, const void* w, const void* w_scales, const void* bias, const int32_t* ends, void* y,
                int64_t rows, int m, int n, int experts, int type, int y_dtype, void* stream) {
  const int rc = product_shape(rows, m, n, experts, type, ends != nullptr);
  if (rc != HTR_OK) return rc;
  if (!is_dtype(y_dtype)) return HTR_ERR_DTYPE;
  if (x_type != type && !(type == HTR_E4M3 && is_16bit(x_type) && takes_16bit_rows(rows, experts, ends != nullptr)) &&
      !(type == HTR_I8 && is_dtype(x_type) && ends == nullptr && rounds_rows(rows, n)))
    return HTR_ERR_DTYPE;
  if (ends == nullptr && experts != 1) return HTR_ERR_NULL;
  if (rows == 0) return HTR_OK;
  if (!x || !w || !y || (is_8bit(x_type) && !x_scales) || (is_8bit(type) && !w_scales)) return HTR_ERR_NULL;
  if (!aligned(x, 16) || !aligned(w, 16) || !aligned(y, 16) || !aligned(x_scales, 4) || !aligned(w_scales, 4) || !aligned(ends, 4) ||
      !aligned(bias, element_bytes(y_dtype)))
    return HTR_ERR_ALIGN;
  const ProductArgs a{x, (const float*)x_scales, w, (const float*)w_scales, bias, y, ends, nullptr, (int)rows, m, n, experts, y_dtype, x_type, nullptr, false};
  TRY_HIP(launch_product(a, type, false, (hipStream_t)stream));
  return HTR_OK;
}

size_t htr_moe_stacked_scratch_bytes(int64_t tokens, int top, int experts, int hidden, int inter, int type) {
  return stacked_shape(tokens, top, experts, hidden, inter, type) == HTR_OK ? StackedScratch(tokens, top, experts, hidden, inter, type).bytes : 0;
}

int htr_moe_stacked(const void* x, int dtype, const void* ids, int ids_int64, const float* weights, int64_t tokens, int top, const void* gate_up,
                    const void* gate_up_scales, const void* down, const void* down_scales, int experts, int hidden, int inter, int type, void* y,
                    void* scratch, size_t scratch_bytes, void* stream) {
  const int rc = stacked_shape(tokens, top, experts, hidden, inter, type);
  if (rc != HTR_OK) return rc;
  if (!is_16bit(dtype) || (!is_8bit(type) && type != dtype)) return HTR_ERR_DTYPE;
  const bool f8 = type == HTR_E4M3, i8 = type == HTR_I8;
  if (!x || !ids || !weights || !gate_up || !down || !y || ((f8 || i8) && (!gate_up_scales || !down_scales))) return HTR_ERR_NULL;
  if (!aligned(x, 16) || !aligned(gate_up, 16) || !aligned(down, 16) || !aligned(y, 16) || !aligned(ids, ids_int64 ? 8 : 4) || !aligned(weights, 4) ||
      !aligned(gate_up_scales, 4) || !aligned(down_scales, 4))
    return HTR_ERR_ALIGN;
  const StackedScratch at(tokens, top, experts, hidden, inter, type);
  if (!scratch || !aligned(scratch, 256) || scratch_bytes < at.bytes) return HTR_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  uint8_t* s = (uint8_t*)scratch;
  const int pairs = (int)(tokens * top);
  int *ends = (int*)(s + at.ends), *token = (int*)(s + at.token), *pos_of = (int*)(s + at.pos_of);
  float *h = (float*)(s + at.h), *out = (float*)(s + at.out);
  if (i8) {
    const dim3 grid((unsigned)(experts + (tokens + ORDER_WAVES - 1) / ORDER_WAVES));
    TRY_HIP(launch(dtype == HTR_BF16 ? k_order_and_round<HTR_BF16> : k_order_and_round<HTR_F16>, grid, ORDER_WAVES * 64, 0, st, ids, ids_int64, pairs, top, experts, ends, token,
                   pos_of, x, (int)tokens, hidden, s + at.xq, (float*)(s + at.xs)));
  } else {
    TRY_HIP(launch(k_expert_order, dim3(experts), ORDER_WAVES * 64, 0, st, ids, ids_int64, pairs, top, experts, ends, token, pos_of));
  }
  ProductArgs a{x, nullptr, gate_up, (const float*)gate_up_scales, nullptr, h, ends, token, pairs, 2 * inter, hidden, experts, HTR_F32, dtype, nullptr, f8};
  if (i8) {
    a.x_type = HTR_I8;
    a.x = s + at.xq; a.xs = (const float*)(s + at.xs);
  } else if (f8 && gates_in_one(pairs, experts, type)) {
    a.x_type = HTR_E4M3;
    TRY_HIP(launch_quantize(x, dtype, tokens, hidden, hidden, s + at.xq, (float*)(s + at.xs), st));
    a.x = s + at.xq; a.xs = (const float*)(s + at.xs);
  }
  if (i8) {
    // silu(gate) up stays float32 until a row's largest is known
    const bool in_one = gates_in_one(pairs, experts, type);
    TRY_HIP(launch_product(a, type, in_one, st));
    const int* last = ends + experts - 1;
    TRY_HIP((in_one ? launch_round<HTR_F32, false>(h, inter, pairs, inter, last, s + at.a, s + at.as, st)
                    : launch_round<HTR_F32, true>(h, 2 * inter, pairs, inter, last, s + at.a, s + at.as, st)));
  } else if (gates_in_one(pairs, experts, type)) {
    a.y = s + at.a; a.ys = (float*)(s + at.as); a.y_dtype = type;
    TRY_HIP(launch_product(a, type, true, st));
  } else {
    TRY_HIP(launch_product(a, type, false, st));
    TRY_HIP(f8 ? launch(k_gated<P_F8>, dim3(pairs), 256, 0, st, h, ends, experts, inter, s + at.a, (float*)(s + at.as))
               : dtype == HTR_BF16 ? launch(k_gated<HTR_BF16>, dim3(pairs), 256, 0, st, h, ends, experts, inter, s + at.a, nullptr)
                                   : launch(k_gated<HTR_F16>, dim3(pairs), 256, 0, st, h, ends, experts, inter, s + at.a, nullptr));
  }
  const ProductArgs d{s + at.a, (const float*)(s + at.as), down, (const float*)down_scales, nullptr, out, ends, nullptr, pairs, hidden, inter, experts, HTR_F32, type, nullptr, false};
  TRY_HIP(launch_product(d, type, false, st));
  const dim3 grid((unsigned)tokens, (hidden + 2047) / 2048);
  TRY_HIP(dtype == HTR_BF16 ? launch(k_weighted_sum<HTR_BF16>, grid, 256, 0, st, out, pos_of, weights, top, hidden, y)
                            : launch(k_weighted_sum<HTR_F16>, grid, 256, 0, st, out, pos_of, weights, top, hidden, y));
  return HTR_OK;
}

int htr_route(const void* logits, int64_t stride, int dtype, int64_t tokens, int experts, int top, int sigmoid, const float* bias, int groups, int top_groups,
              int group_best, int renormalize, double scale, int32_t* ids, float* weights, void* stream) {
  if (tokens < 0 || tokens > 0x7FFFFFFF || experts < 1 || experts > ROUTE_MOST || top < 1 || top > experts || top > 64) return HTR_ERR_SIZE;
  if (groups < 1 || groups > 64 || experts % groups || top_groups < 1 || top_groups > groups || group_best < 1 || group_best > 2 || top > experts / groups * top_groups) return HTR_ERR_SIZE;
  if (!is_dtype(dtype)) return HTR_ERR_DTYPE;
  if (tokens == 0) return HTR_OK;
  if (!logits || !ids || !weights) return HTR_ERR_NULL;
  if (!aligned(logits, element_bytes(dtype)) || !aligned(bias, 4) || !aligned(ids, 4) || !aligned(weights, 4)) return HTR_ERR_ALIGN;
  constexpr int64_t MOST = 1 << 22;      // a launch has fewer than 2^32 threads, 64 of them to a token
  for (int64_t t = 0; t < tokens; t += MOST) {
    const RouteArgs a{(const uint8_t*)logits + t * stride * (int64_t)element_bytes(dtype), bias, ids + t * top, weights + t * top, stride, tokens - t < MOST ? tokens - t : MOST,
                      dtype, experts, top, sigmoid, groups, top_groups, group_best, renormalize, scale, 0, 0};
    TRY_HIP(launch_route(a, (hipStream_t)stream));
  }
  return HTR_OK;
}
}  // extern "C"
