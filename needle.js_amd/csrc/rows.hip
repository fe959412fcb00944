// Products in 8-bit integers: activation rows quantized to int8 with one scale
// a row, times an int8 matrix with one scale per output channel.
//
//   s_m = max(1e-12, max_k |x[m][k]|) / 127     (float64; kept as f32)
//   c[m][k] = roundTiesToEven(x[m][k] / s_m)    (float64 division)
//   y[m][n] = add[m][n] + f32(s_m) s_w[n] sum_k W[n][k] c[m][k]
//
// The quantizer is the KV cache's own (#storeKV, model/runtime.ts:697-714,
// 901-907).  The integer sum is exact (k <= 8192, |W c| <= 2^14: below 2^27), so
// it does not depend on how it is split; the result is add + ((float)sum s_w) s_m with
// each step rounded to f32, the same bits from every form of the kernels.
//
// A handle (nd_rows) holds the quantized rows in the order the matrix cores
// read, the order of nd_tile_weights: 1 KiB blocks [row / 16][k / 64], lane l of
// a block holding row l % 16, k [16 (l / 16), +16).  One quantization serves every
// matrix the rows meet (q, k, v and gate of a layer).
#include <cstdlib>
#include <cstring>
#include <new>
#include <type_traits>

#include "nd_internal.hpp"
#include "nd_wave.hpp"

struct nd_rows {
  uint32_t max_rows = 0, k = 0, count = 0;
  int8_t* codes = nullptr;  // operand order, rows rounded up to 16
  float* scales = nullptr;  // [max_rows rounded up to 16]
};

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

// The code of x under the row's scale: roundTiesToEven(x / s).  r = x * (127 / m)
// in f32 is within 3 roundings, 2^-22 of |r| <= 127 (3.1e-5), of the float64
// quotient, so its nearest integer is the code unless r lies that near a
// half-integer; there (about one value in 5000) the float64 quotient decides.
// A NaN anywhere fails the comparison and takes the same path, to code 0.
__device__ __forceinline__ int code_of(float x, float inv, double s) {
  const float r = x * inv, n = rintf(r);
  if (fabsf(r - n) < 0.4999f) return (int)n;
  const double q = rint((double)x / s);
  return q != q ? 0 : (int)q;
}

// A workgroup of eight waves takes 8 / WPR rows, WPR waves a row.  A lane takes
// float4 units of its row 64 WPR apart, so loads are contiguous and the row is
// read once (VEC units a lane stay in registers, k <= 256 VEC WPR); a chunk of
// columns at a time the codes meet in LDS, where the operand order has them, and
// leave in runs of the rows' 16-byte pieces (WPR = 1: 128 bytes).  Many rows are
// bound by the copy of x (one wave a row keeps its sums in the wave); few rows by
// the chain load, maximum, quotient, so that eight waves share one.
constexpr uint32_t kQuantWaves = 8;
template <int VEC, int WPR>
__global__ __launch_bounds__(64 * kQuantWaves) void quantize_rows_kernel(
    const float* __restrict__ X, uint32_t ldx, uint32_t M, uint32_t K, int8_t* __restrict__ codes,
    float* __restrict__ scales) {
  constexpr uint32_t kRows = kQuantWaves / WPR, kLanes = 64 * WPR;
  constexpr int CH = VEC < 8 ? VEC : 8;  // units of a chunk
  __shared__ uint4 s_codes[CH * kLanes / 4][kRows];  // [16-byte piece of the chunk][row]
  __shared__ float s_top[kQuantWaves];
  const uint32_t wave = threadIdx.x >> 6, row = wave / WPR, l = threadIdx.x % kLanes;
  const uint32_t m0 = blockIdx.x * kRows, m = m0 + row, units = K / 4;
  const bool live = m < M;
  const float4* x = reinterpret_cast<const float4*>(X + (size_t)(live ? m : m0) * ldx);
  float4 v[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const uint32_t u = l + kLanes * i;
    v[i] = u < units ? x[u] : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    for (float e : {v[i].x, v[i].y, v[i].z, v[i].w})
      top = __builtin_elementwise_maximum(top, fabsf(e));  // a NaN stays
  top = nd::wave_max_js(top);
  if constexpr (WPR > 1) {
    if ((threadIdx.x & 63) == 0) s_top[wave] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WPR; ++i) top = nd::js_max(top, s_top[row * WPR + i]);
  }
  const double m64 = top != top ? (double)top : fmax(1e-12, (double)top);
  const double s = m64 / 127.0;
  const float inv = 127.f / (float)m64;
  if (live && l == 0) scales[m] = (float)s;
  // Piece c of the row (columns [16 c, +16)) is bytes [16 row, +16) of quarter
  // c % 4 of block c / 4.
  uint4* out = reinterpret_cast<uint4*>(codes + (size_t)(m0 / 16) * 16 * K) + m0 % 16;
#pragma unroll
  for (int c = 0; c < VEC; c += CH) {
    if (c) __syncthreads();
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const float4 f = v[c + i];
      const uint32_t c0 = code_of(f.x, inv, s) & 255, c1 = code_of(f.y, inv, s) & 255,
                     c2 = code_of(f.z, inv, s) & 255, c3 = code_of(f.w, inv, s) & 255;
      reinterpret_cast<uint32_t*>(&s_codes[(l + kLanes * i) >> 2][row])[l & 3] =
          c0 | c1 << 8 | c2 << 16 | c3 << 24;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < CH * kLanes / 4 * kRows; i += 64 * kQuantWaves) {
      const uint32_t piece = c * kLanes / 4 + i / kRows, r = i % kRows;
      if (piece * 16 < K && m0 + r < M) out[(size_t)piece * 16 + r] = s_codes[i / kRows][r];
    }
  }
}

struct Product {
  const int8_t* w;      // operand order, or row-major codes
  const float* sw;      // [N]
  const int8_t* x;      // operand order
  const float* sx;      // [M]
  const float* add;     // [M][ldy] or null; may be y
  float* y;             // [M][ldy]
  uint32_t M, N, K, ldy;
  bool rowmajor;        // of w
  bool across;          // rows of y or add without 16-byte accesses
};

typedef float v4f __attribute__((ext_vector_type(4)));

// A lane's four outputs of a 16 x 16 tile.  Along a row (weights as the product's
// left operand): row m, columns [n, n + 4), stored in one access.  Where the rows
// of y start at odd places, across them (activations on the left): rows [m, m +
// 4), column n, so that each of the four stores writes 64 B of four rows and not
// 4 B of sixty-four places.
template <bool ACROSS>
struct Four {
  static __device__ __forceinline__ uint32_t row(uint32_t lane) {
    return ACROSS ? (lane >> 4) * 4 : lane & 15;
  }
  static __device__ __forceinline__ uint32_t col(uint32_t lane) {
    return ACROSS ? lane & 15 : (lane >> 4) * 4;
  }
  static __device__ __forceinline__ v4i product(v4i w, v4i x, v4i acc) {
    return ACROSS ? __builtin_amdgcn_mfma_i32_16x16x64_i8(x, w, acc, 0, 0, 0)
                  : __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, acc, 0, 0, 0);
  }
  // Scales; past M or N: those of some row or column, of outputs that nobody stores.
  static __device__ __forceinline__ v4f load_sw(const Product& p, uint32_t n) {
    if constexpr (ACROSS) return v4f(p.sw[min(n, p.N - 1)]);
    return *reinterpret_cast<const v4f*>(p.sw + min(n, p.N - 4));
  }
  static __device__ __forceinline__ v4f load_sx(const Product& p, uint32_t m) {
    if constexpr (!ACROSS) return v4f(p.sx[min(m, p.M - 1)]);
    v4f s;
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = p.sx[min(m + i, p.M - 1)];
    return s;
  }
  // Without contraction (here a multiply-add of the second product would take the
  // place of two roundings in some forms and not in others).
  static __device__ __forceinline__ v4f scaled(v4i c, v4f sw, v4f sx) {
#pragma clang fp contract(off)
    return v4f{(float)c[0], (float)c[1], (float)c[2], (float)c[3]} * sw * sx;
  }
  // What they are added to (WHOLE: all four are there).
  template <bool WHOLE>
  static __device__ __forceinline__ v4f load_add(const Product& p, uint32_t m, uint32_t n) {
    v4f a = {0.f, 0.f, 0.f, 0.f};
    if (!p.add || (!WHOLE && (m >= p.M || n >= p.N))) return a;
    const float* at = p.add + (size_t)m * p.ldy + n;
    if constexpr (!ACROSS) return *reinterpret_cast<const v4f*>(at);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (WHOLE || m + i < p.M) a[i] = at[(size_t)i * p.ldy];
    return a;
  }
  template <bool WHOLE>
  static __device__ __forceinline__ void store(const Product& p, uint32_t m, uint32_t n, v4f v) {
    if (!WHOLE && (m >= p.M || n >= p.N)) return;
    float* at = p.y + (size_t)m * p.ldy + n;
    if constexpr (ACROSS) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (WHOLE || m + i < p.M) at[(size_t)i * p.ldy] = v[i];
    } else {
      *reinterpret_cast<v4f*>(at) = v;
    }
  }
};

// Lane's 16 bytes of weight rows [16 tile, +16), k block kb.  Rows past N of the
// last tile are zero in the copy and row N - 1 again from row-major codes; no
// product of theirs is stored.
template <bool ROWMAJOR>
__device__ __forceinline__ v4i load_w(const Product& p, uint32_t tile, uint32_t kb, uint32_t lane) {
  if constexpr (ROWMAJOR) {
    const uint32_t n = min(tile * 16 + (lane & 15), p.N - 1);
    return *reinterpret_cast<const v4i*>(p.w + (size_t)n * p.K + kb * 64 + (lane >> 4) * 16);
  }
  return *reinterpret_cast<const v4i*>(p.w + ((size_t)tile * (p.K / 64) + kb) * 1024 + lane * 16);
}
__device__ __forceinline__ v4i load_x(const Product& p, uint32_t tile, uint32_t kb, uint32_t lane) {
  return *reinterpret_cast<const v4i*>(p.x + ((size_t)tile * (p.K / 64) + kb) * 1024 + lane * 16);
}

// Few rows, or few tiles for the GPU: workgroup = MT x NT tiles of 16 x 16
// outputs, its eight waves splitting k (exact integer sums, so the split does
// not show), operands from memory to registers, the waves' sums through LDS.
// Bound by the stream of the weights (1 x 4096 x 4096: 3.4 us, 4.9 TB/s).  Every k
// block of a wave waits for memory once unless the next ones are on their way:
// with AHEAD of them 3.4 against 4.0 us; where K leaves a wave one or two, their
// registers would only cost workgroups on a CU (7 x 32768 x 512: 5.1 against 3.5).
// The longer side of the output runs along x, padded to whole rounds of the eight
// XCDs (workgroup L runs on XCD L % 8), so that an XCD's L2 holds an eighth of
// that side's operand and the tiles that share it (4000 x 200 x 8192: 19.4
// against 35.1 us).
constexpr uint32_t kSplitWaves = 8;
template <int MT, int NT, int AHEAD, bool ROWMAJOR, bool ACROSS>
__global__ __launch_bounds__(64 * kSplitWaves) void rows_split_kernel(Product p) {
  __shared__ v4i s_sum[kSplitWaves][MT * NT][64];
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const uint32_t nt0 = (p.M > p.N ? blockIdx.y : blockIdx.x) * NT;
  const uint32_t mt0 = (p.M > p.N ? blockIdx.x : blockIdx.y) * MT;
  const uint32_t last_n = (p.N + 15) / 16 - 1, last_m = (p.M + 15) / 16 - 1, kbs = p.K / 64;
  if (nt0 > last_n || mt0 > last_m) return;
  // The four outputs this thread stores, their scales and addends on the way.
  static_assert(MT * NT <= (int)kSplitWaves, "a group of outputs a thread at most");
  const uint32_t mine = threadIdx.x >> 6;  // tile
  using F = Four<ACROSS>;
  const uint32_t m = (mt0 + mine / NT) * 16 + F::row(lane);
  const uint32_t n = (nt0 + mine % NT) * 16 + F::col(lane);
  v4f sw = {}, sx = {}, add = {};
  if (mine < MT * NT) {
    sw = F::load_sw(p, n);
    sx = F::load_sx(p, m);
    add = F::template load_add<false>(p, m, n);
  }
  // AHEAD > 1: K has at least four k blocks a wave, a power of two of them; the
  // next four, or AHEAD, are on their way at a time.
  v4i acc[MT][NT] = {};
  auto sum_over = [&](auto ahead) {
    constexpr uint32_t STAGES = ahead.value;
    v4i w[STAGES][NT], x[STAGES][MT];
    auto load = [&](uint32_t u, uint32_t kb) {
#pragma unroll
      for (int j = 0; j < NT; ++j) w[u][j] = load_w<ROWMAJOR>(p, min(nt0 + j, last_n), kb, lane);
#pragma unroll
      for (int i = 0; i < MT; ++i) x[u][i] = load_x(p, min(mt0 + i, last_m), kb, lane);
    };
    auto use = [&](uint32_t u) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = F::product(w[u][j], x[u][i], acc[i][j]);
    };
#pragma unroll
    for (uint32_t u = 0; u < STAGES; ++u) load(u, wave + u * kSplitWaves);
    for (uint32_t kb = wave + STAGES * kSplitWaves; kb < kbs; kb += STAGES * kSplitWaves)
#pragma unroll
      for (uint32_t u = 0; u < STAGES; ++u) {
        use(u);
        load(u, kb + u * kSplitWaves);
      }
#pragma unroll
    for (uint32_t u = 0; u < STAGES; ++u) use(u);
  };
  if constexpr (AHEAD == 1) {
    if (wave < kbs) sum_over(std::integral_constant<uint32_t, 1>{});
  } else if (AHEAD == 4 || kbs < AHEAD * kSplitWaves) {
    sum_over(std::integral_constant<uint32_t, 4>{});
  } else {
    sum_over(std::integral_constant<uint32_t, AHEAD>{});
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) s_sum[wave][i * NT + j][lane] = acc[i][j];
  __syncthreads();
  if (mine >= MT * NT) return;
  v4i sum = s_sum[0][mine][lane];
#pragma unroll
  for (uint32_t w = 1; w < kSplitWaves; ++w) sum += s_sum[w][mine][lane];
  v4f v = F::scaled(sum, sw, sx);
  if (p.add) v = add + v;
  F::template store<false>(p, m, n, v);
}

// Many rows: WM x WN waves, a wave TM x TN tiles of 16 x 16 outputs.  The
// activations, which WN waves share, go through LDS, 64 k a stage in two buffers
// (one barrier a stage); the weights, which only WM waves share, go from memory
// to registers.  Half of the operand bytes keep off the LDS that way: with both
// operands in it, its bandwidth bounds the product before the matrix cores do.
// Both operands are on their way three stages ahead (weights in four register
// buffers, activations in two and the LDS).
// Workgroup L runs on XCD L % 8: each XCD takes a contiguous run of tiles, kSuper
// tile columns wide, so that the workgroups on it share rows and columns in its
// L2.
constexpr uint32_t kSuper = 4;
template <int WM, int WN, int TM, int TN, bool ROWMAJOR, bool ACROSS>
__global__ __launch_bounds__(64 * WM * WN) void rows_tile_kernel(Product p) {
  constexpr uint32_t W = WM * WN, XT = WM * TM, XL = (XT + W - 1) / W;
  __shared__ v4i s_x[2][XT][64];
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const uint32_t last_n = (p.N + 15) / 16 - 1, last_m = (p.M + 15) / 16 - 1, kbs = p.K / 64;
  const uint32_t cols = (last_n + WN * TN) / (WN * TN), rows = (last_m + WM * TM) / (WM * TM);
  const uint32_t tiles = cols * rows, per = (tiles + 7) / 8;
  const uint32_t tile = blockIdx.x % 8 * per + blockIdx.x / 8;
  if (blockIdx.x / 8 >= per || tile >= tiles) return;
  const uint32_t group = tile / (rows * kSuper), width = min(kSuper, cols - group * kSuper);
  const uint32_t in = tile - group * rows * kSuper;
  const uint32_t mt0 = in / width * XT, nt0 = (group * kSuper + in % width) * (WN * TN);
  const uint32_t wn = nt0 + wave % WN * TN, wm = wave / WN * TM;
  using F = Four<ACROSS>;
  v4i acc[TM][TN] = {};
  v4i rx[2][XL], rw[4][TN];
  auto load_stage = [&](v4i* r, uint32_t kb) {
#pragma unroll
    for (uint32_t i = 0; i < XL; ++i)
      r[i] = load_x(p, min(mt0 + min(wave + W * i, XT - 1), last_m), min(kb, kbs - 1), lane);
  };
  auto store_stage = [&](uint32_t b, const v4i* r) {
#pragma unroll
    for (uint32_t i = 0; i < XL; ++i)
      if (XT % W == 0 || wave + W * i < XT) s_x[b][wave + W * i][lane] = r[i];
  };
  auto load_weights = [&](v4i* w, uint32_t kb) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
      w[j] = load_w<ROWMAJOR>(p, min(wn + j, last_n), min(kb, kbs - 1), lane);
  };
  load_stage(rx[0], 0);
#pragma unroll
  for (int i = 0; i < 3; ++i) load_weights(rw[i], i);
  load_stage(rx[1], 1);
  store_stage(0, rx[0]);
  load_stage(rx[0], 2);
  nd::lds_barrier();
  for (uint32_t kb = 0; kb < kbs; kb += 4) {
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      load_weights(rw[(u + 3) % 4], kb + u + 3);
      store_stage((u + 1) % 2, rx[(u + 1) % 2]);  // last read before the barrier
      load_stage(rx[(u + 1) % 2], kb + u + 3);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const v4i x = s_x[u % 2][wm + i][lane];
#pragma unroll
        for (int j = 0; j < TN; ++j)
          acc[i][j] = F::product(rw[u][j], x, acc[i][j]);
      }
      nd::lds_barrier();
      if (u == 1 && kb + 2 >= kbs) break;  // k = 128
    }
  }
  // All scales first (the stores could alias them, as far as the compiler knows);
  // a wave whose outputs are all there stores them straight.
  const uint32_t m0 = (mt0 + wm) * 16 + F::row(lane), n0 = wn * 16 + F::col(lane);
  v4f sw[TN], sx = F::load_sx(p, m0);
#pragma unroll
  for (int j = 0; j < TN; ++j) sw[j] = F::load_sw(p, n0 + 16 * j);
  auto store = [&](auto whole) {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      v4f v[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) v[j] = F::scaled(acc[i][j], sw[j], sx);
      if (i + 1 < TM) sx = F::load_sx(p, m0 + 16 * (i + 1));
      if (p.add) {
        v4f a[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j)
          a[j] = F::template load_add<whole.value>(p, m0 + 16 * i, n0 + 16 * j);
#pragma unroll
        for (int j = 0; j < TN; ++j) v[j] = a[j] + v[j];
      }
#pragma unroll
      for (int j = 0; j < TN; ++j)
        F::template store<whole.value>(p, m0 + 16 * i, n0 + 16 * j, v[j]);
    }
  };
  if ((mt0 + wm + TM) * 16 <= p.M && (wn + TN) * 16 <= p.N)
    store(std::true_type{});
  else
    store(std::false_type{});
}

hipError_t launch_quantize(const nd_rows* r, const float* x, uint32_t ldx, uint32_t rows,
                           hipStream_t s) {
  const uint32_t k = r->k;
  auto go = [&](auto kernel, uint32_t per) {
    hipLaunchKernelGGL(kernel, dim3((rows + per - 1) / per), dim3(64 * kQuantWaves), 0, s, x, ldx,
                       rows, k, r->codes, r->scales);
    return hipGetLastError();
  };
  // Few rows: a workgroup each (1 x 4096: 2.6 against 5.8 us).
  if (rows <= 256) {
    if (k <= 2048) return go(quantize_rows_kernel<1, 8>, 1);
    return k <= 4096 ? go(quantize_rows_kernel<2, 8>, 1) : go(quantize_rows_kernel<4, 8>, 1);
  }
  if (k <= 512) return go(quantize_rows_kernel<2, 1>, kQuantWaves);
  if (k <= 2048) return go(quantize_rows_kernel<8, 1>, kQuantWaves);
  if (k <= 4096) return go(quantize_rows_kernel<16, 1>, kQuantWaves);
  return go(quantize_rows_kernel<32, 1>, kQuantWaves);
}

// The form of a product's kernels: weights without a copy in operand order, outputs
// without 16-byte accesses.
template <class F>
hipError_t by_form(const Product& p, F f) {
  using Y = std::true_type;
  using N = std::false_type;
  if (p.rowmajor) return p.across ? f(Y{}, Y{}) : f(Y{}, N{});
  return p.across ? f(N{}, Y{}) : f(N{}, N{});
}
template <int WM, int WN, int TM, int TN>
hipError_t launch_tile(const Product& p, hipStream_t s) {
  const uint32_t mt = (p.M + 15) / 16, nt = (p.N + 15) / 16;
  const uint32_t tiles = ((mt + WM * TM - 1) / (WM * TM)) * ((nt + WN * TN - 1) / (WN * TN));
  return by_form(p, [&](auto r, auto a) {
    hipLaunchKernelGGL((rows_tile_kernel<WM, WN, TM, TN, r.value, a.value>),
                       dim3((tiles + 7) / 8 * 8), dim3(64 * WM * WN), 0, s, p);
    return hipGetLastError();
  });
}
template <int MT, int NT, int AHEAD>
hipError_t launch_split(const Product& p, hipStream_t s) {
  const uint32_t m = ((p.M + 15) / 16 + MT - 1) / MT, n = ((p.N + 15) / 16 + NT - 1) / NT;
  auto up8 = [](uint32_t v) { return (v + 7) / 8 * 8; };
  return by_form(p, [&](auto r, auto a) {
    hipLaunchKernelGGL((rows_split_kernel<MT, NT, AHEAD, r.value, a.value>),
                       p.M > p.N ? dim3(up8(m), n) : dim3(m > 1 ? up8(n) : n, m),
                       dim3(64 * kSplitWaves), 0, s, p);
    return hipGetLastError();
  });
}

hipError_t launch_product(const Product& p, hipStream_t s) {
  const uint32_t mt = (p.M + 15) / 16, nt = (p.N + 15) / 16;
  // By the number of 16 x 16 output tiles and by k; us a call of the form taken and
  // of its neighbours (tile forms by their outputs, split forms by tiles a
  // workgroup):
  //   1368 x 5281 x 8192   28466 tiles  128 x 256: 67    64 x 128: 76
  //   2034 x 4956 x 128    39680        64 x 128: 12.2   128 x 256: 13.3
  //   8026 x 723 x 2048    23092        64 x 128: 20.5   128 x 256: 22.9  64 x 64: 26
  //   180 x 40000 x 2048   30000        64 x 128: 26.7   128 x 256: 34.0 (192 and 256 rows)
  //   181 x 11162 x 128     8376        64 x 128: 5.8    64 x 64: 5.3     128 x 256: 6.8
  // (up to 128 rows the 64 x 128 on eight waves: more of the weights on their way)
  //   60 x 32768 x 8192     8192        eight waves: 43.0  four: 50.0     split 4 x 2: 58.6
  //   128 x 9000 x 2048     4504        eight waves: 9.0   four: 9.3      split 4 x 2: 10.6
  //   128 x 7200 x 4096     3600        split 4 x 2: 11.1  eight waves: 15.6
  //   128 x 131072 x 512   65536        128 x 256: 24.3  eight waves: 29.2
  //   700 x 1536 x 2048     4224        64 x 64: 9.8     split 4 x 2: 9.8
  //   700 x 1536 x 4096     4224        split 4 x 2: 14.5  64 x 64: 17.6
  //   2001 x 512 x 2048     4032        split 4 x 2: 7.7  64 x 64: 8.1    2 x 2: 8.7
  //   4000 x 200 x 8192     3250        split 4 x 2: 19.4  2 x 2: 26.2    64 x 64: 29
  //   300 x 515 x 8192       627        split 2 x 2: 6.1  4 x 2: 7.8      2 x 1: 8.3
  //   250 x 515 x 2048       528        split 2 x 2: 3.1  2 x 1: 3.6      4 x 2: 3.8
  //   24 x 4096 x 8192       512        split 2 x 1: 6.3  2 x 2: 7.4
  //   60 x 9000 x 512       2252        split 2 x 2: 3.4  2 x 1: 3.6      4 x 2: 3.8
  //   1 x 32768 x 1024      2048        split 1 x 2: 4.0  1 x 1: 4.8
  //   1 x 4096 x 8192        256        split 1 x 1: 4.8  1 x 2: 5.8
  const uint64_t outs = (uint64_t)mt * nt;
  const bool deep = p.K >= 64 * 4 * kSplitWaves;  // four k blocks a wave of a split
  if (mt == 1) {
    if (nt >= 1024) return deep ? launch_split<1, 2, 4>(p, s) : launch_split<1, 2, 1>(p, s);
    return deep ? launch_split<1, 1, 8>(p, s) : launch_split<1, 1, 1>(p, s);
  }
  const bool whole = (mt + 7) / 8 * 8 <= mt + mt / 6;  // blocks of 128 rows, mostly full
  if (outs >= 24576 && p.K >= 512 && whole) return launch_tile<1, 8, 8, 2>(p, s);
  if (outs > 4096 && mt > 2 && mt <= 8) return launch_tile<1, 8, 4, 1>(p, s);
  if (outs > 6144 && mt > 2) return launch_tile<1, 4, 4, 2>(p, s);
  if (outs > 4096 && mt > 2 && p.K <= 2048) return launch_tile<1, 4, 4, 1>(p, s);
  if (outs <= 512 || (mt == 2 && deep))
    return deep ? launch_split<2, 1, 4>(p, s) : launch_split<2, 1, 1>(p, s);
  if (!deep) return launch_split<2, 2, 1>(p, s);
  return outs <= 1024 ? launch_split<2, 2, 4>(p, s) : launch_split<4, 2, 4>(p, s);
}

}  // namespace

void nd_rows_release(nd_rows* r) {
  hipFree(r->codes);
  hipFree(r->scales);
  delete r;
}

extern "C" {

nd_status nd_rows_create(nd_ctx* ctx, uint32_t max_rows, uint32_t k, nd_rows** out) {
  if (!ctx) return nd_fail(nullptr, ND_ERR_BACKEND, "context is NULL");
  if (!out) return nd_fail(ctx, ND_ERR_INVALID, "out is NULL");
  *out = nullptr;
  if (max_rows == 0 || max_rows > (1u << 20))
    return nd_fail(ctx, ND_ERR_INVALID, "nd_rows_create: 1..%u rows, got %u", 1u << 20, max_rows);
  if (k < 128 || k > 8192 || (k & (k - 1)) != 0)
    return nd_fail(ctx, ND_ERR_INVALID, "nd_rows_create: k=%u must be a power of two in [128, 8192]",
                   k);
  ND_ON_DEVICE(ctx);
  nd_rows* r = new (std::nothrow) nd_rows();
  if (!r) return nd_fail(ctx, ND_ERR_NOMEM, "no host memory");
  r->max_rows = max_rows;
  r->k = k;
  const size_t padded = ((size_t)max_rows + 15) / 16 * 16;
  hipError_t e = hipMalloc(&r->codes, padded * k);
  if (e == hipSuccess) e = hipMalloc(&r->scales, padded * sizeof(float));
  if (e == hipSuccess) e = hipMemsetAsync(r->codes, 0, padded * k, ctx->stream);
  if (e == hipSuccess) e = hipMemsetAsync(r->scales, 0, padded * sizeof(float), ctx->stream);
  if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
  if (e != hipSuccess) {
    nd_rows_release(r);
    return nd_hip_fail(ctx, e, "activation rows");
  }
  if (!nd_hold(ctx->rows, r)) {
    nd_rows_release(r);
    return nd_fail(ctx, ND_ERR_NOMEM, "no host memory");
  }
  *out = r;
  return ND_OK;
}

nd_status nd_rows_free(nd_ctx* ctx, nd_rows* r) {
  if (!ctx) return nd_fail(nullptr, ND_ERR_BACKEND, "context is NULL");
  if (!r) return ND_OK;
  if (!ctx->rows.erase(r)) return nd_fail(ctx, ND_ERR_INVALID, "rows do not belong to context");
  ND_ON_DEVICE(ctx);
  ND_HIP(ctx, hipDeviceSynchronize());  // calls may have used any stream
  nd_rows_release(r);
  return ND_OK;
}

static nd_status check_rows(nd_ctx* ctx, const nd_rows* r) {
  if (!r || !ctx->rows.count(const_cast<nd_rows*>(r)))
    return nd_fail(ctx, ND_ERR_INVALID, "rows do not belong to context");
  return ND_OK;
}

nd_status nd_rows_quantize_d(nd_ctx* ctx, nd_rows* r, const float* x, uint32_t count, uint32_t ldx,
                             void* stream) {
  if (!ctx) return nd_fail(nullptr, ND_ERR_BACKEND, "context is NULL");
  nd_status st = check_rows(ctx, r);
  if (st != ND_OK) return st;
  if (count > r->max_rows)
    return nd_fail(ctx, ND_ERR_INVALID, "%u rows, room for %u", count, r->max_rows);
  if (ldx == 0) ldx = r->k;
  if (ldx < r->k || ldx % 4 != 0)
    return nd_fail(ctx, ND_ERR_INVALID, "row stride %u: at least k=%u and a multiple of 4", ldx,
                   r->k);
  if (count && (!x || (reinterpret_cast<uintptr_t>(x) & 15)))
    return nd_fail(ctx, ND_ERR_INVALID, "x must be a 16-byte aligned device pointer");
  if (count) {
    ND_ON_DEVICE(ctx);
    ND_HIP(ctx, launch_quantize(r, x, ldx, count, nd_pick_stream(ctx, stream)));
  }
  r->count = count;
  return ND_OK;
}

nd_status nd_rows_read(nd_ctx* ctx, const nd_rows* r, int8_t* codes, float* scales) {
  if (!ctx) return nd_fail(nullptr, ND_ERR_BACKEND, "context is NULL");
  nd_status st = check_rows(ctx, r);
  if (st != ND_OK) return st;
  if (r->count == 0) return ND_OK;
  ND_ON_DEVICE(ctx);
  ND_HIP(ctx, hipDeviceSynchronize());
  if (scales) ND_HIP(ctx, hipMemcpy(scales, r->scales, (size_t)r->count * 4, hipMemcpyDeviceToHost));
  if (codes) {
    const size_t bytes = ((size_t)r->count + 15) / 16 * 16 * r->k;
    int8_t* held = static_cast<int8_t*>(std::malloc(bytes));
    if (!held) return nd_fail(ctx, ND_ERR_NOMEM, "no memory for %zu bytes of codes", bytes);
    const hipError_t e = hipMemcpy(held, r->codes, bytes, hipMemcpyDeviceToHost);
    for (uint32_t m = 0; m < r->count && e == hipSuccess; ++m)
      for (uint32_t c = 0; c < r->k; c += 16)
        std::memcpy(codes + (size_t)m * r->k + c,
                    held + nd_tile_row(m, r->k) + (c / 64) * 1024 + (c / 16 % 4) * 256, 16);
    std::free(held);
    ND_HIP(ctx, e);
  }
  return ND_OK;
}

static nd_status check_product(nd_ctx* ctx, const nd_mat* m, uint32_t k) {
  if (!m || !ctx->mats.count(const_cast<nd_mat*>(m)))
    return nd_fail(ctx, ND_ERR_INVALID, "matrix does not belong to context");
  if (m->bits) return nd_fail(ctx, ND_ERR_INVALID, "int8 products need an int8 matrix");
  if (m->g != m->k || m->k != k)
    return nd_fail(ctx, ND_ERR_INVALID,
                   "int8 products need one scale per matrix row (g == k) and rows of the matrix's "
                   "width (matrix k=%u g=%u, rows k=%u)", m->k, m->g, k);
  return ND_OK;
}

nd_status nd_matmul_rows_d(nd_ctx* ctx, const nd_mat* m, const nd_rows* r, const float* add,
                           float* y, uint32_t ldy, void* stream) {
  if (!ctx) return nd_fail(nullptr, ND_ERR_BACKEND, "context is NULL");
  nd_status st = check_rows(ctx, r);
  if (st == ND_OK) st = check_product(ctx, m, r->k);
  if (st != ND_OK) return st;
  if (ldy == 0) ldy = m->n;
  if (ldy < m->n) return nd_fail(ctx, ND_ERR_INVALID, "row stride %u of %u outputs", ldy, m->n);
  if (r->count == 0) return ND_OK;
  if (!y || (reinterpret_cast<uintptr_t>(y) & 3) || (reinterpret_cast<uintptr_t>(add) & 3))
    return nd_fail(ctx, ND_ERR_INVALID, "y and add must be aligned device pointers");
  const bool across =
      ((m->n | ldy) & 3) != 0 ||
      ((reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(add)) & 15) != 0;
  const Product p{m->wt ? m->wt : m->w, m->scales, r->codes, r->scales, add,    y,
                  r->count,             m->n,      m->k,     ldy,       !m->wt, across};
  ND_ON_DEVICE(ctx);
  ND_HIP(ctx, launch_product(p, nd_pick_stream(ctx, stream)));
  return ND_OK;
}

nd_status nd_matmul_w8a8(nd_ctx* ctx, const nd_mat* m, const float* x, uint32_t rows, float* y) {
  if (!ctx) return nd_fail(nullptr, ND_ERR_BACKEND, "context is NULL");
  nd_status st = check_product(ctx, m, m ? m->k : 0);
  if (st != ND_OK) return st;
  if (rows == 0) return ND_OK;
  if (!x || !y) return nd_fail(ctx, ND_ERR_INVALID, "x or y is NULL");
  ND_ON_DEVICE(ctx);
  nd_rows* r = nullptr;
  st = nd_rows_create(ctx, rows, m->k, &r);
  if (st != ND_OK) return st;
  const size_t xb = (size_t)rows * m->k * 4, yb = (size_t)rows * m->n * 4;
  float *dx = nullptr, *dy = nullptr;
  hipError_t e = hipMalloc(&dx, xb);
  if (e == hipSuccess) e = hipMalloc(&dy, yb);
  if (e == hipSuccess) e = hipMemcpyAsync(dx, x, xb, hipMemcpyHostToDevice, ctx->stream);
  st = e == hipSuccess ? nd_rows_quantize_d(ctx, r, dx, rows, 0, ctx->stream)
                       : nd_hip_fail(ctx, e, "nd_matmul_w8a8");
  if (st == ND_OK) st = nd_matmul_rows_d(ctx, m, r, nullptr, dy, 0, ctx->stream);
  if (st == ND_OK) {
    e = hipMemcpyAsync(y, dy, yb, hipMemcpyDeviceToHost, ctx->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
    if (e != hipSuccess) st = nd_hip_fail(ctx, e, "nd_matmul_w8a8");
  }
  hipStreamSynchronize(ctx->stream);
  hipFree(dx);
  hipFree(dy);
  nd_rows_free(ctx, r);
  return st;
}

}  // extern "C"
