// int8_rows.cu -- rows of activations to 8-bit integers with one scale a row, and back.
//
//   int8(v) of a row v[0 .. K):  m = max(max_k |v_k|, 2^-100),  scale = m / 127,
//                                code_k = rint(v_k * (127 / m))          (ties to even)
// The floor 2^-100 keeps the scale and its reciprocal normal numbers for an all-zero or a
// subnormal row; |v_k * (127 / m)| <= 127 (1 + 2^-22), so no code needs clamping.  A row
// that holds an infinity or a NaN gets scale NaN and codes 0: its products are NaN.
//
// v is the row itself (quantize), silu(gate) * up of a packed gate|up row (swiglu), or the
// weighted root-mean-square norm of x + residual (rmsnorm); everything up to the code is
// kept in fp32, and the sum x + residual is rounded once, when it is stored.
#include <math.h>

#include "sd_common.cuh"
#include "sd_internal.h"

namespace sd {

constexpr float kInt8Max = 127.f;
constexpr int kInt8MaxRow = 1 << 24;
constexpr float kInt8Floor = 7.888609052210118e-31f;  // 2^-100

template <typename T>
SD_DEV float widen(T v);
template <>
SD_DEV float widen<float>(float v) {
  return v;
}
template <>
SD_DEV float widen<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <typename T>
SD_DEV T narrow(float v);
template <>
SD_DEV float narrow<float>(float v) {
  return v;
}
template <>
SD_DEV __nv_bfloat16 narrow<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

constexpr int kWarpRows = 4;
enum RowOp { kRowQuantize = 0, kRowSwiglu = 1, kRowNorm = 2, kRowNormAdd = 3 };  // Add: with a residual

struct RowArgs {
  const void* x;
  int64_t x_stride;  // elements between rows of x (residual and summed: r_stride, s_stride)
  const void* residual;
  int64_t r_stride;
  const void* weight;
  float eps;
  void* summed;
  int64_t s_stride;
  int8_t* codes;
  int64_t c_stride;
  float* scale;
  int64_t rows;
  int32_t width;
};

// rint(y) for |y| < 2^22 in the low byte of the sum with 1.5 * 2^23 (a product and a sum, each
// rounded: the codes are those of the formula in IEEE fp32)
SD_DEV uint32_t code_of(float v, float inv) { return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.f)); }

// max that returns NaN when an operand is one (fmaxf drops it)
SD_DEV float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// silu(g) * u with the hardware exponential and reciprocal: for |g| < 16 within 2^-19 of the exact
// value, far under what decides a code; -0 where exp(-g) overflows
SD_DEV float silu_mul(float g, float u) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + fast_exp2(g * -1.4426950408889634f)));
  return g * r * u;
}

// N consecutive values (N = 1, or 16 bytes of them) as they lie in memory
template <typename T, int N>
struct Piece {
  T e[N];
};
template <typename T>
struct alignas(16) Piece<T, 16 / sizeof(T)> {
  T e[16 / sizeof(T)];
};
template <typename T, int N>
SD_DEV Piece<T, N> load_piece(const T* p) {
  return *reinterpret_cast<const Piece<T, N>*>(p);
}
template <typename T, int N>
SD_DEV void store_values(T* p, const float (&v)[N]) {
  Piece<T, N> raw;
#pragma unroll
  for (int k = 0; k < N; ++k) raw.e[k] = narrow<T>(v[k]);
  *reinterpret_cast<Piece<T, N>*>(p) = raw;
}
SD_DEV uint32_t pack_codes(const float* v, float inv) {
  const uint32_t lo = __byte_perm(code_of(v[0], inv), code_of(v[1], inv), 0x0040);
  const uint32_t hi = __byte_perm(code_of(v[2], inv), code_of(v[3], inv), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}
template <int N>
SD_DEV void store_codes(int8_t* p, const float (&v)[N], float inv) {
  if constexpr (N == 1)
    *p = static_cast<int8_t>(code_of(v[0], inv) & 0xFFu);
  else if constexpr (N == 4)
    *reinterpret_cast<uint32_t*>(p) = pack_codes(v, inv);
  else
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_codes(v, inv), pack_codes(v + 4, inv));
}

// Reductions over the G threads of a row (sum; maximum that keeps a NaN), the result in every
// thread.  `part`: one word per warp, used by one reduction only (G > 32: a row per block).
template <int G, bool SUM>
SD_DEV float row_reduce(float v, float* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = SUM ? v + w : max_nan(v, w);
  }
  if constexpr (G > 32) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[threadIdx.x & (G / 32 - 1)];
#pragma unroll
    for (int o = G / 64; o > 0; o >>= 1) {
      const float w = __shfl_xor_sync(0xffffffffu, v, o);
      v = SUM ? v + w : max_nan(v, w);
    }
  }
  return v;
}

// What is quantised, before the norm's factors, from the values x and (second half of a gate|up row,
// or the residual) y
template <int OP>
SD_DEV float row_value(float x, float y) {
  if (OP == kRowSwiglu) return silu_mul(x, y);
  return OP == kRowNormAdd ? x + y : x;
}
template <int OP>
constexpr bool kTwoInputs = OP == kRowSwiglu || OP == kRowNormAdd;
template <int OP>
constexpr bool kIsNorm = OP == kRowNorm || OP == kRowNormAdd;
template <typename T, int OP>
SD_DEV const T* second_row(const RowArgs& a, int64_t row) {
  if (OP == kRowSwiglu) return static_cast<const T*>(a.x) + row * a.x_stride + a.width;
  return static_cast<const T*>(a.residual) + row * a.r_stride;
}
SD_DEV float inv_rms_of(const RowArgs& a, float ss) {
  return __fdiv_rn(1.f, __fsqrt_rn(ss / static_cast<float>(a.width) + a.eps));
}
struct RowScale {
  float inv, scale;  // inv = 0 and scale NaN for a row that is not finite
};
SD_DEV RowScale row_scale(float m) {
  if (!(m <= 3.4028234663852886e38f)) return {0.f, __int_as_float(0x7FC00000)};
  m = fmaxf(m, kInt8Floor);
  return {__fdiv_rn(kInt8Max, m), __fdiv_rn(m, kInt8Max)};
}

// G threads a row (32: kWarpRows rows a block, no block-wide step; else a row per block), each with up
// to CH pieces of N values held in registers as fp32 between the passes: a row is read once, and
// the only waits are the reductions (two for the norm, one else).
template <typename T, int OP, int G, int N, int CH>
__global__ void __launch_bounds__(G == 32 ? 32 * kWarpRows : G) int8_rows_kernel(const RowArgs a) {
  __shared__ float part[2][G == 32 ? 1 : G / 32];
  const int t = threadIdx.x & (G - 1);
  const int64_t row = G == 32 ? static_cast<int64_t>(blockIdx.x) * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
  grid_dep_wait();  // launched programmatically: x is the preceding work's output
  grid_dep_launch();
  if (G == 32 && row >= a.rows) return;
  // every load of the row is under way before the first value is used
  const T* xr = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* yr = second_row<T, OP>(a, row);
  Piece<T, N> px[CH] = {}, py[CH] = {};
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = (t + G * c) * N;
    if (i < a.width) px[c] = load_piece<T, N>(xr + i);
    if (kTwoInputs<OP> && i < a.width) py[c] = load_piece<T, N>(yr + i);
  }
  float v[CH][N];
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int k = 0; k < N; ++k) v[c][k] = row_value<OP>(widen<T>(px[c].e[k]), widen<T>(py[c].e[k]));
  float m = 0.f;
  if constexpr (kIsNorm<OP>) {
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int k = 0; k < N; ++k) ss += v[c][k] * v[c][k];
    const float inv_rms = inv_rms_of(a, row_reduce<G, true>(ss, part[0]));
    const T* w = static_cast<const T*>(a.weight);
    T* summed = static_cast<T*>(a.summed) + row * a.s_stride;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = (t + G * c) * N;
      if (i < a.width) px[c] = load_piece<T, N>(w + i);
      if (OP == kRowNormAdd && i < a.width) store_values<T, N>(summed + i, v[c]);
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int k = 0; k < N; ++k) v[c][k] = v[c][k] * inv_rms * widen<T>(px[c].e[k]);
  }
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int k = 0; k < N; ++k) m = max_nan(m, fabsf(v[c][k]));
  const RowScale s = row_scale(row_reduce<G, false>(m, part[1]));
  if (s.inv == 0.f) {  // the same for the whole row: its codes are 0, whatever it holds
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int k = 0; k < N; ++k) v[c][k] = 0.f;
  }
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = (t + G * c) * N;
    if (i < a.width) store_codes<N>(a.codes + row * a.c_stride + i, v[c], s.inv);
  }
  if (t == 0) a.scale[row] = s.scale;
}

// Rows too long for the registers of a block: read again in each pass.
template <typename T, int OP>
__global__ void __launch_bounds__(1024) int8_long_rows_kernel(const RowArgs a) {
  __shared__ float part[2][32];
  const int64_t row = blockIdx.x;
  grid_dep_wait();
  grid_dep_launch();
  const T* xr = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* yr = second_row<T, OP>(a, row);
  const T* w = static_cast<const T*>(a.weight);
  const auto value = [&](int i) { return row_value<OP>(widen<T>(xr[i]), kTwoInputs<OP> ? widen<T>(yr[i]) : 0.f); };
  float inv_rms = 1.f, m = 0.f;
  if (kIsNorm<OP>) {
    float ss = 0.f;
    for (int i = threadIdx.x; i < a.width; i += 1024) {
      const float v = value(i);
      ss += v * v;
    }
    inv_rms = inv_rms_of(a, row_reduce<1024, true>(ss, part[0]));
  }
  for (int i = threadIdx.x; i < a.width; i += 1024) {
    float v = value(i);
    if (kIsNorm<OP>) v = v * inv_rms * widen<T>(w[i]);
    m = max_nan(m, fabsf(v));
  }
  const RowScale s = row_scale(row_reduce<1024, false>(m, part[1]));
  for (int i = threadIdx.x; i < a.width; i += 1024) {
    float v[1] = {value(i)};
    if (OP == kRowNormAdd) static_cast<T*>(a.summed)[row * a.s_stride + i] = narrow<T>(v[0]);
    if (kIsNorm<OP>) v[0] = v[0] * inv_rms * widen<T>(w[i]);
    if (s.inv == 0.f) v[0] = 0.f;
    store_codes<1>(a.codes + row * a.c_stride + i, v, s.inv);
  }
  if (threadIdx.x == 0) a.scale[row] = s.scale;
}

// code * scale: a warp per row and 1024 columns, 16 codes a lane and load where the rows allow it
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dequantize_int8_kernel(const int8_t* __restrict__ codes, int64_t c_stride,
                                                              const float* __restrict__ scale, T* __restrict__ out,
                                                              int64_t o_stride, int64_t rows, int width) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  grid_dep_wait();
  grid_dep_launch();
  if (row >= rows) return;
  const float s = scale[row];
  const int8_t* c = codes + row * c_stride;
  T* o = out + row * o_stride;
  const int begin = blockIdx.y * 1024, end = min(width, begin + 1024);
  if constexpr (VEC) {
    constexpr int kOut = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = begin + (j * 32 + lane) * 16;
      if (i >= end) break;
      const uint4 raw = *reinterpret_cast<const uint4*>(c + i);
      const int8_t* e = reinterpret_cast<const int8_t*>(&raw);
#pragma unroll
      for (int k = 0; k < 16; k += kOut) {
        float v[kOut];
#pragma unroll
        for (int q = 0; q < kOut; ++q) v[q] = static_cast<float>(e[k + q]) * s;
        store_values<T, kOut>(o + i + k, v);
      }
    }
  } else {
    for (int i = begin + lane; i < end; i += 32) o[i] = narrow<T>(static_cast<float>(c[i]) * s);
  }
}

static int check_rows(const char* what, const void* x, int64_t x_stride, int64_t need, const void* codes,
                      int64_t c_stride, const void* scale, int32_t dtype, int64_t rows, int32_t width) {
  if (rows < 0 || rows > 0x7fffffff) return fail(SPECDEC_ERR_INVALID, "%s: row count out of range", what);
  if (width <= 0) return fail(SPECDEC_ERR_INVALID, "%s: empty row", what);
  if (width > kInt8MaxRow) return fail(SPECDEC_ERR_INVALID, "%s: row longer than %d", what, kInt8MaxRow);
  if (dtype != SPECDEC_F32 && dtype != SPECDEC_BF16)
    return fail(SPECDEC_ERR_INVALID, "%s supports float32 and bfloat16", what);
  if (rows == 0) return SPECDEC_OK;
  if (!x || !codes || !scale) return fail(SPECDEC_ERR_INVALID, "%s: tensors must be CUDA", what);
  if (x_stride < need || c_stride < width)
    return fail(SPECDEC_ERR_INVALID, "%s: a row stride is smaller than its row", what);
  return SPECDEC_OK;
}

template <typename T, int OP, int G, int N, int CH>
static int launch_rows_as(const char* what, const RowArgs& a, cudaStream_t st) {
  const int64_t blocks = G == 32 ? (a.rows + kWarpRows - 1) / kWarpRows : a.rows;
  return launch_pdl(what, int8_rows_kernel<T, OP, G, N, CH>, dim3(static_cast<unsigned>(blocks)),
                    dim3(G == 32 ? 32 * kWarpRows : G), 0, st, a);
}

// Threads a row: with at least eight rows an SM a warp takes a row as long as 8 pieces of 16 bytes a
// lane hold it (no block-wide waits, the most loads in flight a thread); fewer rows are spread over a
// block each, a piece a thread, which is the shortest chain from the first load to the last store.
template <typename T, int OP>
static int launch_rows_t(const char* what, const RowArgs& a, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool many = a.rows >= 8 * device_sm_count();
  uintptr_t bits = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.residual) |
                   reinterpret_cast<uintptr_t>(a.weight) | reinterpret_cast<uintptr_t>(a.summed);
  bits |= static_cast<uintptr_t>(a.x_stride | a.r_stride | a.s_stride) * sizeof(T);
  const bool vec = bits % 16 == 0 && a.width % V == 0 &&
                   (reinterpret_cast<uintptr_t>(a.codes) | static_cast<uintptr_t>(a.c_stride)) % V == 0;
  if (vec) {
    const int need = a.width / V;
    if (many && need <= 64) return launch_rows_as<T, OP, 32, V, 2>(what, a, st);
    if (many && need <= 128) return launch_rows_as<T, OP, 32, V, 4>(what, a, st);
    if (many && need <= 192) return launch_rows_as<T, OP, 32, V, 6>(what, a, st);
    if (many && need <= 256) return launch_rows_as<T, OP, 32, V, 8>(what, a, st);
    if (many && need <= 384 && V == 4) return launch_rows_as<T, OP, 32, V, 48 / V>(what, a, st);
    if (need <= 256) return launch_rows_as<T, OP, 256, V, 1>(what, a, st);
    if (!many && need <= 1024) return launch_rows_as<T, OP, 1024, V, 1>(what, a, st);
    if (many && need <= 512) return launch_rows_as<T, OP, 128, V, 4>(what, a, st);
    if (many && need <= 640) return launch_rows_as<T, OP, 128, V, 5>(what, a, st);
    if (many && need <= 768) return launch_rows_as<T, OP, 256, V, 3>(what, a, st);
    if (many && need <= 1024) return launch_rows_as<T, OP, 256, V, 4>(what, a, st);
    if (many && need <= 1280) return launch_rows_as<T, OP, 256, V, 5>(what, a, st);
    if (many && need <= 2048) return launch_rows_as<T, OP, 256, V, 8>(what, a, st);
    if (need <= 2048) return launch_rows_as<T, OP, 1024, V, 2>(what, a, st);
    if (need <= 4096) return launch_rows_as<T, OP, 1024, V, 4>(what, a, st);
  } else {
    if (many && a.width <= 256) return launch_rows_as<T, OP, 32, 1, 8>(what, a, st);
    if (many && a.width <= 512) return launch_rows_as<T, OP, 32, 1, 16>(what, a, st);
    if (a.width <= 1024) return launch_rows_as<T, OP, 256, 1, 4>(what, a, st);
    if (a.width <= 2048) return launch_rows_as<T, OP, 256, 1, 8>(what, a, st);
    if (a.width <= 8192) return launch_rows_as<T, OP, 1024, 1, 8>(what, a, st);
    if (a.width <= 32768) return launch_rows_as<T, OP, 1024, 1, 32>(what, a, st);
  }
  return launch_pdl(what, int8_long_rows_kernel<T, OP>, dim3(static_cast<unsigned>(a.rows)), dim3(1024), 0, st, a);
}
template <int OP>
static int launch_rows(const char* what, const RowArgs& a, int32_t dtype, cudaStream_t st) {
  return dtype == SPECDEC_F32 ? launch_rows_t<float, OP>(what, a, st) : launch_rows_t<__nv_bfloat16, OP>(what, a, st);
}

template <typename T>
static int launch_dequantize(const int8_t* codes, int64_t c_stride, const float* scale, T* out, int64_t o_stride,
                             int64_t rows, int32_t width, cudaStream_t st) {
  const bool vec = (reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(out) |
                    static_cast<uintptr_t>(c_stride) | static_cast<uintptr_t>(o_stride) * sizeof(T) |
                    static_cast<uintptr_t>(width)) %
                       16 == 0;
  const dim3 grid(static_cast<unsigned>((rows + 7) / 8), static_cast<unsigned>((width + 1023) / 1024));
  return launch_pdl("dequantize_int8", vec ? dequantize_int8_kernel<T, true> : dequantize_int8_kernel<T, false>, grid,
                    dim3(256), 0, st, codes, c_stride, scale, out, o_stride, rows, width);
}

}  // namespace sd

using namespace sd;

extern "C" int specdec_quantize_int8(const void* x, int64_t x_stride, void* codes, int64_t codes_stride, float* scale,
                                     int32_t dtype, int64_t rows, int32_t width, specdec_stream_t stream) {
  if (int rc = check_rows("quantize_int8", x, x_stride, width, codes, codes_stride, scale, dtype, rows, width))
    return rc;
  if (rows == 0) return SPECDEC_OK;
  RowArgs a = {};
  a.x = x;
  a.x_stride = x_stride;
  a.codes = static_cast<int8_t*>(codes);
  a.c_stride = codes_stride;
  a.scale = scale;
  a.rows = rows;
  a.width = width;
  return launch_rows<kRowQuantize>("quantize_int8", a, dtype, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int specdec_swiglu_int8(const void* gate_up, int64_t x_stride, void* codes, int64_t codes_stride,
                                   float* scale, int32_t dtype, int64_t rows, int32_t inter, specdec_stream_t stream) {
  if (int rc = check_rows("swiglu_int8", gate_up, x_stride, 2 * static_cast<int64_t>(inter), codes, codes_stride,
                          scale, dtype, rows, inter))
    return rc;
  if (rows == 0) return SPECDEC_OK;
  RowArgs a = {};
  a.x = gate_up;
  a.x_stride = x_stride;
  a.codes = static_cast<int8_t*>(codes);
  a.c_stride = codes_stride;
  a.scale = scale;
  a.rows = rows;
  a.width = inter;
  return launch_rows<kRowSwiglu>("swiglu_int8", a, dtype, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int specdec_rmsnorm_int8(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                                    const void* weight, float eps, void* summed, int64_t summed_stride, void* codes,
                                    int64_t codes_stride, float* scale, int32_t dtype, int64_t rows, int32_t hidden,
                                    specdec_stream_t stream) {
  if (int rc = check_rows("rmsnorm_int8", x, x_stride, hidden, codes, codes_stride, scale, dtype, rows, hidden))
    return rc;
  if (rows == 0) return SPECDEC_OK;
  if (!weight) return fail(SPECDEC_ERR_INVALID, "rmsnorm_int8: tensors must be CUDA");
  if ((residual == nullptr) != (summed == nullptr))
    return fail(SPECDEC_ERR_INVALID, "rmsnorm_int8: residual and summed come together");
  if (residual && (residual_stride < hidden || summed_stride < hidden))
    return fail(SPECDEC_ERR_INVALID, "rmsnorm_int8: a row stride is smaller than its row");
  RowArgs a = {};
  a.x = x;
  a.x_stride = x_stride;
  a.residual = residual;
  a.r_stride = residual_stride;
  a.weight = weight;
  a.eps = eps;
  a.summed = summed;
  a.s_stride = summed_stride;
  a.codes = static_cast<int8_t*>(codes);
  a.c_stride = codes_stride;
  a.scale = scale;
  a.rows = rows;
  a.width = hidden;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return residual ? launch_rows<kRowNormAdd>("rmsnorm_int8", a, dtype, st)
                  : launch_rows<kRowNorm>("rmsnorm_int8", a, dtype, st);
}

extern "C" int specdec_dequantize_int8(const void* codes, int64_t codes_stride, const float* scale, void* out,
                                       int64_t out_stride, int32_t dtype, int64_t rows, int32_t width,
                                       specdec_stream_t stream) {
  if (int rc = check_rows("dequantize_int8", out, out_stride, width, codes, codes_stride, scale, dtype, rows, width))
    return rc;
  if (rows == 0) return SPECDEC_OK;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int8_t* c = static_cast<const int8_t*>(codes);
  return dtype == SPECDEC_F32
             ? launch_dequantize(c, codes_stride, scale, static_cast<float*>(out), out_stride, rows, width, st)
             : launch_dequantize(c, codes_stride, scale, static_cast<__nv_bfloat16*>(out), out_stride, rows, width, st);
}
