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

enum RowOp { kRowQuantize = 0, kRowSwiglu = 1, kRowNorm = 2 };

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

// rint(y) for |y| < 2^22 in the low byte of the sum with 1.5 * 2^23
SD_DEV int8_t code_of(float v, float inv) {
  return static_cast<int8_t>(__float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.f)) & 0xFFu);
}

// Block-wide reductions (sum; maximum that keeps a NaN), the result in every thread.
template <bool SUM>
SD_DEV float block_reduce(float v, float* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = SUM ? v + w : amax_nan(v, w);
  }
  __syncthreads();  // the previous use of `part` is over
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[0];
  for (int k = 1; k < (blockDim.x >> 5); ++k) v = SUM ? v + part[k] : amax_nan(v, part[k]);
  return v;
}

template <typename T, int OP>
SD_DEV float row_value(const RowArgs& a, int64_t row, int i) {
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const float v = widen<T>(x[i]);
  if (OP == kRowSwiglu) return v / (1.f + expf(-v)) * widen<T>(x[a.width + i]);
  if (OP == kRowNorm && a.residual)
    return v + widen<T>(static_cast<const T*>(a.residual)[row * a.r_stride + i]);
  return v;
}

template <typename T, int OP>
__global__ void __launch_bounds__(256) int8_rows_kernel(const RowArgs a) {
  __shared__ float part[8];
  const int64_t row = blockIdx.x;
  float inv_rms = 1.f;
  const T* w = static_cast<const T*>(a.weight);
  if (OP == kRowNorm) {
    float ss = 0.f;
    for (int i = threadIdx.x; i < a.width; i += blockDim.x) {
      const float v = row_value<T, OP>(a, row, i);
      ss += v * v;
    }
    ss = block_reduce<true>(ss, part);
    inv_rms = __fdiv_rn(1.f, __fsqrt_rn(ss / static_cast<float>(a.width) + a.eps));
  }
  float m = 0.f;
  for (int i = threadIdx.x; i < a.width; i += blockDim.x) {
    float v = row_value<T, OP>(a, row, i);
    if (OP == kRowNorm) v = v * inv_rms * widen<T>(w[i]);
    m = amax_nan(m, fabsf(v));
  }
  m = block_reduce<false>(m, part);
  const bool finite = m <= 3.4028234663852886e38f;  // false for NaN, too
  m = fmaxf(m, kInt8Floor);
  const float inv = __fdiv_rn(kInt8Max, m);
  for (int i = threadIdx.x; i < a.width; i += blockDim.x) {
    float v = row_value<T, OP>(a, row, i);
    if (OP == kRowNorm) {
      if (a.summed) static_cast<T*>(a.summed)[row * a.s_stride + i] = narrow<T>(v);
      v = v * inv_rms * widen<T>(w[i]);
    }
    a.codes[row * a.c_stride + i] = finite ? code_of(v, inv) : int8_t(0);
  }
  if (threadIdx.x == 0) a.scale[row] = finite ? __fdiv_rn(m, kInt8Max) : __int_as_float(0x7FC00000);
}

template <typename T>
__global__ void __launch_bounds__(256) dequantize_int8_kernel(const int8_t* __restrict__ codes, int64_t c_stride,
                                                              const float* __restrict__ scale, T* __restrict__ out,
                                                              int64_t o_stride, int width) {
  const int64_t row = blockIdx.x;
  const float s = scale[row];
  for (int i = threadIdx.x; i < width; i += blockDim.x)
    out[row * o_stride + i] = narrow<T>(static_cast<float>(codes[row * c_stride + i]) * s);
}

static int check_rows(const char* what, const void* x, int64_t x_stride, int64_t need, const void* codes,
                      int64_t c_stride, const void* scale, int32_t dtype, int64_t rows, int32_t width) {
  if (rows < 0 || rows > 0x7fffffff) return fail(SPECDEC_ERR_INVALID, "%s: row count out of range", what);
  if (width <= 0) return fail(SPECDEC_ERR_INVALID, "%s: empty row", what);
  if (dtype != SPECDEC_F32 && dtype != SPECDEC_BF16)
    return fail(SPECDEC_ERR_INVALID, "%s supports float32 and bfloat16", what);
  if (rows == 0) return SPECDEC_OK;
  if (!x || !codes || !scale) return fail(SPECDEC_ERR_INVALID, "%s: tensors must be CUDA", what);
  if (x_stride < need || c_stride < width)
    return fail(SPECDEC_ERR_INVALID, "%s: a row stride is smaller than its row", what);
  return SPECDEC_OK;
}

template <int OP>
static int launch_rows(const char* what, const RowArgs& a, int32_t dtype, cudaStream_t st) {
  if (dtype == SPECDEC_F32)
    int8_rows_kernel<float, OP><<<static_cast<unsigned>(a.rows), 256, 0, st>>>(a);
  else
    int8_rows_kernel<__nv_bfloat16, OP><<<static_cast<unsigned>(a.rows), 256, 0, st>>>(a);
  return after_launch(what);
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
  return launch_rows<kRowNorm>("rmsnorm_int8", a, dtype, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int specdec_dequantize_int8(const void* codes, int64_t codes_stride, const float* scale, void* out,
                                       int64_t out_stride, int32_t dtype, int64_t rows, int32_t width,
                                       specdec_stream_t stream) {
  if (int rc = check_rows("dequantize_int8", out, out_stride, width, codes, codes_stride, scale, dtype, rows, width))
    return rc;
  if (rows == 0) return SPECDEC_OK;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(rows);
  if (dtype == SPECDEC_F32)
    dequantize_int8_kernel<float><<<grid, 256, 0, st>>>(static_cast<const int8_t*>(codes), codes_stride, scale,
                                                        static_cast<float*>(out), out_stride, width);
  else
    dequantize_int8_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(static_cast<const int8_t*>(codes), codes_stride, scale,
                                                                static_cast<__nv_bfloat16*>(out), out_stride, width);
  return after_launch("dequantize_int8");
}
