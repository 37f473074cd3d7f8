// int8_linear.cu -- linear layer over 8-bit activations and weights:
//   y[r][n] = (sum_k a[r][k] w[n][k]) * a_scale[r] * w_scale[n] + bias[n]
// The integer sum is exact: |sum| <= K 127^2 < 2^31 for K <= 131072.  Scales and bias are
// applied in fp32 and the result is rounded once to the output type.
//
// One block per 64 x 64 outputs, 64 codes of K at a time through shared memory, four
// products per dot-product instruction.
#include "sd_common.cuh"
#include "sd_internal.h"

namespace sd {

constexpr int kMaxWidth = 131072;
constexpr int kMaxRows = 1 << 21;

struct LinParams {
  const int8_t* a;
  const int8_t* w;
  const float* a_scale;
  const float* w_scale;
  const float* bias;
  void* out;
  int64_t a_stride, w_stride, out_stride;
  int32_t rows, width, n;
};

// four codes of row `row` from column k on (zero past the row's end and past the last row)
SD_DEV int load4(const int8_t* p, int64_t stride, int row, int rows, int k, int width) {
  if (row >= rows || k >= width) return 0;
  const int8_t* q = p + row * stride + k;
  if (k + 4 <= width) return *reinterpret_cast<const int*>(q);
  uint32_t v = 0;
  for (int i = 0; k + i < width; ++i) v |= static_cast<uint32_t>(static_cast<uint8_t>(q[i])) << (8 * i);
  return static_cast<int>(v);
}

template <typename T>
__global__ void __launch_bounds__(256) linear_int8_kernel(const LinParams p) {
  __shared__ int sa[64][17], sw[64][17];
  const int r0 = blockIdx.y * 64, n0 = blockIdx.x * 64;
  const int tr = (threadIdx.x >> 4) * 4, tn = (threadIdx.x & 15) * 4;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < p.width; k0 += 64) {
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
      sa[i >> 4][i & 15] = load4(p.a, p.a_stride, r0 + (i >> 4), p.rows, k0 + (i & 15) * 4, p.width);
      sw[i >> 4][i & 15] = load4(p.w, p.w_stride, n0 + (i >> 4), p.n, k0 + (i & 15) * 4, p.width);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(sa[tr + i][k], sw[tn + j][k], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int r = r0 + tr + i, n = n0 + tn + j;
      if (r >= p.rows || n >= p.n) continue;
      const float y = static_cast<float>(acc[i][j]) * p.a_scale[r] * p.w_scale[n] + (p.bias ? p.bias[n] : 0.f);
      T* o = static_cast<T*>(p.out) + r * p.out_stride + n;
      if constexpr (sizeof(T) == 4)
        *o = y;
      else
        *o = __float2bfloat16_rn(y);
    }
}

}  // namespace sd

using namespace sd;

extern "C" int specdec_linear_int8(const void* a, int64_t a_stride, const float* a_scale, const void* w,
                                   int64_t w_stride, const float* w_scale, const float* bias, void* out,
                                   int64_t out_stride, int32_t out_dtype, int64_t rows, int32_t width,
                                   int32_t out_features, int32_t weight_ready, int32_t* status,
                                   specdec_stream_t stream) {
  (void)weight_ready;
  (void)status;
  if (rows < 0 || rows > kMaxRows) return fail(SPECDEC_ERR_INVALID, "linear_int8: row count out of range");
  if (width <= 0 || width > kMaxWidth)
    return fail(SPECDEC_ERR_INVALID, "linear_int8: width must be in 1 .. %d", kMaxWidth);
  if (out_features <= 0 || out_features > (1 << 24))
    return fail(SPECDEC_ERR_INVALID, "linear_int8: out_features out of range");
  if (out_dtype != SPECDEC_F32 && out_dtype != SPECDEC_BF16)
    return fail(SPECDEC_ERR_INVALID, "linear_int8 writes float32 or bfloat16");
  if (rows == 0) return SPECDEC_OK;
  if (!a || !a_scale || !w || !w_scale || !out) return fail(SPECDEC_ERR_INVALID, "linear_int8: tensors must be CUDA");
  if (a_stride < width || w_stride < width || out_stride < out_features)
    return fail(SPECDEC_ERR_INVALID, "linear_int8: a row stride is smaller than its row");
  if ((a_stride | w_stride) & 15)
    return fail(SPECDEC_ERR_INVALID, "linear_int8: the row strides of the codes must be multiples of 16");
  if ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(w)) & 15u)
    return fail(SPECDEC_ERR_INVALID, "linear_int8: the codes must be 16-byte aligned");
  LinParams p = {static_cast<const int8_t*>(a), static_cast<const int8_t*>(w), a_scale, w_scale, bias, out, a_stride,
                 w_stride, out_stride, static_cast<int32_t>(rows), width, out_features};
  const dim3 grid(static_cast<unsigned>((out_features + 63) / 64), static_cast<unsigned>((rows + 63) / 64));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (out_dtype == SPECDEC_F32)
    linear_int8_kernel<float><<<grid, 256, 0, st>>>(p);
  else
    linear_int8_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p);
  return after_launch("linear_int8_kernel");
}
