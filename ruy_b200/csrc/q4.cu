// Muls with 4-bit weights (ruyb200_mul_q4_async, ruyb200_mul_grouped_q4_async).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "grouped.h"

namespace ruyb200 {

namespace {

__device__ __forceinline__ float load_real(const void* p, uint8_t dtype, int64_t i) {
  switch (dtype) {
    case RUYB200_F16: return __half2float(((const __half*)p)[i]);
    case RUYB200_BF16: return __bfloat162float(((const __nv_bfloat16*)p)[i]);
    default: return ((const float*)p)[i];
  }
}

// Bias, clamp (a NaN stays one), rounding to the destination's type.
__device__ __forceinline__ void store_q4(const Q4Mul& m, int g, int64_t r, int64_t c, float v) {
  if (m.bias) v += m.bias[(int64_t)g * m.groups.channel_stride + r];
  if (v > m.clamp_max) v = m.clamp_max;
  if (v < m.clamp_min) v = m.clamp_min;
  const int64_t off = c * m.dst_stride_c + r * m.dst_stride_r;
  switch (m.dst_dtype) {
    case RUYB200_F16: ((__half*)m.dst)[off] = __float2half_rn(v); break;
    case RUYB200_BF16: ((__nv_bfloat16*)m.dst)[off] = __float2bfloat16_rn(v); break;
    default: ((float*)m.dst)[off] = v; break;
  }
}

// ---- any layout: CUDA cores --------------------------------------------------------------------------
//
// One warp per weight row, eight columns at a time; lanes stride through the depth.  Lane sums are compensated, so that a
// long depth costs no accuracy.
constexpr int kAnyWarps = 8;
constexpr int kAnyCols = 8;

__global__ void __launch_bounds__(32 * kAnyWarps) q4_any_kernel(const Q4Mul m) {
  const int lane = threadIdx.x % 32;
  const long long r = (long long)blockIdx.x * kAnyWarps + threadIdx.x / 32;
  const int g = blockIdx.y;
  int begin, end;
  group_columns(m.groups, g, m.cols, &begin, &end);
  if (r >= m.rows) return;
  const uint8_t* w_row = (const uint8_t*)m.w + ((int64_t)g * m.groups.lhs_stride + r * m.w_stride) / 2;
  const int64_t scale_at = (int64_t)g * m.groups.scale_stride + r * m.scale_row;
  for (long long c0 = begin + (long long)blockIdx.z * kAnyCols; c0 < end; c0 += (long long)gridDim.z * kAnyCols) {
    const int n = (int)min((long long)kAnyCols, end - c0);
    float sum[kAnyCols] = {}, comp[kAnyCols] = {};
    for (long long k = lane; k < m.depth; k += 32) {
      const uint32_t byte = w_row[k >> 1];
      int q = (k & 1) ? byte >> 4 : byte & 15;
      if (m.w_signed) q = (q ^ 8) - 8;
      const int64_t at = scale_at + k / m.block;
      if (m.zero_points) q -= m.zero_points[at];
      const float w = (float)q * load_real(m.scales, m.scale_dtype, at);
#pragma unroll
      for (int j = 0; j < kAnyCols; j++) {
        if (j < n) {
          const float y = fmaf(w, load_real(m.x, m.x_dtype, (c0 + j) * m.x_stride_c + k * m.x_stride_k), -comp[j]);
          const float t = sum[j] + y;
          // an infinite sum has no rounding error to carry on (inf - inf would turn it into a NaN)
          comp[j] = isfinite(t) ? (t - sum[j]) - y : 0.f;
          sum[j] = t;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kAnyCols; j++) {
      float v = sum[j];
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
      if (lane == 0 && j < n) store_q4(m, g, r, c0 + j, v);
    }
  }
}

cudaError_t launch_any(const Q4Mul& m, cudaStream_t stream) {
  const int z = (int)min((long long)32, ((long long)m.cols + kAnyCols - 1) / kAnyCols);
  const dim3 grid((unsigned)(((long long)m.rows + kAnyWarps - 1) / kAnyWarps), m.groups.count, z);
  q4_any_kernel<<<grid, 32 * kAnyWarps, 0, stream>>>(m);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_q4(const Q4Mul& m, int sm_count, cudaStream_t stream, int* kernel) {
  (void)sm_count;
  *kernel = RUYB200_KERNEL_GENERIC;
  return launch_any(m, stream);
}

}  // namespace ruyb200
