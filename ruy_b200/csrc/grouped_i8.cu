// Grouped 8-bit muls (ruyb200_mul_grouped_async).
#include "grouped.h"

namespace ruyb200 {

namespace {

// ---- any layout: CUDA cores --------------------------------------------------------------------------
//
// One warp per weight row, eight columns of a group at a time: lanes stride through the depth, so the weights' row is
// read coalesced once per eight columns.  Zero points are subtracted while loading, as ReferenceMul does.
constexpr int kAnyWarps = 8;
constexpr int kAnyCols = 8;

__device__ __forceinline__ int32_t load_8bit(const void* p, uint8_t dtype, int64_t i) {
  return dtype == RUYB200_I8 ? (int32_t)((const int8_t*)p)[i] : (int32_t)((const uint8_t*)p)[i];
}

__global__ void __launch_bounds__(32 * kAnyWarps) grouped_i8_any_kernel(const GroupedI8Mul m) {
  const int lane = threadIdx.x % 32;
  const long long r = (long long)blockIdx.x * kAnyWarps + threadIdx.x / 32;
  const int g = blockIdx.y;
  int begin, end;
  group_columns(m.groups, g, m.cols, &begin, &end);
  if (r >= m.rows) return;
  const int64_t w_at = (int64_t)g * m.groups.lhs_stride + r * m.w_stride;
  const int64_t ch = (int64_t)g * m.groups.channel_stride + r;
  for (long long c0 = begin + (long long)blockIdx.z * kAnyCols; c0 < end; c0 += (long long)gridDim.z * kAnyCols) {
    const int n = (int)min((long long)kAnyCols, end - c0);
    uint32_t acc[kAnyCols] = {};
    for (long long k = lane; k < m.depth; k += 32) {
      const int32_t w = load_8bit(m.w, m.w_dtype, w_at + k) - m.zp_w;
#pragma unroll
      for (int j = 0; j < kAnyCols; j++) {
        if (j < n) acc[j] += (uint32_t)(w * (load_8bit(m.x, m.x_dtype, (c0 + j) * m.x_stride + k) - m.zp_x));
      }
    }
#pragma unroll
    for (int j = 0; j < kAnyCols; j++) {
      const uint32_t sum = __reduce_add_sync(0xffffffffu, acc[j]);
      if (lane == j && j < n) {
        store_grouped(m, (int)r, (int)c0 + j,
                      finish_grouped((int32_t)sum, m.bias ? m.bias[ch] : 0, m.mfp_pc ? m.mfp_pc[ch] : m.mfp,
                                     m.mexp_pc ? m.mexp_pc[ch] : m.mexp, m));
      }
    }
  }
}

cudaError_t launch_any(const GroupedI8Mul& m, cudaStream_t stream) {
  // the column axis of a group is also spread over the grid; its length is only known on the device
  const int z = (int)min((long long)32, ((long long)m.cols + kAnyCols - 1) / kAnyCols);
  const dim3 grid((unsigned)(((long long)m.rows + kAnyWarps - 1) / kAnyWarps), m.groups.count, z);
  grouped_i8_any_kernel<<<grid, 32 * kAnyWarps, 0, stream>>>(m);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_grouped_i8(const GroupedI8Mul& m, int sm_count, cudaStream_t stream, int* kernel) {
  (void)sm_count;
  *kernel = RUYB200_KERNEL_GENERIC;
  return launch_any(m, stream);
}

}  // namespace ruyb200
