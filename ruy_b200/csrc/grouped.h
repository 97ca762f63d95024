// Internal declarations of the muls with weights in groups and with weights of 4 bits (grouped.cu, grouped_i8.cu, q4.cu).
#pragma once

#include <atomic>

#include "common.cuh"

namespace ruyb200 {

constexpr int kMaxGroups = 1024;

// ruyb200_groups as the kernels see it.  offsets == nullptr: one group that owns every column.
struct GroupList {
  const int32_t* offsets;
  int64_t lhs_stride;       // elements
  int64_t channel_stride;   // entries
  int64_t scale_stride;     // entries
  int32_t count;
};

// First and past-the-last column of group g.  The offsets are the caller's data and cannot be checked on the host, so
// they are brought into [0, cols] here: whatever they hold, no column outside the matrices is touched.
__device__ __forceinline__ void group_columns(const GroupList& groups, int g, int cols, int* begin, int* end) {
  if (groups.offsets == nullptr) {
    *begin = 0;
    *end = cols;
    return;
  }
  const int b = min(max(__ldg(groups.offsets + g), 0), cols);
  const int e = min(max(__ldg(groups.offsets + g + 1), 0), cols);
  *begin = b;
  *end = max(e, b);
}

// A grid's second axis has a slot for every group, or, where tokens are far fewer than groups, for every group that can have
// a column: CTAs of empty groups cost their start (60 groups x 3728 x 597 of 4 bits, 4 columns: 14.0 us with all, 9.7 with 4).
// In the second form slot n stands for the n-th group that has columns, found by a scan of the offsets, which costs about
// 1 us and is not worth it for half as many tokens as groups (64 x 1024 x 2048, 32 columns: 18.4 us against 16.8).
//
// The group of a slot; false when it has none, or an empty one.  A whole warp calls it.  More groups than slots have columns
// only when offsets decrease; callers go on to slot + gridDim.y.
__device__ __forceinline__ bool nth_group(const GroupList& groups, int cols, int slot, int* g, int* begin, int* end) {
  if (gridDim.y == (unsigned)groups.count) {
    if (slot >= groups.count) return false;
    *g = slot;
    group_columns(groups, slot, cols, begin, end);
    return *end > *begin;
  }
  const int lane = threadIdx.x & 31;
  if (slot >= groups.count) return false;
  int seen = 0;
  for (int g0 = 0; g0 < groups.count; g0 += 32) {
    int b = 0, e = 0;
    if (g0 + lane < groups.count) group_columns(groups, g0 + lane, cols, &b, &e);
    const uint32_t there = __ballot_sync(0xffffffffu, e > b);
    const int n = __popc(there);
    if (slot < seen + n) {
      const int at = __fns(there, 0, slot - seen + 1);
      *g = g0 + at;
      *begin = __shfl_sync(0xffffffffu, b, at);
      *end = __shfl_sync(0xffffffffu, e, at);
      return true;
    }
    seen += n;
  }
  return false;
}
// Slots of a launch.
inline unsigned group_slots(const GroupList& groups, int cols) {
  return (unsigned)(groups.offsets && groups.count / 4 >= cols ? cols : groups.count);
}

// A grouped 8-bit mul.  Element (r, k) of group g's weights is w[g * lhs_stride + r * w_stride + k], element (k, c) of the
// activations x[c * x_stride + k], element (r, c) of the destination dst[c * dst_stride + r].
struct GroupedI8Mul {
  const void* w;
  const void* x;
  void* dst;
  int64_t w_stride, x_stride, dst_stride;
  int32_t rows, depth, cols;
  int32_t zp_w, zp_x, zp_dst;
  int32_t mfp, mexp, clamp_min, clamp_max;
  const int32_t* bias;       // per row, or nullptr
  const int32_t* mfp_pc;     // per row, or nullptr
  const int32_t* mexp_pc;
  uint8_t w_dtype, x_dtype, dst_dtype, rounding_x86;
  uint8_t force_any;         // keep the mul on the CUDA-core kernel
  GroupList groups;
  int* status;               // receives a non-zero code when a bounded wait gives up
};
// Launches the kernel that fits and names it in *kernel (RUYB200_KERNEL_*).
cudaError_t launch_grouped_i8(const GroupedI8Mul& m, int sm_count, cudaStream_t stream, int* kernel);

// A mul with 4-bit weights: w[(g * lhs_stride + r * w_stride + k) / 2], low half for even k; activations at
// x[c * x_stride_c + k * x_stride_k], destination at dst[c * dst_stride_c + r * dst_stride_r] (elements).
struct Q4Mul {
  const void* w;
  const void* x;
  void* dst;
  int64_t w_stride, x_stride_c, x_stride_k, dst_stride_c, dst_stride_r;
  int32_t rows, depth, cols;
  const void* scales;
  const int8_t* zero_points;   // or nullptr
  int64_t scale_row;           // entries between the scales of one row and the next
  int32_t block;
  const float* bias;           // per row, or nullptr
  float clamp_min, clamp_max;
  uint8_t w_signed, x_dtype, dst_dtype, scale_dtype;
  uint8_t force_any;           // keep the mul on the CUDA-core kernel
  GroupList groups;
  int* status;
};
cudaError_t launch_q4(const Q4Mul& m, int sm_count, cudaStream_t stream, int* kernel);

// Raises a kernel's limit of dynamic shared memory, once per device and kernel (`done`, one entry per device); contexts on
// several threads may get here together, and the call may repeat.
constexpr int kMaxDevices = 64;
inline cudaError_t allow_smem(const void* kernel, size_t bytes, std::atomic<bool>* done) {
  int dev = 0;
  cudaGetDevice(&dev);
  const bool known = dev >= 0 && dev < kMaxDevices;
  if (known && done[dev].load(std::memory_order_relaxed)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess && known) done[dev].store(true, std::memory_order_relaxed);
  return e;
}

// Accumulator (zero points taken care of, bias not yet added) -> destination value before the narrowing cast.
__device__ __forceinline__ int32_t finish_grouped(int32_t acc, int32_t bias, int32_t mfp, int32_t mexp, const GroupedI8Mul& m) {
  int32_t v = (int32_t)((uint32_t)acc + (uint32_t)bias);
  if (m.dst_dtype != RUYB200_I32) {
    v = m.rounding_x86 ? requant_x86(v, mfp, mexp) : requant_reference(v, mfp, mexp);
    v = (int32_t)((uint32_t)v + (uint32_t)m.zp_dst);
    return max(min(v, m.clamp_max), m.clamp_min);
  }
  return (int32_t)((uint32_t)v + (uint32_t)m.zp_dst);
}

__device__ __forceinline__ void store_grouped(const GroupedI8Mul& m, int r, int c, int32_t v) {
  const int64_t off = (int64_t)c * m.dst_stride + r;
  switch (m.dst_dtype) {
    case RUYB200_I8: ((int8_t*)m.dst)[off] = (int8_t)v; break;
    case RUYB200_U8: ((uint8_t*)m.dst)[off] = (uint8_t)v; break;
    case RUYB200_I16: ((int16_t*)m.dst)[off] = (int16_t)v; break;
    default: ((int32_t*)m.dst)[off] = v; break;
  }
}

}  // namespace ruyb200
