// Entry points of the muls with weights in groups and with weights of 4 bits: checks of the arguments and the
// flattening of the descriptors into what the kernels take (grouped_i8.cu, q4.cu).  No device memory is allocated and
// nothing is kept between calls.  What can be checked without a device is checked first.
#include <cuda_runtime.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "grouped.h"
#include "plan.h"

using namespace ruyb200;

namespace {

// Device memory of the context's device (or managed memory): what every pointer of these calls has to be.
bool on_device(int device, const void* p) {
  cudaPointerAttributes attr;
  if (cudaPointerGetAttributes(&attr, p) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  return attr.type == cudaMemoryTypeManaged || (attr.type == cudaMemoryTypeDevice && attr.device == device);
}

struct Pointer {
  const void* p;
  size_t align;   // of its elements
};

int check_pointers(int device, const char* call, const Pointer* list, int n) {
  char msg[160];
  for (int i = 0; i < n; i++) {
    if (!list[i].p) continue;
    if ((uintptr_t)list[i].p % list[i].align != 0) {
      snprintf(msg, sizeof(msg), "%s: a pointer is not aligned to its elements", call);
      return ctx_fail(RUYB200_ERR_INVALID, msg);
    }
    if (!on_device(device, list[i].p)) {
      snprintf(msg, sizeof(msg), "%s needs device pointers of the context's device", call);
      return ctx_fail(RUYB200_ERR_INVALID, msg);
    }
  }
  return RUYB200_OK;
}

size_t element_bytes(int dtype) {
  switch (dtype) {
    case RUYB200_I8:
    case RUYB200_U8:
      return 1;
    case RUYB200_I16:
    case RUYB200_F16:
    case RUYB200_BF16:
      return 2;
    default:
      return 4;
  }
}

int check_groups(const char* call, const ruyb200_groups* g) {
  char msg[160];
  const char* wrong = nullptr;
  if (g->count < 0 || g->count > kMaxGroups) wrong = "the number of groups is outside [0, 1024]";
  else if (g->count > 0 && !g->offsets) wrong = "null offsets";
  else if (g->lhs_stride < 0 || g->channel_stride < 0 || g->scale_stride < 0) wrong = "negative stride between groups";
  if (!wrong) return RUYB200_OK;
  snprintf(msg, sizeof(msg), "%s: %s", call, wrong);
  return ctx_fail(RUYB200_ERR_INVALID, msg);
}

GroupList group_list(const ruyb200_groups* g) {
  GroupList out;
  memset(&out, 0, sizeof(out));
  out.count = 1;
  if (g) {
    out.offsets = g->offsets;
    out.lhs_stride = g->lhs_stride;
    out.channel_stride = g->channel_stride;
    out.scale_stride = g->scale_stride;
    out.count = g->count;
  }
  return out;
}

bool is_real(int t) { return t == RUYB200_F32 || t == RUYB200_F16 || t == RUYB200_BF16; }

// What validate_desc is for ruy's own types.
int validate_q4(const ruyb200_mul_desc& d, const ruyb200_q4_scales& s) {
  if (d.lhs.dtype != RUYB200_I4 && d.lhs.dtype != RUYB200_U4)
    return ctx_fail(RUYB200_ERR_UNSUPPORTED, "4-bit mul: lhs must be RUYB200_I4 or RUYB200_U4");
  if (!is_real(d.rhs.dtype)) return ctx_fail(RUYB200_ERR_UNSUPPORTED, "4-bit mul: rhs must be F32, F16 or BF16");
  if (d.dst.dtype != RUYB200_F32 && d.dst.dtype != d.rhs.dtype)
    return ctx_fail(RUYB200_ERR_UNSUPPORTED, "4-bit mul: dst must be F32 or of the type of rhs");
  if (d.params.accum_dtype != RUYB200_F32) return ctx_fail(RUYB200_ERR_UNSUPPORTED, "4-bit mul: accumulation is in F32");
  const ruyb200_matrix* ms[3] = {&d.lhs, &d.rhs, &d.dst};
  for (const ruyb200_matrix* m : ms) {
    if (m->order > 1) return ctx_fail(RUYB200_ERR_INVALID, "4-bit mul: bad order");
    if (m->cache_policy > RUYB200_ALWAYS_CACHE) return ctx_fail(RUYB200_ERR_INVALID, "4-bit mul: bad cache policy");
    if (m->rows < 0 || m->cols < 0) return ctx_fail(RUYB200_ERR_INVALID, "4-bit mul: negative dimension");
    if (m->stride < (m->order == RUYB200_COL_MAJOR ? m->rows : m->cols))
      return ctx_fail(RUYB200_ERR_INVALID, "4-bit mul: stride below the contiguous dimension");
    if (m->rows > 0 && m->cols > 0 && !m->data) return ctx_fail(RUYB200_ERR_INVALID, "4-bit mul: null data");
    if (m->zero_point) return ctx_fail(RUYB200_ERR_INVALID, "4-bit mul: zero points belong to the scales, not to a matrix");
  }
  if (d.lhs.cols != d.rhs.rows || d.lhs.rows != d.dst.rows || d.rhs.cols != d.dst.cols)
    return ctx_fail(RUYB200_ERR_INVALID, "4-bit mul: shape mismatch");
  if (d.lhs.order != RUYB200_ROW_MAJOR) return ctx_fail(RUYB200_ERR_UNSUPPORTED, "4-bit mul: lhs must be row-major");
  if (d.lhs.stride & 1) return ctx_fail(RUYB200_ERR_INVALID, "4-bit mul: the stride of lhs must be even (rows start on bytes)");
  if (d.params.channel_dimension > 1) return ctx_fail(RUYB200_ERR_INVALID, "bad channel_dimension");
  if (d.params.bias && d.params.channel_dimension != RUYB200_CHANNEL_ROW)
    return ctx_fail(RUYB200_ERR_UNSUPPORTED, "4-bit mul: the bias runs along the rows");
  if (!is_real(s.dtype)) return ctx_fail(RUYB200_ERR_UNSUPPORTED, "4-bit mul: scales must be F32, F16 or BF16");
  if (s.block <= 0 || s.block % 32 != 0)
    return ctx_fail(RUYB200_ERR_INVALID, "4-bit mul: the block of a scale must be a positive multiple of 32");
  if (s.stride < (int)(((int64_t)d.lhs.cols + s.block - 1) / s.block))
    return ctx_fail(RUYB200_ERR_INVALID, "4-bit mul: the scales' stride is below the number of blocks of a row");
  if (d.lhs.rows > 0 && d.lhs.cols > 0 && !s.scales) return ctx_fail(RUYB200_ERR_INVALID, "4-bit mul: null scales");
  return RUYB200_OK;
}

int run_q4(ruyb200_ctx* ctx, const char* call, const ruyb200_mul_desc* desc, const ruyb200_q4_scales* scales,
           const ruyb200_groups* groups) {
  if (!desc || !scales) return ctx_fail(RUYB200_ERR_INVALID, "null descriptor");
  const ruyb200_mul_desc& d = *desc;
  int rc = validate_q4(d, *scales);
  if (rc) return rc;
  if (groups) {
    rc = check_groups(call, groups);
    if (rc) return rc;
    if (groups->lhs_stride & 1) return ctx_fail(RUYB200_ERR_INVALID, "4-bit mul: lhs_stride must be even");
  }
  if (!ctx) return ctx_fail(RUYB200_ERR_INVALID, "null context");
  if (d.dst.rows == 0 || d.dst.cols == 0 || (groups && groups->count == 0)) return RUYB200_OK;
  ScopedDevice guard(ctx_device(ctx));
  const Pointer list[] = {{d.lhs.data, 1}, {d.rhs.data, element_bytes(d.rhs.dtype)}, {d.dst.data, element_bytes(d.dst.dtype)},
                          {d.params.bias, 4}, {scales->scales, element_bytes(scales->dtype)}, {scales->zero_points, 1},
                          {groups ? groups->offsets : nullptr, 4}};
  rc = check_pointers(ctx_device(ctx), call, list, 7);
  if (rc) return rc;
  Q4Mul m;
  memset(&m, 0, sizeof(m));
  m.w = d.lhs.data;
  m.x = d.rhs.data;
  m.dst = d.dst.data;
  m.w_stride = d.lhs.stride;
  const bool rhs_col = d.rhs.order == RUYB200_COL_MAJOR, dst_col = d.dst.order == RUYB200_COL_MAJOR;
  m.x_stride_c = rhs_col ? d.rhs.stride : 1;
  m.x_stride_k = rhs_col ? 1 : d.rhs.stride;
  m.dst_stride_c = dst_col ? d.dst.stride : 1;
  m.dst_stride_r = dst_col ? 1 : d.dst.stride;
  m.rows = d.lhs.rows;
  m.depth = d.lhs.cols;
  m.cols = d.rhs.cols;
  m.scales = scales->scales;
  m.zero_points = scales->zero_points;
  m.scale_row = scales->stride;
  m.block = scales->block;
  m.bias = (const float*)d.params.bias;
  m.clamp_min = d.params.clamp_min.f;
  m.clamp_max = d.params.clamp_max.f;
  m.w_signed = d.lhs.dtype == RUYB200_I4;
  m.x_dtype = d.rhs.dtype;
  m.dst_dtype = d.dst.dtype;
  m.scale_dtype = scales->dtype;
  m.force_any = ctx_forces_generic(ctx);
  m.groups = group_list(groups);
  m.status = ctx_status_word(ctx);
  int kernel = RUYB200_KERNEL_NONE;
  const cudaError_t ce = launch_q4(m, ctx_sm_count(ctx), ctx_stream(ctx), &kernel);
  if (ce != cudaSuccess) return ctx_fail(RUYB200_ERR_CUDA, cudaGetErrorString(ce));
  ctx_count_launch(ctx, kernel);
  if (ctx_trace(ctx)) {
    fprintf(stderr, "ruy_b200: 4-bit mul %dx%dx%d groups=%d block=%d kernel=%s\n", m.rows, m.depth, m.cols, m.groups.count, m.block,
            kernel == RUYB200_KERNEL_Q4 ? "q4 (copy-engine staged, register-level MMAs)" : "generic (CUDA cores, any layout)");
  }
  return RUYB200_OK;
}

}  // namespace

extern "C" {

int ruyb200_mul_grouped_async(ruyb200_ctx* ctx, const ruyb200_mul_desc* desc, const ruyb200_groups* groups) {
  const char* call = "ruyb200_mul_grouped_async";
  if (!groups) return ctx_fail(RUYB200_ERR_INVALID, "null groups");
  int rc = ctx_validate(desc);
  if (rc) return rc;
  const ruyb200_mul_desc& d = *desc;
  if (d.params.accum_dtype != RUYB200_I32 || element_bytes(d.lhs.dtype) != 1 || element_bytes(d.rhs.dtype) != 1)
    return ctx_fail(RUYB200_ERR_UNSUPPORTED, "ruyb200_mul_grouped_async: 8-bit operands with int32 accumulation only");
  if (d.lhs.order != RUYB200_ROW_MAJOR || d.rhs.order != RUYB200_COL_MAJOR || d.dst.order != RUYB200_COL_MAJOR)
    return ctx_fail(RUYB200_ERR_UNSUPPORTED, "ruyb200_mul_grouped_async: lhs must be row-major, rhs and dst column-major");
  const bool requant = d.dst.dtype != RUYB200_I32;
  const bool per_channel = d.params.bias || (requant && d.params.multiplier_fixedpoint_perchannel);
  if (per_channel && d.params.channel_dimension != RUYB200_CHANNEL_ROW)
    return ctx_fail(RUYB200_ERR_UNSUPPORTED, "ruyb200_mul_grouped_async: per-channel buffers run along the rows");
  rc = check_groups(call, groups);
  if (rc) return rc;
  if (!ctx) return ctx_fail(RUYB200_ERR_INVALID, "null context");
  ScopedDevice guard(ctx_device(ctx));
  GroupedI8Mul m;
  memset(&m, 0, sizeof(m));
  m.rounding_x86 = (uint8_t)ctx_rounding_is_x86(ctx, d.params.rounding_mode);
  if (d.dst.rows == 0 || d.dst.cols == 0 || groups->count == 0) return RUYB200_OK;
  m.w = d.lhs.data;
  m.x = d.rhs.data;
  m.dst = d.dst.data;
  m.w_stride = d.lhs.stride;
  m.x_stride = d.rhs.stride;
  m.dst_stride = d.dst.stride;
  m.rows = d.lhs.rows;
  m.depth = d.lhs.cols;
  m.cols = d.rhs.cols;
  m.zp_w = d.lhs.zero_point;
  m.zp_x = d.rhs.zero_point;
  m.zp_dst = d.dst.zero_point;
  m.bias = (const int32_t*)d.params.bias;
  if (requant) {
    m.mfp_pc = d.params.multiplier_fixedpoint_perchannel;
    m.mexp_pc = d.params.multiplier_exponent_perchannel;
    m.mfp = d.params.multiplier_fixedpoint;
    m.mexp = d.params.multiplier_exponent;
  }
  m.clamp_min = d.params.clamp_min.i;
  m.clamp_max = d.params.clamp_max.i;
  m.w_dtype = d.lhs.dtype;
  m.x_dtype = d.rhs.dtype;
  m.dst_dtype = d.dst.dtype;
  const Pointer list[] = {{m.w, 1}, {m.x, 1}, {m.dst, element_bytes(m.dst_dtype)}, {m.bias, 4}, {m.mfp_pc, 4}, {m.mexp_pc, 4},
                          {groups->offsets, 4}};
  rc = check_pointers(ctx_device(ctx), call, list, 7);
  if (rc) return rc;
  m.force_any = ctx_forces_generic(ctx);
  m.groups = group_list(groups);
  m.status = ctx_status_word(ctx);
  int kernel = RUYB200_KERNEL_NONE;
  const cudaError_t ce = launch_grouped_i8(m, ctx_sm_count(ctx), ctx_stream(ctx), &kernel);
  if (ce != cudaSuccess) return ctx_fail(RUYB200_ERR_CUDA, cudaGetErrorString(ce));
  ctx_count_launch(ctx, kernel);
  if (ctx_trace(ctx)) {
    fprintf(stderr, "ruy_b200: grouped mul %dx%dx%d groups=%d kernel=%s, rounding=%s\n", m.rows, m.depth, m.cols, m.groups.count,
            kernel == RUYB200_KERNEL_GROUPED_TC ? "grouped_tc (tcgen05 kind::i8)"
            : kernel == RUYB200_KERNEL_GROUPED_MMA ? "grouped_mma (one pass over the weights)"
                                                   : "generic (CUDA cores, any layout)",
            m.rounding_x86 ? "x86" : "reference");
  }
  return RUYB200_OK;
}

int ruyb200_mul_q4_async(ruyb200_ctx* ctx, const ruyb200_mul_desc* desc, const ruyb200_q4_scales* scales) {
  return run_q4(ctx, "ruyb200_mul_q4_async", desc, scales, nullptr);
}

int ruyb200_mul_grouped_q4_async(ruyb200_ctx* ctx, const ruyb200_mul_desc* desc, const ruyb200_q4_scales* scales,
                                 const ruyb200_groups* groups) {
  if (!groups) return ctx_fail(RUYB200_ERR_INVALID, "null groups");
  return run_q4(ctx, "ruyb200_mul_grouped_q4_async", desc, scales, groups);
}

}  // extern "C"
