// Muls with 4-bit weights (ruyb200_mul_q4_async, ruyb200_mul_grouped_q4_async).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstring>

#include "async.cuh"
#include "batch_i8.h"
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

// ---- the tensor-core form ----------------------------------------------------------------------------
//
//   y[r, c] = sum over blocks b of s[r, b] * sum over k in b of (q[r, k] - z[r, b]) x[k, c]
//
// The inner sums are matrix products of small whole numbers with the activations: q - z is exact in 8 bits of significand,
// so bf16 (f16 for f16 activations) holds it without rounding, the register-level MMAs (m16n8k16, 32-bit accumulators)
// form exact products, and the scale is applied to the 32-bit sums.  fp32 activations are cut into three bf16 pieces of 8
// significant bits each (24 in all: exact), which occupy three MMA columns instead of one.
//
// Bound by the weights' bytes for a few columns.  A CTA owns 128 weight rows and a part of the depth; the CTAs of a cluster
// split the depth between them and add up their sums through distributed shared memory, in a fixed order, so few rows
// still use the whole machine and no workspace is needed.  One thread keeps a ring of copy-engine loads going (a slab: 256
// depth x 128 rows, 128 bytes per row, swizzled so that the fragment loads below hit every bank once); eight warps, 16 rows
// each, widen and multiply.  The activations go through two shared-memory buffers: while one is multiplied the next part's
// are on their way in registers.  The scales of a slab are fetched two slabs ahead, one row per two lanes, and handed to
// the lanes that need them by shuffles.
//
// Measured on one B200: 16384 x 16384, one f16 column 48.4 us (138.5 MB at 2.9 TB/s); 4096 x 16384, 16 bf16 columns 25.3 us;
// 4096 x 4096, one bf16 column 8.6 us, of which 6 are launch, set-up and the cluster's barriers.  The large one is bound by
// instruction issue and the ALU pipe (45 instructions per 16 rows x 32 deep, 25 of them the arithmetic above): the same
// kernel without its arithmetic takes 28 us.
//
// Fragments.  The MMAs may take the depth in any order as long as both operands take the same.  Lane t of a quad owns
// 8 consecutive depth positions of every 32 (a step): one 32-bit word of weights holds its share for two MMAs, and masks
// pick out the pairs (0,4), (1,5), (2,6), (3,7) that end up in the halves of a register.  The activations are stored in
// shared memory in that pair order, so one 16-byte load is a lane's share of both MMAs.
constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kRows = 16 * kWarps;          // weight rows per CTA
constexpr int kSlabShift = 8;
constexpr int kSlab = 1 << kSlabShift;      // depth per ring stage
constexpr int kSteps = kSlab / 32;
constexpr int kStageBytes = kRows * kSlab / 2;
constexpr int kMaxSplit = 8;                // CTAs of a cluster that share the depth (the portable cluster size)

struct Q4Args {
  Q4Mul m;
  int64_t group_rows;   // map rows from one group's weights to the next
  int32_t x_bytes;      // shared memory for the activations of a segment
  int32_t room;         // columns per pass
  int32_t split;        // CTAs per cluster
  int32_t pass_lanes;   // CTAs that share a group's passes
  int32_t slabs_per;    // slabs of depth per CTA
  int32_t blocks;       // per row
  int32_t block_steps;  // steps per block
  int32_t block_shift;  // its logarithm, or -1 when it is no power of two
  int32_t x_vec;        // activations can be loaded 16 bytes at a time
};

enum { kHalf = 0, kBf16 = 1, kFloat3 = 2 };   // how the activations are multiplied
// ring stages: what leaves room for two CTAs per SM beside the activations
template <int kType>
constexpr int kStages = kType == kFloat3 ? 3 : 4;

template <int kType>
__device__ __forceinline__ void mma_16816(float (&c)[4], bool fresh, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  const float z0 = fresh ? 0.f : c[0], z1 = fresh ? 0.f : c[1], z2 = fresh ? 0.f : c[2], z3 = fresh ? 0.f : c[3];
  if (kType == kHalf) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(z0), "f"(z1), "f"(z2), "f"(z3));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(z0), "f"(z1), "f"(z2), "f"(z3));
  }
}

// Widening.  Masks leave a 4-bit number q in the low bits of a 16-bit half, or four bits further up, and q - z comes out of
// one multiply-add, exactly (`flip` has bit 3 of every element set for signed weights, whose z is 8 larger then):
//   f16   the significand of 1024 with q in its low bits reads as 1024 + q, four bits up as 1024 + 16 q
//   bf16  the significand of 128 with q in its low bits reads as 128 + q; four bits up there is no room, but there the bare
//         bits (a subnormal number, or one of the smallest normal ones) read as 16 q * 2**-133, which times 2**127 is q / 4.
//         The whole product is formed in quarters, and the sums are multiplied by kUnit at the end
// One shift per word serves both halves of the bytes.
template <int kType>
constexpr float kUnit = kType == kHalf ? 1.f : 4.f;

// The addends of one row: for elements from the lower and from the upper half of a byte, each twice.
template <int kType>
__device__ __forceinline__ uint32_t low_offset(int z) {
  if (kType == kHalf) {
    const __half2 v = __half2half2(__int2half_rn(-(1024 + z)));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __nv_bfloat162 v = __float2bfloat162_rn(-0.25f * (float)(128 + z));
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <int kType>
__device__ __forceinline__ uint32_t high_offset(int z) {
  if (kType == kHalf) {
    const __half2 v = __half2half2(__int2half_rn(-(64 + z)));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __nv_bfloat162 v = __float2bfloat162_rn(-0.25f * (float)z);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Eight 4-bit elements -> four pairs (0,4), (1,5), (2,6), (3,7).
template <int kType>
__device__ __forceinline__ void widen(uint32_t w, uint32_t flip, uint32_t low, uint32_t high, uint32_t (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const uint32_t u = w >> (8 * i);
    if (kType == kHalf) {
      const uint32_t a = (u & 0x000f000fu) ^ (0x64006400u | (flip & 0x000f000fu)), b = (u & 0x00f000f0u) ^ (0x64006400u | (flip & 0x00f000f0u));
      const __half2 x = __hadd2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&low));
      const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&b), __float2half2_rn(0.0625f), *reinterpret_cast<const __half2*>(&high));
      v[2 * i] = *reinterpret_cast<const uint32_t*>(&x);
      v[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&y);
    } else {
      const uint32_t a = (u & 0x000f000fu) ^ (0x43004300u | (flip & 0x000f000fu)), b = (u & 0x00f000f0u) ^ (flip & 0x00f000f0u);
      const uint32_t quarter = 0x3e803e80u, large = 0x7f007f00u;   // 1/4 and 2**127, twice
      asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(v[2 * i]) : "r"(a), "r"(quarter), "r"(low));
      asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(v[2 * i + 1]) : "r"(b), "r"(large), "r"(high));
    }
  }
}

// Eight consecutive activations of one column as they are in memory; zero beyond the depth.
template <int kType>
struct X8 {
  uint32_t v[kType == kFloat3 ? 8 : 4];
};
template <int kType>
__device__ __forceinline__ void load_x8(const Q4Args& a, int col, int k, X8<kType>& out) {
  const Q4Mul& m = a.m;
  const int64_t at = (int64_t)col * m.x_stride_c + (int64_t)k * m.x_stride_k;
  if (a.x_vec && k + 8 <= m.depth) {
    if constexpr (kType == kFloat3) {
      const uint4 p = __ldg(reinterpret_cast<const uint4*>((const float*)m.x + at));
      const uint4 q = __ldg(reinterpret_cast<const uint4*>((const float*)m.x + at) + 1);
      out.v[0] = p.x; out.v[1] = p.y; out.v[2] = p.z; out.v[3] = p.w;
      out.v[4] = q.x; out.v[5] = q.y; out.v[6] = q.z; out.v[7] = q.w;
    } else {
      const uint4 p = __ldg(reinterpret_cast<const uint4*>((const uint16_t*)m.x + at));
      out.v[0] = p.x; out.v[1] = p.y; out.v[2] = p.z; out.v[3] = p.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < (int)(sizeof(out.v) / 4); i++) {
    if (kType == kFloat3) {
      out.v[i] = k + i < m.depth ? __ldg((const uint32_t*)m.x + at + i * m.x_stride_k) : 0u;
    } else {
      const uint32_t l = k + 2 * i < m.depth ? (uint32_t)__ldg((const uint16_t*)m.x + at + 2 * i * m.x_stride_k) : 0u;
      const uint32_t h = k + 2 * i + 1 < m.depth ? (uint32_t)__ldg((const uint16_t*)m.x + at + (2 * i + 1) * m.x_stride_k) : 0u;
      out.v[i] = l | (h << 16);
    }
  }
}

// The upper 16 bits of a float are a bf16 that differs from it by less than one step, so what is left after taking them
// away is exact, and three times 8 bits are all of the significand's 24.  Infinities and NaN live in the first piece alone.
// The smallest bf16 is 2**-133: of activations below about 2**-112 the lowest bits are lost, at most 2**-133 each.
__device__ __forceinline__ void split3(uint32_t bits, uint32_t (&piece)[3]) {
  const float x = __uint_as_float(bits);
  const uint32_t h = bits & 0xffff0000u;
  if ((bits & 0x7f800000u) == 0x7f800000u) {
    piece[0] = (bits & 0x007fffffu) ? 0x7fffu : h >> 16;
    piece[1] = piece[2] = 0;
    return;
  }
  const float r1 = x - __uint_as_float(h);
  const uint32_t m = __float_as_uint(r1) & 0xffff0000u;
  const float r2 = r1 - __uint_as_float(m);
  piece[0] = h >> 16;
  piece[1] = m >> 16;
  piece[2] = __float_as_uint(r2) >> 16;
}

// The activations of a segment (some slabs of depth of all columns of the pass) on their way into shared memory: one row of
// `pitch` bytes per MMA column (pieces of fp32 columns: all first pieces, all second ones, all third ones), every eight
// positions in pair order.  Each thread carries kItems pieces of eight, so a segment is at most kSlabColumns slabs times
// columns.
template <int kType>
struct Carried {
  static constexpr int kItems = kType == kFloat3 ? 2 : 4;
  static constexpr int kSlabColumns = kItems * kThreads / (kSlab / 8);
  X8<kType> x[kItems];

  // A segment of 1 << shift slabs from depth k0 on; what lies at or beyond `end` (whole slabs) is left out.
  __device__ __forceinline__ void load(const Q4Args& a, int shift, int c0, int n, int k0, int end) {
    const int lg = shift + kSlabShift - 3;
#pragma unroll
    for (int u = 0; u < kItems; u++) {
      const int i = threadIdx.x + u * kThreads;
      const int c = i >> lg, k = k0 + 8 * (i - (c << lg));
      if (c < n && k < end) load_x8<kType>(a, c0 + c, k, x[u]);
    }
  }

  __device__ __forceinline__ void store(uint8_t* xs, int pitch, int shift, int n) const {
    const int lg = shift + kSlabShift - 3;
#pragma unroll
    for (int u = 0; u < kItems; u++) {
      const int i = threadIdx.x + u * kThreads;
      const int c = i >> lg, p = i - (c << lg);
      if (c >= n) break;
      uint8_t* const to = xs + c * pitch + 16 * p;
      const uint32_t (&v)[sizeof(x[u].v) / 4] = x[u].v;
      if constexpr (kType == kFloat3) {
        uint32_t w[3][8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          uint32_t piece[3];
          split3(v[e], piece);
#pragma unroll
          for (int s = 0; s < 3; s++) w[s][e] = piece[s];
        }
#pragma unroll
        for (int s = 0; s < 3; s++) {
          *reinterpret_cast<uint4*>(to + s * n * pitch) =
              make_uint4(w[s][0] | (w[s][4] << 16), w[s][1] | (w[s][5] << 16), w[s][2] | (w[s][6] << 16), w[s][3] | (w[s][7] << 16));
        }
      } else {
        *reinterpret_cast<uint4*>(to) = make_uint4(__byte_perm(v[0], v[2], 0x5410), __byte_perm(v[0], v[2], 0x7632),
                                                   __byte_perm(v[1], v[3], 0x5410), __byte_perm(v[1], v[3], 0x7632));
      }
    }
  }
};

// Scales and zero points of a warp's 16 rows for one slab, as fetched: lanes 2 r and 2 r + 1 hold row r's for the first
// and the second half of the slab, kPer of them (kFlush = 4 / kPer steps each).
template <int kPer>
struct SlabScales {
  uint32_t scale[kPer];
  int8_t zero[kPer];
};

template <int kPer>
__device__ __forceinline__ void fetch_scales(const Q4Args& a, int64_t row_at, bool row_there, int slab, SlabScales<kPer>& out) {
  const Q4Mul& m = a.m;
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const int step = slab * kSteps + (threadIdx.x & 1) * (kSteps / 2) + i * (4 / kPer);
    const int b = a.block_shift >= 0 ? step >> a.block_shift : step / a.block_steps;
    out.scale[i] = 0;
    out.zero[i] = 0;
    if (row_there && b < a.blocks) {
      out.scale[i] = m.scale_dtype == RUYB200_F32 ? __ldg((const uint32_t*)m.scales + row_at + b)
                                                  : (uint32_t)__ldg((const uint16_t*)m.scales + row_at + b);
      if (m.zero_points) out.zero[i] = __ldg(m.zero_points + row_at + b);
    }
  }
}

__device__ __forceinline__ float scale_value(const Q4Mul& m, uint32_t raw) {
  if (m.scale_dtype == RUYB200_F32) return __uint_as_float(raw);
  if (m.scale_dtype == RUYB200_BF16) return __uint_as_float(raw << 16);
  return __half2float(__ushort_as_half((unsigned short)raw));
}

// Loads by shared-memory address; volatile, so that they stay behind the waits that precede them.
__device__ __forceinline__ uint32_t load_shared(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint4 load_shared4(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

// The ring of slabs.  Warp 0 refills it between its own multiplications, one slab behind the consumption so that the
// other warps need not keep exact step with it.
struct Ring {
  uint64_t* full;
  uint64_t* empty;
  uint8_t* data;
  const CUtensorMap* map;
  int row;                        // map row of the CTA's first weight row
  uint32_t stage, phase;          // next to multiply
  uint32_t fill_stage, fill_phase;   // next to fill
  bool ok;                        // no wait has given up
};

__device__ __forceinline__ void ring_gave_up(const Q4Args& a, Ring& ring, int code, volatile int* abort_flag) {
  if (!*abort_flag) atomicCAS(a.m.status, 0, code);
  *abort_flag = 1;
  ring.ok = false;
}

// One thread: the load of a slab into the next stage, once its former content has been used.
template <int kStagesOf>
__device__ __forceinline__ void ring_fill(const Q4Args& a, Ring& ring, int slab, volatile int* abort_flag) {
  if (!mbarrier_wait(&ring.empty[ring.fill_stage], ring.fill_phase ^ 1, abort_flag)) {
    ring_gave_up(a, ring, 12, abort_flag);
    return;
  }
  mbarrier_expect(&ring.full[ring.fill_stage], kStageBytes);
  copy_box_2d(ring.data + ring.fill_stage * kStageBytes, ring.map, slab * (kSlab / 2), ring.row, &ring.full[ring.fill_stage]);
  if (++ring.fill_stage == kStagesOf) {
    ring.fill_stage = 0;
    ring.fill_phase ^= 1;
  }
}

// One pass over the CTA's part of the depth for n columns from c0 on; leaves the sums in `part` ([MMA column][row]).
// After a wait that gave up the remaining barriers are still passed, without work in between.
template <int kType, int kPer, int kTiles>
__device__ __forceinline__ void multiply_pass(const Q4Args& a, Ring& ring, uint8_t* xs, float* part, int g, int row0, int c0, int n,
                                              int slab0, int slab1, volatile int* abort_flag) {
  constexpr int kPieces = kType == kFloat3 ? 3 : 1;
  constexpr int kFlush = 4 / kPer;                // steps per partial sum
  constexpr int kChains = kTiles == 1 ? 2 : 1;    // independent accumulators, so that an MMA need not wait for the last one
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, t = lane & 3, quad = lane >> 2;
  const int used = n * kPieces;
  const int seg_shift = 31 - __clz(Carried<kType>::kSlabColumns / n);   // slabs per segment: as many as fit, a power of two
  const int seg_slabs = 1 << seg_shift;
  const int pitch = seg_slabs * kSlab * 2 + 64;   // 64 modulo 128: a quarter-warp's fragment loads hit every bank once
  const uint32_t flip = a.m.w_signed ? 0x88888888u : 0u;
  const int base_z = a.m.w_signed ? 8 : 0;
  // MMA columns are independent of one another: those without an activation multiply column 0 again and are not stored
  uint32_t xat[kTiles];
#pragma unroll
  for (int j = 0; j < kTiles; j++) xat[j] = smem_addr(xs) + (uint32_t)((8 * j + quad < used ? 8 * j + quad : 0) * pitch + 16 * t);
  // row `quad` of the warp's 16 in the first stage; the swizzle puts the 16 bytes of step b at b ^ (row % 8)
  const uint32_t wat = smem_addr(ring.data) + (uint32_t)((warp * 16 + quad) * 128 + (quad << 4) + 4 * t);
  // where this lane fetches scales, and from which lanes it takes those of its rows `quad` and `quad` + 8
  const int my_row = row0 + warp * 16 + (lane >> 1);
  const bool row_there = my_row < a.m.rows;
  const int64_t row_at = (int64_t)g * a.m.groups.scale_stride + my_row * a.m.scale_row;
  const int from0 = 2 * quad, from1 = from0 + 16;
  float total[kTiles][4], acc[kChains][kTiles][4];
#pragma unroll
  for (int j = 0; j < kTiles; j++) {
#pragma unroll
    for (int e = 0; e < 4; e++) total[j][e] = 0.f;
  }
  int fill = slab0;                               // next slab to load
  if (threadIdx.x == 0) {
    for (; fill < min(slab0 + kStages<kType>, slab1) && ring.ok; fill++) ring_fill<kStages<kType>>(a, ring, fill, abort_flag);
  }
  __syncwarp();
  SlabScales<kPer> next[2];
  fetch_scales<kPer>(a, row_at, row_there && slab0 < slab1, slab0, next[0]);
  fetch_scales<kPer>(a, row_at, row_there && slab0 + 1 < slab1, slab0 + 1, next[1]);
  Carried<kType> carried;
  carried.load(a, seg_shift, c0, n, slab0 * kSlab, slab1 * kSlab);
  uint32_t low[kPer], high[kPer];
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    low[i] = low_offset<kType>(base_z);
    high[i] = high_offset<kType>(base_z);
  }
  int buffer = 0;
  for (int s0 = slab0; s0 < slab1; s0 += seg_slabs, buffer ^= 1) {
    const int count = min(seg_slabs, slab1 - s0);
    carried.store(xs + buffer * a.x_bytes, pitch, seg_shift, n);
    // one barrier per segment: whoever fills a buffer again has passed the barrier of the segment in between, which
    // every warp reaches after its last load from that buffer
    __syncthreads();
    if (s0 + seg_slabs < slab1) carried.load(a, seg_shift, c0, n, (s0 + seg_slabs) * kSlab, slab1 * kSlab);
    uint32_t xb = (uint32_t)(buffer * a.x_bytes);
    for (int s = s0; s < s0 + count; s++, xb += kSteps * 64) {
      float scale[kPer];
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        scale[i] = scale_value(a.m, next[0].scale[i]);
        if (a.m.zero_points) {
          low[i] = low_offset<kType>(base_z + next[0].zero[i]);
          high[i] = high_offset<kType>(base_z + next[0].zero[i]);
        }
      }
      next[0] = next[1];
      fetch_scales<kPer>(a, row_at, row_there && s + 2 < slab1, s + 2, next[1]);
      const bool there = ring.ok && mbarrier_wait(&ring.full[ring.stage], ring.phase, abort_flag);
      if (!__all_sync(0xffffffffu, there)) {
        ring_gave_up(a, ring, 11, abort_flag);
        break;
      }
      const uint32_t wbase = wat + ring.stage * kStageBytes;
      uint32_t l0 = low[0], l1 = low[0], h0 = high[0], h1 = high[0];
#pragma unroll
      for (int b = 0; b < kSteps; b++) {
        const int i = (b & 3) / kFlush, half = b >> 2, chain = kChains == 2 ? 1 : 0;
        if (b % kFlush == 0 && a.m.zero_points) {   // a block's zero points
          l0 = __shfl_sync(0xffffffffu, low[i], from0 + half);
          l1 = __shfl_sync(0xffffffffu, low[i], from1 + half);
          h0 = __shfl_sync(0xffffffffu, high[i], from0 + half);
          h1 = __shfl_sync(0xffffffffu, high[i], from1 + half);
        }
        const uint32_t w0 = load_shared(wbase ^ (b << 4)), w1 = load_shared((wbase ^ (b << 4)) + 1024);
        uint32_t v0[4], v1[4];
        widen<kType>(w0, flip, l0, h0, v0);
        widen<kType>(w1, flip, l1, h1, v1);
        const bool fresh = b % kFlush == 0;
#pragma unroll
        for (int j = 0; j < kTiles; j++) {
          const uint4 x = load_shared4(xat[j] + xb + b * 64);
          mma_16816<kType>(acc[0][j], fresh, v0[0], v1[0], v0[1], v1[1], x.x, x.y);
          mma_16816<kType>(acc[chain][j], fresh && chain != 0, v0[2], v1[2], v0[3], v1[3], x.z, x.w);
        }
        if (b % kFlush == kFlush - 1) {
          const float s0v = __shfl_sync(0xffffffffu, scale[i], from0 + half), s1v = __shfl_sync(0xffffffffu, scale[i], from1 + half);
#pragma unroll
          for (int j = 0; j < kTiles; j++) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const float sum = kChains == 2 ? acc[0][j][e] + acc[chain][j][e] : acc[0][j][e];
              total[j][e] = fmaf(e < 2 ? s0v : s1v, sum, total[j][e]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbarrier_arrive(&ring.empty[ring.stage]);
      if (++ring.stage == kStages<kType>) {
        ring.stage = 0;
        ring.phase ^= 1;
      }
      if (warp == 0 && s > slab0) {
        if (lane == 0 && fill < slab1) ring_fill<kStages<kType>>(a, ring, fill++, abort_flag);
        __syncwarp();
      }
    }
  }
  __syncthreads();   // `part` lies in the ring, whose slabs all warps have used by now
#pragma unroll
  for (int j = 0; j < kTiles; j++) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int row = warp * 16 + 8 * (e >> 1) + quad;
      const int col = 8 * j + 2 * t + (e & 1);
      if (col < used) part[col * kRows + row] = total[j][e];
    }
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Only meets: for reads that have returned their values.
__device__ __forceinline__ void cluster_barrier_relaxed() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

__device__ __forceinline__ float load_of_rank(const float* p, uint32_t rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

// kPer: partial sums per 128 of depth, 1, 2 or 4.  kMaxTiles: 8-column MMA tiles per pass at most.
template <int kType, int kPer, int kMaxTiles>
__global__ void __launch_bounds__(kThreads, 2) q4_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ Q4Args a) {
  constexpr int kPieces = kType == kFloat3 ? 3 : 1;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[kStages<kType>], empty[kStages<kType>];
  __shared__ int abort_flag;
  int slot = blockIdx.y, g, begin, end;
  if (!nth_group(a.m.groups, a.m.cols, slot, &g, &begin, &end)) return;   // the whole cluster has the same slot
  uint8_t* const data = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  float* const part = reinterpret_cast<float*>(data);   // between two passes, when the ring is empty
  uint8_t* const xs = data + kStages<kType> * kStageBytes;
  const int rank = a.split > 1 ? (int)cluster_rank() : 0;
  const int row0 = (int)(blockIdx.x / a.split) * kRows;
  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map) : "memory");
    for (int s = 0; s < kStages<kType>; s++) {
      mbarrier_init(&full[s], 1);
      mbarrier_init(&empty[s], kWarps);
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();
  const int slabs = (a.m.depth + kSlab - 1) / kSlab;
  const int slab0 = min(rank * a.slabs_per, slabs), slab1 = min(slab0 + a.slabs_per, slabs);
  volatile int* abortp = &abort_flag;
  Ring ring = {full, empty, data, &map, 0, 0, 0, 0, 0, true};
  for (;;) {
    ring.row = (int)(g * a.group_rows + row0);
    // a long group's passes are shared out along the grid's third axis
    for (int c0 = begin + (int)blockIdx.z * a.room; c0 < end; c0 += (int)gridDim.z * a.room) {
      const int n = min(a.room, end - c0);
      const int tiles = (n * kPieces + 7) / 8;
      if (kMaxTiles <= 2) {
        if (tiles == 1) multiply_pass<kType, kPer, 1>(a, ring, xs, part, g, row0, c0, n, slab0, slab1, abortp);
        else multiply_pass<kType, kPer, 2>(a, ring, xs, part, g, row0, c0, n, slab0, slab1, abortp);
      } else {
        if (tiles <= 2) multiply_pass<kType, kPer, 2>(a, ring, xs, part, g, row0, c0, n, slab0, slab1, abortp);
        else if (tiles <= 4) multiply_pass<kType, kPer, 4>(a, ring, xs, part, g, row0, c0, n, slab0, slab1, abortp);
        else multiply_pass<kType, kPer, kMaxTiles>(a, ring, xs, part, g, row0, c0, n, slab0, slab1, abortp);
      }
      if (a.split > 1) cluster_barrier(); else __syncthreads();
      // every CTA of the cluster finishes its share of the rows
      const int mine = (kRows + a.split - 1) / a.split;
      for (int i = threadIdx.x; i < n * mine; i += kThreads) {
        const int c = i / mine, r = rank * mine + (i - c * mine);
        if (r >= kRows) continue;
        float v = 0.f;
        for (int s = 0; s < a.split; s++) {
#pragma unroll
          for (int p = 0; p < kPieces; p++) {
            const float* at = part + (p * n + c) * kRows + r;
            v += a.split > 1 ? load_of_rank(at, s) : *at;
          }
        }
        if (row0 + r < a.m.rows) store_q4(a.m, g, row0 + r, c0 + c, v * kUnit<kType>);
      }
      // `part` may be overwritten by the copy engine, or its CTA be gone, once everybody has read it.  Neither needs this pass's
      // stores to have arrived anywhere, and waiting for them would cost microseconds, so the barrier orders nothing.
      const bool more = c0 + (int)gridDim.z * a.room < end;
      if (more) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      if (a.split > 1) cluster_barrier_relaxed();
      else if (more) __syncthreads();
      if (more) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    slot += gridDim.y;
    if (!nth_group(a.m.groups, a.m.cols, slot, &g, &begin, &end)) break;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // as between two passes
    __syncthreads();
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (abort_flag && threadIdx.x == 0) {
    // give copies in flight a bounded chance to land before the CTA exits: every stage that was filled and not waited for
    for (int s = 0; s < kStages<kType>; s++) {
      const bool wrapped = s >= (int)ring.fill_stage;
      const uint32_t parity = ring.fill_phase ^ (wrapped ? 1u : 0u);   // of the stage's last fill
      for (uint32_t i = 0; i < kAsyncSpinLimit / 64 && !mbarrier_try(&full[s], parity); i++) __nanosleep(100);
    }
  }
}

template <int kType, int kPer, int kMaxTiles>
cudaError_t launch_staged(const Q4Args& a, cudaStream_t stream) {
  const Q4Mul& m = a.m;
  CUtensorMap map;
  const int64_t map_rows = (m.groups.count - 1) * a.group_rows + m.rows;
  if (!make_i8_tile_map(&map, m.w, (m.depth + 1) / 2, (int)map_rows, m.w_stride / 2, kRows)) return cudaErrorInvalidValue;
  static_assert(kMaxTiles * 8 * kRows * 4 <= kStages<kType> * kStageBytes, "the sums of a pass fit into the ring");
  const size_t smem = 1024 + (size_t)kStages<kType> * kStageBytes + 2 * (size_t)a.x_bytes;
  static std::atomic<bool> allowed[kMaxDevices];   // smem is the same for every launch of an instantiation
  const cudaError_t e = allow_smem((const void*)q4_kernel<kType, kPer, kMaxTiles>, smem, allowed);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)(((long long)m.rows + kRows - 1) / kRows * a.split), group_slots(m.groups, m.cols), a.pass_lanes);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, q4_kernel<kType, kPer, kMaxTiles>, map, a);
}

template <int kType, int kMaxTiles>
cudaError_t launch_by_block(const Q4Args& a, cudaStream_t stream) {
  if (a.block_steps % 4 == 0) return launch_staged<kType, 1, kMaxTiles>(a, stream);
  if (a.block_steps % 2 == 0) return launch_staged<kType, 2, kMaxTiles>(a, stream);
  return launch_staged<kType, 4, kMaxTiles>(a, stream);
}

// The copy engine's needs: 16-byte aligned rows, groups a whole number of rows apart; indices of 32 bits.
bool staged_layout(const Q4Mul& m) {
  if (m.depth == 0 || m.depth > (1 << 30) || m.rows > (1 << 30) || m.cols > (1 << 30) || ((uintptr_t)m.w & 15) != 0 || m.w_stride % 32 != 0) return false;
  if (m.groups.lhs_stride % m.w_stride != 0) return false;
  const int64_t per = m.groups.lhs_stride / m.w_stride;
  if (per > 0x7fffffff) return false;
  return (m.groups.count - 1) * per + m.rows + 128 <= 0x7fffffff;
}

cudaError_t launch_tensor(const Q4Mul& m, int sm_count, cudaStream_t stream) {
  Q4Args a;
  memset(&a, 0, sizeof(a));
  a.m = m;
  a.group_rows = m.groups.lhs_stride / m.w_stride;
  a.block_steps = m.block / 32;
  a.blocks = (int)((m.depth + (long long)m.block - 1) / m.block);
  a.block_shift = -1;
  for (int i = 0; i < 26; i++) {
    if (a.block_steps == 1 << i) a.block_shift = i;
  }
  const int pieces = m.x_dtype == RUYB200_F32 ? 3 : 1;
  // Columns per pass, a whole number of MMA tiles: 16 half or 5 fp32 ones (two tiles), or 32 and 16 (four and six), whose
  // warps hold more sums and so hide less of each other's latency.  A group of about 12 columns or fewer is better served
  // by several narrow passes side by side (16 groups x 2048 x 2048, 131 columns: bf16 26 us against 36, fp32 45 against 50),
  // one of 32 by wide passes (8 x 1024 x 1024, 256 fp32 columns: 27 us against 50).
  const long long share = m.groups.offsets ? (m.cols + (long long)m.groups.count - 1) / m.groups.count : m.cols;
  const bool few = m.groups.offsets ? share <= 12 : share * pieces <= 16;
  a.room = few ? 16 / pieces : (pieces == 3 ? 16 : 32);
  const int esz = pieces == 3 ? 4 : 2;
  a.x_vec = m.x_stride_k == 1 && (((uintptr_t)m.x | (uintptr_t)(m.x_stride_c * esz)) & 15) == 0;
  const long long active = m.groups.offsets ? min((long long)m.groups.count, (long long)m.cols) : 1;
  // CTAs side by side for the passes that a group of four times the mean share would take (a CTA without a pass still has to
  // start: 45 groups x 2396 x 363, 120 columns: 40 us with eight each, 28 with one)
  a.pass_lanes = (int)min(8ll, (min((long long)m.cols, m.groups.offsets ? 4 * share : share) + a.room - 1) / a.room);
  const long long row_tiles = ((long long)m.rows + kRows - 1) / kRows * active * ((share + a.room - 1) / a.room);
  const int slabs = (int)(((long long)m.depth + kSlab - 1) / kSlab);
  // as many CTAs per cluster as still let all run at once, two per SM
  const int split = (int)max(1ll, min(min((long long)kMaxSplit, (long long)slabs), 2 * sm_count / row_tiles));
  a.split = split;
  a.slabs_per = (slabs + a.split - 1) / a.split;
  // the largest segment: its rows, and the padding between them
  const int slab_columns = pieces == 3 ? Carried<kFloat3>::kSlabColumns : Carried<kBf16>::kSlabColumns;
  a.x_bytes = pieces * (slab_columns * kSlab * 2 + a.room * 64);
  if (pieces == 3) return few ? launch_by_block<kFloat3, 2>(a, stream) : launch_by_block<kFloat3, 6>(a, stream);
  if (m.x_dtype == RUYB200_F16) return few ? launch_by_block<kHalf, 2>(a, stream) : launch_by_block<kHalf, 4>(a, stream);
  return few ? launch_by_block<kBf16, 2>(a, stream) : launch_by_block<kBf16, 4>(a, stream);
}

}  // namespace

cudaError_t launch_q4(const Q4Mul& m, int sm_count, cudaStream_t stream, int* kernel) {
  if (!m.force_any && staged_layout(m)) {
    *kernel = RUYB200_KERNEL_Q4;
    return launch_tensor(m, sm_count, stream);
  }
  *kernel = RUYB200_KERNEL_GENERIC;
  return launch_any(m, stream);
}

}  // namespace ruyb200
