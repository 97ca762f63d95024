// Grouped 8-bit muls (ruyb200_mul_grouped_async).
#include <cuda.h>

#include <cstring>

#include "async.cuh"
#include "batch_i8.h"
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

// ---- few columns per group: register-level MMAs --------------------------------------------------------
//
// Bound by the weights' bytes.  A CTA owns 16 weight rows of a group and its warps split the depth; every weight byte is
// loaded once per 8 columns, straight into MMA fragments (m16n8k32): the depth may be taken in any order as long as
// both operands take the same, so a lane's 16 consecutive bytes are its share of two MMAs.  Sums for the zero points come
// from the same registers.  Measured: two columns in two of eight groups of 4096 x 4096,
// 33.6 MB of weights, 10.9 us, of which launch, offsets and the first loads' latency are about half.
constexpr int kMmaWarps = 4;

template <bool kWSigned, bool kXSigned>
__device__ __forceinline__ void mma_16832(int32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
#define RUYB200_MMA(A, B)                                                                                             \
  asm("mma.sync.aligned.m16n8k32.row.col.s32." A "." B ".s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};" \
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])                                                                \
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1))
  if (kWSigned && kXSigned) RUYB200_MMA("s8", "s8");
  else if (kWSigned) RUYB200_MMA("s8", "u8");
  else if (kXSigned) RUYB200_MMA("u8", "s8");
  else RUYB200_MMA("u8", "u8");
#undef RUYB200_MMA
}

template <bool kSigned>
__device__ __forceinline__ int32_t add4(uint32_t v, int32_t sum) {
  return kSigned ? __dp4a((int)v, 0x01010101, sum) : (int32_t)__dp4a(v, 0x01010101u, (uint32_t)sum);
}
template <bool kSigned>
__device__ __forceinline__ int32_t add16(const uint4& v, int32_t sum) {
  return add4<kSigned>(v.w, add4<kSigned>(v.z, add4<kSigned>(v.y, add4<kSigned>(v.x, sum))));
}

// 16 bytes of a row from position k on; those at and beyond `depth` count as 0 and are not read.
__device__ __forceinline__ uint4 load_piece(const uint8_t* row, int k, int depth, bool stream) {
  if (k + 16 <= depth) return stream ? __ldcs(reinterpret_cast<const uint4*>(row + k)) : __ldg(reinterpret_cast<const uint4*>(row + k));
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 16; i++) {
    if (k + i < depth) w[i / 4] |= (uint32_t)__ldg(row + k + i) << (8 * (i % 4));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <bool kWSigned, bool kXSigned>
__global__ void __launch_bounds__(32 * kMmaWarps) grouped_i8_mma_kernel(const __grid_constant__ GroupedI8Mul m) {
  constexpr int kPart = 7;   // per lane: 4 sums, an activation sum, 2 weight sums
  __shared__ int32_t part[kMmaWarps - 1][kPart][32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, quad = lane >> 2, t = lane & 3;
  const int r0 = blockIdx.x * 16 + quad, r1 = r0 + 8;
  const bool need_w = m.zp_x != 0, need_x = m.zp_w != 0;
  int g, begin, end;
  for (int slot = blockIdx.y; nth_group(m.groups, m.cols, slot, &g, &begin, &end); slot += gridDim.y) {
    const uint8_t* const base = (const uint8_t*)m.w + (int64_t)g * m.groups.lhs_stride;
    const uint8_t* const row0 = base + (int64_t)min(r0, m.rows - 1) * m.w_stride;
    const uint8_t* const row1 = base + (int64_t)min(r1, m.rows - 1) * m.w_stride;
    for (int c0 = begin; c0 < end; c0 += 8) {
      int32_t acc[4] = {}, xsum = 0, wsum0 = 0, wsum1 = 0;
      // columns past the group's last repeat it; their sums are not stored
      const uint8_t* const xrow = (const uint8_t*)m.x + (int64_t)min(c0 + quad, end - 1) * m.x_stride;
      // a step is 256 bytes of every row: 4 pieces of 16 per lane, all loads before the first use
      for (int k0 = warp * 256; k0 < m.depth; k0 += 256 * kMmaWarps) {
        uint4 a[4], b[4], x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          a[i] = load_piece(row0, k0 + 64 * i + 16 * t, m.depth, true);
          b[i] = load_piece(row1, k0 + 64 * i + 16 * t, m.depth, true);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = load_piece(xrow, k0 + 64 * i + 16 * t, m.depth, false);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          mma_16832<kWSigned, kXSigned>(acc, a[i].x, b[i].x, a[i].y, b[i].y, x[i].x, x[i].y);
          mma_16832<kWSigned, kXSigned>(acc, a[i].z, b[i].z, a[i].w, b[i].w, x[i].z, x[i].w);
          if (need_x) xsum = add16<kXSigned>(x[i], xsum);
          if (need_w) {
            wsum0 = add16<kWSigned>(a[i], wsum0);
            wsum1 = add16<kWSigned>(b[i], wsum1);
          }
        }
      }
      if (warp > 0) {
        int32_t(*const p)[32] = part[warp - 1];
#pragma unroll
        for (int e = 0; e < 4; e++) p[e][lane] = acc[e];
        p[4][lane] = xsum;
        p[5][lane] = wsum0;
        p[6][lane] = wsum1;
      }
      __syncthreads();
      if (warp == 0) {
#pragma unroll
        for (int w = 0; w < kMmaWarps - 1; w++) {
#pragma unroll
          for (int e = 0; e < 4; e++) acc[e] += part[w][e][lane];
          xsum += part[w][4][lane];
          wsum0 += part[w][5][lane];
          wsum1 += part[w][6][lane];
        }
        // the lanes of a quad hold the quarters of each step
#pragma unroll
        for (int d = 1; d <= 2; d <<= 1) {
          xsum += __shfl_xor_sync(0xffffffffu, xsum, d);
          wsum0 += __shfl_xor_sync(0xffffffffu, wsum0, d);
          wsum1 += __shfl_xor_sync(0xffffffffu, wsum1, d);
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int r = h ? r1 : r0;
          const bool there = r < m.rows;
          const int64_t ch = (int64_t)g * m.groups.channel_stride + r;
          const int32_t bias = there && m.bias ? m.bias[ch] : 0;
          const int32_t mfp = there && m.mfp_pc ? m.mfp_pc[ch] : m.mfp;
          const int32_t mexp = there && m.mexp_pc ? m.mexp_pc[ch] : m.mexp;
          const uint32_t row_term = (uint32_t)bias - (uint32_t)m.zp_x * (uint32_t)(h ? wsum1 : wsum0) +
                                    (uint32_t)m.zp_x * (uint32_t)m.zp_w * (uint32_t)m.depth;
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const int c = c0 + 2 * t + e;
            const int32_t xs = __shfl_sync(0xffffffffu, xsum, (2 * t + e) * 4);   // the quad that summed this column
            if (there && c < end) {
              store_grouped(m, r, c,
                            finish_grouped((int32_t)((uint32_t)acc[2 * h + e] - (uint32_t)m.zp_w * (uint32_t)xs), (int32_t)row_term, mfp, mexp, m));
            }
          }
        }
      }
      __syncthreads();   // `part` may be written again
    }
  }
}

cudaError_t launch_mma(const GroupedI8Mul& m, cudaStream_t stream) {
  const dim3 grid((unsigned)((m.rows + 15) / 16), group_slots(m.groups, m.cols));
  const bool ws = m.w_dtype == RUYB200_I8, xs = m.x_dtype == RUYB200_I8;
  if (ws && xs) grouped_i8_mma_kernel<true, true><<<grid, 32 * kMmaWarps, 0, stream>>>(m);
  else if (ws) grouped_i8_mma_kernel<true, false><<<grid, 32 * kMmaWarps, 0, stream>>>(m);
  else if (xs) grouped_i8_mma_kernel<false, true><<<grid, 32 * kMmaWarps, 0, stream>>>(m);
  else grouped_i8_mma_kernel<false, false><<<grid, 32 * kMmaWarps, 0, stream>>>(m);
  return cudaGetLastError();
}

// ---- many columns per group: the 5th-generation tensor cores --------------------------------------------
//
// A persistent kernel: tiles of 128 weight rows x up to 256 columns of one group, tcgen05 kind::i8 with the weights on the
// M side and the tokens on the N side, whose width follows the group (any multiple of 16), so a group of 20 columns pays
// for 32.  Where the groups lie is only known on the device: every CTA works out the list of column tiles from the offsets
// first (a scan in shared memory), then takes every gridDim.x-th tile.  One thread loads (128 bytes of depth per stage,
// 128-byte swizzle), one warp issues the MMAs, eight warps drain the accumulators (two of them in tensor memory, so the
// next tile multiplies meanwhile) and write rows of the column-major destination, 32 lanes side by side.
//
// With enough columns two CTAs on neighbouring SMs share a tile of 256 weight rows (cta_group::2): each loads its own 128
// rows and half of the tokens, one thread issues for both.  What bounds the large case is the traffic from L2 into shared
// memory, and the pair moves 32 KB where two single CTAs move 48 KB per 128 x 256 x 128 of products.
//
// Zero points.  The sums of the weights' rows (needed for a zero point of the activations) are one more MMA of 16 columns
// against ones; the sums of the tokens (needed for one of the weights) are one more MMA of ones against the tokens, whose
// every row then holds them: each lane finds what it needs in its own row of tensor memory, and no pass over the operands
// and no workspace is needed.  Tiles are narrower then, to leave room in tensor memory.
//
// Measured: 8 x 4096 x 4096, 8192 columns 128 us (2.1 POP/s; 9 rounds of tiles of 205 columns on average, a stage of 58 KB
// per pair every 375 ns, 11.4 TB/s from L2); 64 x 1024 x 2048, 512 columns 32.6 us (4 us until the first stage is there, then
// 5.5 TB/s of weights).
constexpr int kTileM = 128;
constexpr int kTileK = 128;                 // bytes of depth per stage
constexpr int kTcWBytes = kTileM * kTileK;
constexpr int kTcOnesBytes = kTileM * kTileK;
constexpr int kTcEpilogueWarps = 8;
constexpr int kTcThreads = 64 + 32 * kTcEpilogueWarps;
constexpr int kTcAccCols = 256;             // tensor-memory columns per accumulator buffer
constexpr int kTcTokenCol = 112;            // where in them the tokens' sums are (one-CTA tiles only)
template <bool kPair>
struct TcShape {
  static constexpr int kStages = kPair ? 6 : 4;
  static constexpr int kStageBytes = kTcWBytes + (kPair ? 128 : 256) * kTileK;   // this CTA's weight and token rows
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kTcOnesBytes;
  static constexpr int kStep = kPair ? 32 : 16;                  // tile widths are multiples of this
  static constexpr int kSumCol = kTcAccCols - kStep;             // the row sums' columns
  static constexpr int kUnitM = kPair ? 2 * kTileM : kTileM;
};

struct TcGroupedArgs {
  GroupedI8Mul m;
  int64_t group_rows;   // map rows from one group's weights to the next
  int32_t tiles_m;
  int32_t cap;          // widest column tile, a multiple of 16
  int32_t k_blocks;
  uint32_t idesc;       // instruction descriptor without N
  int32_t row_sums, token_sums;
  int32_t clamp;        // the clamp is tighter than an 8-bit destination's type, or the destination is wider
  int32_t dst_words;    // 8-bit destinations: four rows of a column are an aligned word
};

// The four MMAs of 32 bytes of depth that a stage holds.  The issuing thread is alone and the tensor core's queue is short,
// so what it executes between two MMAs counts: the descriptors advance by one addition each.  `accumulate` is false for the
// first stage of a tile.
template <bool kPair>
__device__ __forceinline__ void tc_mma_stage(uint32_t tmem, uint32_t desc_a, uint32_t desc_b, uint32_t idesc, bool accumulate) {
  // 128-byte swizzled, depth-contiguous tiles: rows 128 bytes apart, groups of 8 rows 1024 bytes apart
  constexpr uint32_t kHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
  if (kPair) {
    asm volatile(
        "{\n\t.reg .pred p, t;\n\t.reg .b64 da, db;\n\t.reg .b32 la, lb;\n\t"
        "setp.ne.u32 p, %4, 0;\n\tsetp.eq.u32 t, 0, 0;\n\t"
        "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], da, db, %3, p;\n\t"
        "add.u32 la, %1, 2;\n\tadd.u32 lb, %2, 2;\n\tmov.b64 da, {la, %5};\n\tmov.b64 db, {lb, %5};\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], da, db, %3, t;\n\t"
        "add.u32 la, %1, 4;\n\tadd.u32 lb, %2, 4;\n\tmov.b64 da, {la, %5};\n\tmov.b64 db, {lb, %5};\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], da, db, %3, t;\n\t"
        "add.u32 la, %1, 6;\n\tadd.u32 lb, %2, 6;\n\tmov.b64 da, {la, %5};\n\tmov.b64 db, {lb, %5};\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], da, db, %3, t;\n\t}"
        ::"r"(tmem), "r"(desc_a), "r"(desc_b), "r"(idesc), "r"((uint32_t)accumulate), "r"(kHigh)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p, t;\n\t.reg .b64 da, db;\n\t.reg .b32 la, lb;\n\t"
        "setp.ne.u32 p, %4, 0;\n\tsetp.eq.u32 t, 0, 0;\n\t"
        "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], da, db, %3, p;\n\t"
        "add.u32 la, %1, 2;\n\tadd.u32 lb, %2, 2;\n\tmov.b64 da, {la, %5};\n\tmov.b64 db, {lb, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], da, db, %3, t;\n\t"
        "add.u32 la, %1, 4;\n\tadd.u32 lb, %2, 4;\n\tmov.b64 da, {la, %5};\n\tmov.b64 db, {lb, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], da, db, %3, t;\n\t"
        "add.u32 la, %1, 6;\n\tadd.u32 lb, %2, 6;\n\tmov.b64 da, {la, %5};\n\tmov.b64 db, {lb, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], da, db, %3, t;\n\t}"
        ::"r"(tmem), "r"(desc_a), "r"(desc_b), "r"(idesc), "r"((uint32_t)accumulate), "r"(kHigh)
        : "memory");
  }
}
__device__ __forceinline__ uint32_t tc_desc(uint32_t addr) { return ((addr & 0x3FFFF) >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t tc_width(int n) { return (uint32_t)(n >> 3) << 17; }
// Arrives on the barrier (of both CTAs of a pair) once the MMAs issued so far are done.
template <bool kPair>
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  if (kPair) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_addr(bar)),
                 "h"((uint16_t)3)
                 : "memory");
  } else {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
  }
}
// A load whose completion is signalled on a barrier of the pair's even CTA; each CTA fetches its own part.
__device__ __forceinline__ void copy_box_2d_pair(void* smem_dst, const CUtensorMap* map, int c0, int c1, uint32_t bar_of_even) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(smem_addr(smem_dst)), "l"(map), "r"(c0), "r"(c1), "r"(bar_of_even)
      : "memory");
}
__device__ __forceinline__ uint32_t addr_of_rank(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void pair_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ bool tc_elect() {
  uint32_t pred;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(pred));
  return pred != 0;
}
__device__ __forceinline__ void tc_load_32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tc_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Where a tile lies.
struct TcTile {
  int g, row0, c0, n;
};

// A group's columns are cut into the fewest tiles of at most `cap`, of about the same width.
__device__ __forceinline__ int tiles_of(int columns, int cap) { return (columns + cap - 1) / cap; }

// What the CTA has worked out from the offsets.
struct TcPlan {
  int first[kMaxGroups + 1];   // column tiles before each group
  int begin[kMaxGroups];
  int end[kMaxGroups];
};

template <bool kPair>
__device__ __forceinline__ TcTile find_tile(const TcGroupedArgs& a, const TcPlan& plan, int tile) {
  using S = TcShape<kPair>;
  const int ct = tile / a.tiles_m;
  int lo = 0, hi = a.m.groups.count - 1;   // the last group whose first tile is at or before ct
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (plan.first[mid] <= ct) lo = mid; else hi = mid - 1;
  }
  const int columns = plan.end[lo] - plan.begin[lo];
  const int count = tiles_of(columns, a.cap);
  const int width = ((columns + count - 1) / count + S::kStep - 1) / S::kStep * S::kStep;
  TcTile t;
  t.g = lo;
  t.row0 = (tile - ct * a.tiles_m) * S::kUnitM;
  t.c0 = plan.begin[lo] + (ct - plan.first[lo]) * width;
  t.n = min(width, plan.end[lo] - t.c0);
  return t;
}

// Copies of 16 token rows each for narrow tiles, of 64 for wider ones.
__device__ __forceinline__ int token_box(int n) { return n <= 48 ? 16 : 64; }

// Four values within the range of int8 or uint8, or to be saturated to it, as bytes.
__device__ __forceinline__ uint32_t narrow4(const int32_t* v, uint8_t dtype) {
  uint32_t high, all;
  if (dtype == RUYB200_U8) {
    asm("cvt.pack.sat.u8.s32.b32 %0, %1, %2, %3;" : "=r"(high) : "r"(v[3]), "r"(v[2]), "r"(0u));
    asm("cvt.pack.sat.u8.s32.b32 %0, %1, %2, %3;" : "=r"(all) : "r"(v[1]), "r"(v[0]), "r"(high));
  } else {
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(high) : "r"(v[3]), "r"(v[2]), "r"(0u));
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(all) : "r"(v[1]), "r"(v[0]), "r"(high));
  }
  return all;
}

template <int kDstBytes, bool kPair>
__global__ void __launch_bounds__(kTcThreads, 1)
grouped_i8_tc_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x16,
                     const __grid_constant__ CUtensorMap map_x64, const __grid_constant__ TcGroupedArgs a) {
  using S = TcShape<kPair>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ TcPlan plan;
  __shared__ __align__(8) uint64_t full[S::kStages], empty[S::kStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const GroupedI8Mul& m = a.m;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  uint32_t rank = 0;
  if (kPair) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int unit = kPair ? blockIdx.x / 2 : blockIdx.x, units = kPair ? gridDim.x / 2 : gridDim.x;
  uint8_t* const smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  uint8_t* const ones = smem + S::kStages * S::kStageBytes;

  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x16) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x64) : "memory");
    for (int s = 0; s < S::kStages; s++) {
      mbarrier_init(&full[s], 1);    // pair: the even CTA's, which expects both CTAs' bytes
      mbarrier_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; b++) {
      mbarrier_init(&acc_full[b], 1);
      mbarrier_init(&acc_empty[b], kTcEpilogueWarps * (kPair ? 2 : 1));
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if (kPair) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(512) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(512) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  if (a.row_sums || a.token_sums) {
    for (int i = threadIdx.x; i < kTcOnesBytes / 16; i += kTcThreads)
      reinterpret_cast<uint4*>(ones)[i] = make_uint4(0x01010101u, 0x01010101u, 0x01010101u, 0x01010101u);
  }
  for (int g = threadIdx.x; g < m.groups.count; g += kTcThreads) group_columns(m.groups, g, m.cols, &plan.begin[g], &plan.end[g]);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc_before_sync();
  __syncthreads();
  tc_after_sync();
  if (warp == 0) {
    // exclusive scan of the groups' tile counts, 32 groups at a time
    int before = 0;
    for (int g0 = 0; g0 < m.groups.count; g0 += 32) {
      const int g = g0 + lane;
      int v = g < m.groups.count ? tiles_of(plan.end[g] - plan.begin[g], a.cap) : 0;
      int sum = v;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += up;
      }
      if (g < m.groups.count) plan.first[g] = before + sum - v;
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) plan.first[m.groups.count] = before;
  }
  __syncthreads();
  if (kPair) pair_barrier();   // the partner's barriers are set up before anything signals them
  const uint32_t tmem = tmem_slot;
  const int tiles = plan.first[m.groups.count] * a.tiles_m;
  volatile int* abortp = &abort_flag;

  if (warp == 0) {
    // ---------------- loads ----------------
    if (lane == 0) {
      uint32_t s = 0, ph = 0, issued = 0;
      bool ok = true;
      const uint32_t full_of_even = kPair ? addr_of_rank(&full[0], 0) : 0;
      for (int tile = unit; tile < tiles && ok; tile += units) {
        const TcTile t = find_tile<kPair>(a, plan, tile);
        // this CTA's token rows: all, or its half of the tile's width
        const int width = (t.n + S::kStep - 1) / S::kStep * S::kStep;
        const int mine = kPair ? width / 2 : t.n, c0 = t.c0 + (kPair ? (int)rank * mine : 0);
        const int box = token_box(mine), boxes = (mine + box - 1) / box;
        const CUtensorMap* map_x = box == 16 ? &map_x16 : &map_x64;
        const int row = (int)(t.g * a.group_rows + t.row0 + rank * kTileM);
        const uint32_t bytes = (uint32_t)(kTcWBytes + boxes * box * kTileK);
        for (int kb = 0; kb < a.k_blocks; kb++) {
          if (!mbarrier_wait(&empty[s], ph ^ 1, abortp)) {
            if (!*abortp) atomicCAS(m.status, 0, 21);
            *abortp = 1;
            ok = false;
            break;
          }
          uint8_t* const sw = smem + s * S::kStageBytes;
          uint8_t* const sx = sw + kTcWBytes;
          if (kPair) {
            // only the even CTA arrives, expecting the bytes of both; its partner's may land first, which a transaction
            // count tolerates because the phase cannot complete before the one pending arrival
            const uint32_t bar = full_of_even + s * 8;
            if (rank == 0) mbarrier_expect(&full[s], 2 * bytes);
            copy_box_2d_pair(sw, &map_w, kb * kTileK, row, bar);
            for (int i = 0; i < boxes; i++) copy_box_2d_pair(sx + i * box * kTileK, map_x, kb * kTileK, c0 + i * box, bar);
          } else {
            mbarrier_expect(&full[s], bytes);
            copy_box_2d(sw, &map_w, kb * kTileK, row, &full[s]);
            for (int i = 0; i < boxes; i++) copy_box_2d(sx + i * box * kTileK, map_x, kb * kTileK, c0 + i * box, &full[s]);
          }
          issued++;
          if (++s == S::kStages) { s = 0; ph ^= 1; }
        }
      }
      if (!ok && issued > 0 && rank == 0) {
        // give copies in flight a bounded chance to land before the CTA exits
        const uint32_t last = issued - 1;
        for (uint32_t i = 0; i < kAsyncSpinLimit / 64 && !mbarrier_try(&full[last % S::kStages], (last / S::kStages) & 1); i++) __nanosleep(100);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMAs (of both CTAs of a pair): the warp stays converged, one elected lane issues ----------------
    uint32_t s = 0, ph = 0, count = 0;
    bool ok = true;
    const uint32_t desc0 = tc_desc(smem_addr(smem)), desc_ones = tc_desc(smem_addr(ones));
    for (int tile = unit; tile < tiles && ok && rank == 0; tile += units, count++) {
      const TcTile t = find_tile<kPair>(a, plan, tile);
      const uint32_t buf = count & 1;
      const int width = (t.n + S::kStep - 1) / S::kStep * S::kStep;
      ok = __all_sync(0xffffffffu, mbarrier_wait(&acc_empty[buf], ((count >> 1) & 1) ^ 1, abortp));
      tc_after_sync();
      const uint32_t acc = tmem + buf * kTcAccCols;
      const uint32_t idesc = a.idesc | tc_width(width), idesc_sums = a.idesc | tc_width(S::kStep);
      for (int kb = 0; kb < a.k_blocks && ok; kb++) {
        if (!mbarrier_try(&full[s], ph)) ok = mbarrier_wait(&full[s], ph, abortp);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_after_sync();
        const uint32_t dw = desc0 + s * (S::kStageBytes >> 4), dx = dw + (kTcWBytes >> 4);
        if (tc_elect()) {
          tc_mma_stage<kPair>(acc, dw, dx, idesc, kb != 0);
          if (a.row_sums) tc_mma_stage<kPair>(acc + S::kSumCol, dw, desc_ones, idesc_sums, kb != 0);
          if (!kPair && a.token_sums) tc_mma_stage<kPair>(acc + kTcTokenCol, desc_ones, dx, idesc, kb != 0);
          tc_commit<kPair>(&empty[s]);
          if (kb == a.k_blocks - 1) tc_commit<kPair>(&acc_full[buf]);
        }
        __syncwarp();
        if (++s == S::kStages) { s = 0; ph ^= 1; }
      }
    }
    if (!ok && lane == 0) {
      if (!*abortp) atomicCAS(m.status, 0, 22);
      *abortp = 1;
    }
  } else {
    // ---------------- epilogue ----------------
    const int quarter = warp % 4;               // the tensor-memory lanes this warp may read
    const int first_chunk = (warp - 2) / 4;     // two warps per quarter take the 32-column chunks in turn
    uint32_t count = 0;
    for (int tile = unit; tile < tiles; tile += units, count++) {
      const TcTile t = find_tile<kPair>(a, plan, tile);
      const uint32_t buf = count & 1;
      const int row_base = t.row0 + (int)rank * kTileM + quarter * 32, r = row_base + lane;
      const bool there = r < m.rows;
      const int64_t ch = (int64_t)t.g * m.groups.channel_stride + r;
      uint32_t add = there && m.bias ? (uint32_t)__ldg(m.bias + ch) : 0u;
      const int32_t mfp = there && m.mfp_pc ? __ldg(m.mfp_pc + ch) : m.mfp;
      const int32_t mexp = there && m.mexp_pc ? __ldg(m.mexp_pc + ch) : m.mexp;
      add += (uint32_t)m.zp_x * (uint32_t)m.zp_w * (uint32_t)m.depth;
      // When every shift of the warp is 32 or more, requantising is a multiply-add whose high word is shifted on, and the
      // destination's zero point rides in the rounding term where it cannot overflow there.
      const int shift = 31 - mexp;
      const bool high_word = kDstBytes != 4 && !m.rounding_x86 && __all_sync(0xffffffffu, shift >= 32 && shift <= 62);
      const bool fold_zp = shift <= 45 && m.zp_dst > -32768 && m.zp_dst < 32768;
      const long long rounding = (1ll << ((shift - 1) & 63)) + (fold_zp ? (long long)m.zp_dst * (1ll << (shift & 63)) : 0ll);
      const int32_t late_zp = fold_zp ? 0 : m.zp_dst;
      const int shift_high = (shift - 32) & 31;
      const bool ok = __all_sync(0xffffffffu, mbarrier_wait(&acc_full[buf], (count >> 1) & 1, abortp));
      if (!ok) {
        if (lane == 0) {
          if (!*abortp) atomicCAS(m.status, 0, 23);
          *abortp = 1;
        }
        break;
      }
      tc_after_sync();
      const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16) + buf * kTcAccCols;
      if (a.row_sums) {
        uint32_t sum;
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(sum) : "r"(acc + S::kSumCol) : "memory");
        tc_load_wait();
        add -= (uint32_t)m.zp_x * sum;
      }
      for (int c = 32 * first_chunk; c < t.n; c += 64) {
        uint32_t v[32];
        tc_load_32(acc + c, v);
        tc_load_wait();
        if (!kPair && a.token_sums) {
          uint32_t x[32];
          tc_load_32(acc + kTcTokenCol + c, x);
          tc_load_wait();
#pragma unroll
          for (int i = 0; i < 32; i++) v[i] -= (uint32_t)m.zp_w * x[i];
        }
        int32_t y[32];
        if (kDstBytes != 4 && high_word) {
#pragma unroll
          for (int i = 0; i < 32; i++) {
            const long long p = (long long)(int32_t)(v[i] + add) * (long long)mfp + rounding;
            y[i] = (int32_t)((uint32_t)((int32_t)(p >> 32) >> shift_high) + (uint32_t)late_zp);
            if (a.clamp) y[i] = max(min(y[i], m.clamp_max), m.clamp_min);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; i++) y[i] = finish_grouped((int32_t)v[i], (int32_t)add, mfp, mexp, m);
        }
        if (kDstBytes == 1 && a.dst_words && row_base + 32 <= m.rows) {   // uniform over the warp
          // Four lanes turn their four rows x four columns of bytes round, so that each stores four rows of one column.
          const int q = lane & 3;
          char* at = (char*)m.dst + (int64_t)(t.c0 + c + q) * m.dst_stride + row_base + (lane & ~3);
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            uint32_t w = narrow4(y + i, m.dst_dtype);
            w = __byte_perm(w, __shfl_xor_sync(0xffffffffu, w, 1), (q & 1) ? 0x3715 : 0x6240);
            w = __byte_perm(w, __shfl_xor_sync(0xffffffffu, w, 2), (q & 2) ? 0x3276 : 0x5410);
            if (c + i + q < t.n) *reinterpret_cast<uint32_t*>(at) = w;
            at += 4 * m.dst_stride;
          }
        } else if (there) {
          char* at = (char*)m.dst + ((int64_t)(t.c0 + c) * m.dst_stride + r) * kDstBytes;
#pragma unroll
          for (int i = 0; i < 32; i++) {
            if (c + i < t.n) {
              if (kDstBytes == 1) *reinterpret_cast<int8_t*>(at) = (int8_t)y[i];
              else if (kDstBytes == 2) *reinterpret_cast<int16_t*>(at) = (int16_t)y[i];
              else *reinterpret_cast<int32_t*>(at) = y[i];
            }
            at += m.dst_stride * kDstBytes;
          }
        }
      }
      tc_before_sync();
      __syncwarp();
      if (lane == 0) {
        if (kPair) {
          asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr_of_rank(&acc_empty[buf], 0)) : "memory");
        } else {
          mbarrier_arrive(&acc_empty[buf]);
        }
      }
    }
  }
  tc_before_sync();
  __syncthreads();
  if (kPair) pair_barrier();   // neither CTA frees tensor memory or exits while its partner may still signal it
  tc_after_sync();
  if (warp == 1) {
    if (kPair) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// How many pairs of CTAs the device can hold at once (the tiles are dealt out in advance, so all must run from the start).
int resident_pairs(int sm_count) {
  static std::atomic<int> cached[kMaxDevices];
  int dev = 0;
  cudaGetDevice(&dev);
  const bool known = dev >= 0 && dev < kMaxDevices;
  int n = known ? cached[dev].load(std::memory_order_relaxed) : 0;
  if (n > 0) return n;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(sm_count / 2 * 2);
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = TcShape<true>::kSmem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, grouped_i8_tc_kernel<1, true>, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    n = sm_count / 2;
  }
  n = min(n, sm_count / 2);
  if (known) cached[dev].store(n, std::memory_order_relaxed);
  return n;
}

template <int kDstBytes, bool kPair>
cudaError_t launch_tc_variant(const CUtensorMap& w, const CUtensorMap& x16, const CUtensorMap& x64, const TcGroupedArgs& a, int sm_count,
                              cudaStream_t stream) {
  static std::atomic<bool> allowed[kMaxDevices];
  const cudaError_t e = allow_smem((const void*)grouped_i8_tc_kernel<kDstBytes, kPair>, TcShape<kPair>::kSmem, allowed);
  if (e != cudaSuccess) return e;
  if (kPair) {   // the pairs' count is asked of one variant for all of them
    static std::atomic<bool> asked[kMaxDevices];
    const cudaError_t q = allow_smem((const void*)grouped_i8_tc_kernel<1, true>, TcShape<true>::kSmem, asked);
    if (q != cudaSuccess) return q;
  }
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(kPair ? 2 * resident_pairs(sm_count) : sm_count);
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = TcShape<kPair>::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kPair ? 2 : 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, grouped_i8_tc_kernel<kDstBytes, kPair>, w, x16, x64, a);
}

template <bool kPair>
cudaError_t launch_tc_by_type(const CUtensorMap& w, const CUtensorMap& x16, const CUtensorMap& x64, const TcGroupedArgs& a, int sm_count,
                              cudaStream_t stream) {
  if (a.m.dst_dtype == RUYB200_I32) return launch_tc_variant<4, kPair>(w, x16, x64, a, sm_count, stream);
  if (a.m.dst_dtype == RUYB200_I16) return launch_tc_variant<2, kPair>(w, x16, x64, a, sm_count, stream);
  return launch_tc_variant<1, kPair>(w, x16, x64, a, sm_count, stream);
}

cudaError_t launch_tc(const GroupedI8Mul& m, int sm_count, cudaStream_t stream) {
  TcGroupedArgs a;
  memset(&a, 0, sizeof(a));
  a.m = m;
  a.group_rows = m.groups.lhs_stride / m.w_stride;
  a.k_blocks = (m.depth + kTileK - 1) / kTileK;
  a.row_sums = m.zp_x != 0;
  a.token_sums = m.zp_w != 0;
  const long long active = min((long long)m.groups.count, (long long)m.cols);
  const auto column_tiles = [&](int cap) { return max(active, (m.cols + (long long)cap - 1) / cap); };
  const int pairs_m = (m.rows + 2 * kTileM - 1) / (2 * kTileM);
  // Pairs where there is a tile for each: also for few columns, since each CTA then loads half of the tokens (64 experts x
  // 1024 x 2048, 512 tokens: 32.8 us against 34.8; 8 x 4096 x 4096, 64 tokens: 30.0 against 32.7; 8192 tokens, before
  // later steps: 138 against 172).  With fewer tiles than pairs, one CTA per tile uses twice as many SMs (8 x 1024 x 1024, 256 tokens: 10.0 against
  // 12.3).
  const bool pair = !a.token_sums && m.rows > kTileM && pairs_m * column_tiles(kTcAccCols) >= sm_count / 2;
  a.tiles_m = pair ? pairs_m : (m.rows + kTileM - 1) / kTileM;
  const int step = pair ? TcShape<true>::kStep : TcShape<false>::kStep;
  a.cap = a.token_sums ? kTcTokenCol : (a.row_sums ? kTcAccCols - step : kTcAccCols);
  // narrower tiles when there are too few to go round (each reads its weights again, from L2)
  while (!pair && a.cap > 32 && a.tiles_m * column_tiles(a.cap) < sm_count) a.cap = (a.cap / 2 + 15) / 16 * 16;
  // int32 accumulation, operand signedness, both depth-contiguous, M = 128 or, of a pair, 256
  a.idesc = (2u << 4) | ((m.w_dtype == RUYB200_I8 ? 1u : 0u) << 7) | ((m.x_dtype == RUYB200_I8 ? 1u : 0u) << 10) |
            ((uint32_t)((pair ? 2 * kTileM : kTileM) >> 4) << 24);
  // the saturating narrowing of the word stores clamps to the whole type by itself
  a.dst_words = (((uintptr_t)m.dst | (uintptr_t)m.dst_stride) & 3) == 0;
  const bool whole = (m.dst_dtype == RUYB200_I8 && m.clamp_min == -128 && m.clamp_max == 127) ||
                     (m.dst_dtype == RUYB200_U8 && m.clamp_min == 0 && m.clamp_max == 255);
  a.clamp = !(whole && a.dst_words && m.rows % 32 == 0);
  CUtensorMap w, x16, x64;
  const int64_t map_rows = (m.groups.count - 1) * a.group_rows + m.rows;
  if (!make_i8_tile_map(&w, m.w, m.depth, (int)map_rows, m.w_stride, kTileM) ||
      !make_i8_tile_map(&x16, m.x, m.depth, m.cols, m.x_stride, 16) || !make_i8_tile_map(&x64, m.x, m.depth, m.cols, m.x_stride, 64))
    return cudaErrorInvalidValue;
  return pair ? launch_tc_by_type<true>(w, x16, x64, a, sm_count, stream) : launch_tc_by_type<false>(w, x16, x64, a, sm_count, stream);
}

// 16-byte aligned rows (the copy engine, and 16-byte loads), groups a whole number of rows apart; indices of 32 bits.
bool aligned_layout(const GroupedI8Mul& m) {
  if (m.depth == 0 || m.depth > (1 << 30) || m.rows > (1 << 30) || m.cols > (1 << 30)) return false;
  if ((((uintptr_t)m.w | (uintptr_t)m.x | (uintptr_t)m.w_stride | (uintptr_t)m.x_stride) & 15) != 0) return false;
  if (m.groups.lhs_stride % m.w_stride != 0) return false;
  const int64_t per = m.groups.lhs_stride / m.w_stride;
  return per <= 0x7fffffff && (m.groups.count - 1) * per + m.rows + 2 * kTileM <= 0x7fffffff;
}

}  // namespace

cudaError_t launch_grouped_i8(const GroupedI8Mul& m, int sm_count, cudaStream_t stream, int* kernel) {
  if (m.force_any || !aligned_layout(m)) {
    *kernel = RUYB200_KERNEL_GENERIC;
    return launch_any(m, stream);
  }
  const long long active = min((long long)m.groups.count, (long long)m.cols);
  // Up to three columns per group the register-level kernel is faster (8 experts x 4096 x 4096: 2 tokens 10.5 us against 16.4,
  // 16 tokens 28.4 against 29.9; 64 x 1024 x 2048, 128 tokens: 30.7 against 32.1), from four on the tensor-memory one (32
  // tokens 32.1 against 29.9; 256 tokens 33.9 against 32.4).
  if (m.cols <= 3 * active) {
    *kernel = RUYB200_KERNEL_GROUPED_MMA;
    return launch_mma(m, stream);
  }
  *kernel = RUYB200_KERNEL_GROUPED_TC;
  return launch_tc(m, sm_count, stream);
}

}  // namespace ruyb200
