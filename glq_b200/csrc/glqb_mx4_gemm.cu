// Products of microscaled 4-bit weights on the tensor cores (tcgen05.mma, accumulators in tensor memory).
//
// One CTA computes 128 weight rows x up to tn rows of x at a time and takes such tiles in turn; accumulators alternate, so
// that one is drained while the other fills.  A tile's sum over the values may be shared by the CTAs of a cluster (few
// tiles: decode batches, small layers): each sums its part of the values, and the parts are added in rank order through the
// cluster's shared memory.  Every wait is bounded: on expiry the status word is set, tensor memory is freed and the kernel
// returns.
#include "glqb_mx4_gemm.cuh"
#include "glqb_launch.h"
#include <cuda.h>
#include <algorithm>

namespace glqb {
namespace {

// ---- PTX ------------------------------------------------------------------------------------------
// `bar`: of this CTA, or (PAIR) its namesake in the pair's first CTA
template <bool PAIR>
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  if constexpr (PAIR) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(smem_u32(bar)));
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
                 "l"(map), "r"(x), "r"(y), "r"(at)
                 : "memory");
    return;
  }
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
               "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                 "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr)
               : "memory");
}
// 16 lanes x 32 columns as fragments of 16 x 8 values: r[4g + 0, 1] columns 8g + 2t, + 1 of row l / 4 (t = l % 4), r[4g + 2, 3] of row l / 4 + 8
__device__ __forceinline__ void tmem_ld_frag(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                 "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void stmatrix_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// A from tensor memory, B from shared memory; of a pair of CTAs: 128 rows from each one's tensor memory, half of the columns from each
// one's shared memory
template <bool PAIR>
__device__ __forceinline__ void umma16(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (PAIR)
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d), "r"(a), "l"(b),
                 "r"(idesc), "r"(accumulate)
                 : "memory");
  else
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d), "r"(a), "l"(b),
                 "r"(idesc), "r"(accumulate)
                 : "memory");
}
// arrives at the barrier (of a pair: of both CTAs) when the MMAs issued so far are done
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (PAIR)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3)
                 : "memory");
  else
    umma_commit(bar);
}
template <bool PAIR>
__device__ __forceinline__ void alloc_all(uint32_t* slot) {
  __syncwarp();                                    // (thread 0 comes from the barriers)
  if constexpr (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tmem_alloc(slot, 512);
    tmem_relinquish();
  }
}
template <bool PAIR>
__device__ __forceinline__ void dealloc_all(uint32_t taddr) {
  if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(taddr) : "memory");
  else tmem_dealloc(taddr, 512);
}
// Arrives at the first CTA's barrier, from either CTA of a pair.  What it hands over is tensor memory, which the tcgen05 fences order; a
// release of all memory at cluster scope took a thousand clocks.
template <bool PAIR>
__device__ __forceinline__ void arrive_first(uint64_t* bar) {
  if constexpr (PAIR) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(bar)));
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(a) : "memory");
  } else {
    mbar_arrive(bar);
  }
}
// both from shared memory, 4-bit, scales of blocks in tensor memory
template <int FMT, bool PAIR>
__device__ __forceinline__ void umma4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
#define GLQB_UMMA4(GROUP, KIND)                                                                                                              \
  asm volatile("{ .reg .pred p; setp.ne.b32 p, %6, 0; tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, [%4], [%5], p; }" ::"r"(d), \
               "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)                                                                   \
               : "memory")
  if constexpr (FMT == GLQB_MX4_MXFP4) {
    if constexpr (PAIR) GLQB_UMMA4("2", "mxf4.block_scale.scale_vec::2X");
    else GLQB_UMMA4("1", "mxf4.block_scale.scale_vec::2X");
  } else {
    if constexpr (PAIR) GLQB_UMMA4("2", "mxf4nvf4.block_scale.scale_vec::4X");
    else GLQB_UMMA4("1", "mxf4nvf4.block_scale.scale_vec::4X");
  }
#undef GLQB_UMMA4
}
// 512 bytes of scales (32 rows of 16) to four columns of tensor memory, the same in all four quarters; of a pair: in each CTA from its
// own shared memory
template <bool PAIR>
__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint64_t desc) {
  if constexpr (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// rows of 16 bytes, eight of them 128 bytes after the eight before, no swizzle
__device__ __forceinline__ uint64_t scale_desc(uint32_t smem_addr) {
  return (uint64_t)((smem_addr >> 4) & 0x3FFF) | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}
// fp32 accumulator, both operands K-major; `type` 0: fp16, 1: bf16
__device__ __forceinline__ uint32_t idesc16(int type, int rows, int cols) {
  return (1u << 4) | (uint32_t)type << 7 | (uint32_t)type << 10 | (uint32_t)(cols >> 3) << 17 | (uint32_t)(rows >> 4) << 24;
}
// e2m1 operands, K = 64; scales e8m0 or e4m3, `sf`: the first of a word's four bytes that an instruction takes
template <int FMT>
__device__ __forceinline__ uint32_t idesc4(int rows, int cols, uint32_t sf) {
  return sf << 4 | 1u << 7 | 1u << 10 | (uint32_t)(cols >> 3) << 17 | (FMT == GLQB_MX4_MXFP4 ? 1u << 23 : 0u) | (uint32_t)(rows >> 7) << 27 | sf << 29;
}

// ---- parts of both kernels ------------------------------------------------------------------------
struct __align__(16) Bars {     // in shared memory
  uint8_t turn[4][32 * 80];    // results on their way out, per draining warp
  uint64_t full_w[8], empty_w[8], full_x[8], empty_x[8], full_a[4], empty_a[4], acc_full[2], acc_empty[2], drain;
  uint32_t tmem;
  volatile int abort;
};

template <int FMT, typename T, bool QUANT>
__device__ __forceinline__ Mx4Factor row_factor(const Mx4Job& J, int expert, int row) {
  if constexpr (!QUANT) return mx4_row_factor<FMT, T>(J, expert, row);
  else if constexpr (FMT == GLQB_MX4_NVFP4) return Mx4Factor{J.w_scale[expert], *J.x_scale};
  else return Mx4Factor{1.0f, 1.0f};
}
// Columns of a finished accumulator to y, or (a cluster's CTA) to shared memory as [column][row].  Rows of y lie across the
// accumulator's columns: 32 rows x 32 columns come as fragments, are turned by stmatrix in the warp's shared memory (columns TURN bytes
// apart, so that eight of them are in different banks) and are stored 16 bytes per lane, the next 16 rows on their way.  (A
// 2-byte store per value took 4000 clocks per 32 columns, 24,000 per tile of 192, which is a mainloop of 4096 values; turned by 2-byte
// stores 1050.)  Other results go eight columns at a time.
constexpr int TURN = 80;
template <int FMT, bool QUANT, bool BF16>
__device__ __forceinline__ void drain_wide(const Mx4Job& J, const Mx4Walk& t, int row, uint32_t acc, int lane, uint8_t* stage, const Mx4Factor& own) {
  // factors of rows lane / 4 + 8 i
  float fa[4], fb[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    fa[i] = __shfl_sync(0xFFFFFFFFu, own.a, (lane >> 2) + 8 * i);
    fb[i] = __shfl_sync(0xFFFFFFFFu, own.b, (lane >> 2) + 8 * i);
  }
  const uint32_t put = smem_u32(stage) + (uint32_t)(((lane >> 4) * 8 + (lane & 7)) * TURN + ((lane >> 3) & 1) * 16);
  const uint8_t* get = stage + (lane >> 2) * TURN + (lane & 3) * 16;
  uint16_t* y = reinterpret_cast<uint16_t*>(J.y) + (long long)(t.row0 + (lane >> 2)) * J.y_stride + row + (lane & 3) * 8;
  auto pack = [&](uint32_t a, uint32_t b, int i) -> uint32_t {
    const float u = __uint_as_float(a) * fa[i] * fb[i], v = __uint_as_float(b) * fa[i] * fb[i];
    if constexpr (BF16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(u, v);
      return *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(u, v);
      return *reinterpret_cast<const uint32_t*>(&h);
    }
  };
  auto turn = [&](const uint32_t (&v)[16], int h) {      // rows 16 h .. 16 h + 15
#pragma unroll
    for (int g = 0; g < 4; g += 2)
      stmatrix_trans(put + (uint32_t)(g * 8 * TURN + h * 32), pack(v[4 * g], v[4 * g + 1], 2 * h), pack(v[4 * g + 2], v[4 * g + 3], 2 * h + 1),
                     pack(v[4 * g + 4], v[4 * g + 5], 2 * h), pack(v[4 * g + 6], v[4 * g + 7], 2 * h + 1));
  };
  uint32_t upper[16], lower[16];
  tmem_ld_frag(acc, upper);
#pragma unroll 1
  for (int c0 = 0; c0 < t.rows; c0 += 32) {
    tmem_ld_wait();
    tmem_ld_frag(acc + (16u << 16) + (uint32_t)c0, lower);
    __syncwarp();
    turn(upper, 0);
    tmem_ld_wait();
    if (c0 + 32 < t.rows) tmem_ld_frag(acc + (uint32_t)c0 + 32u, upper);
    turn(lower, 1);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c0 + i * 8 + (lane >> 2) < t.rows) *reinterpret_cast<uint4*>(y + (long long)(c0 + i * 8) * J.y_stride) = *reinterpret_cast<const uint4*>(get + i * 8 * TURN);
  }
}
template <int FMT, typename T, bool QUANT>
__device__ __forceinline__ void drain_tile(const Mx4Job& J, const Mx4Walk& t, int mt, const Mx4Factor& f, uint32_t acc, int quarter, int lane, uint8_t* stage, float* red) {
  const int r = quarter * 32 + lane, row = mt * MX4_ROWS + r;
  acc += (uint32_t)(quarter * 32) << 16;
  if (red) {
#pragma unroll 1
    for (int c0 = 0; c0 < t.rows; c0 += 16) {
      uint32_t v[16];
      tmem_ld16(acc + (uint32_t)c0, v);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) red[(c0 + i) * MX4_ROWS + r] = __uint_as_float(v[i]);    // (room for whole sixteens)
    }
    return;
  }
  if (J.y_wide && mt * MX4_ROWS + quarter * 32 + 32 <= J.m) {
    const int row0 = mt * MX4_ROWS + quarter * 32;
    if (J.y_dtype == GLQB_DT_BF16) drain_wide<FMT, QUANT, true>(J, t, row0, acc, lane, stage, f);
    else drain_wide<FMT, QUANT, false>(J, t, row0, acc, lane, stage, f);
    return;
  }
#pragma unroll 1
  for (int c0 = 0; c0 < t.rows; c0 += 8) {
    uint32_t v[8];
    tmem_ld8(acc + (uint32_t)c0, v);
    tmem_ld_wait();
    if (row < J.m) {
      const long long at = (long long)(t.row0 + c0) * J.y_stride + row;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + i < t.rows) mx4_put(J, at + i * J.y_stride, __uint_as_float(v[i]) * f.a * f.b);
    }
    __syncwarp();                                  // (the next load is the whole warp's)
  }
}
// The cluster's parts of a tile, added in rank order; the columns are shared out over the CTAs, then over their warps, a lane four rows
// of 16 bytes.  (By 4-byte loads and 2-byte stores this took 3.5 us of 26 for 333 tokens of 2048 x 11008, four CTAs to a tile.)
template <int FMT, typename T, bool QUANT>
__device__ __forceinline__ void add_parts(const Mx4Job& J, const Mx4Walk& t, float* red, int rank) {
  const int r = (threadIdx.x & 31) * 4, row = t.mt * MX4_ROWS + r, warps = blockDim.x >> 5;
  if (row >= J.m) return;
  Mx4Factor f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = row_factor<FMT, T, QUANT>(J, t.expert, min(row + i, J.m - 1));
  const uint32_t base = smem_u32(red) + (uint32_t)r * 4u;
  for (int c = rank + J.split * (int)(threadIdx.x >> 5); c < t.rows; c += J.split * warps) {
    const float4 s = sum_cluster4(base + (uint32_t)(c * MX4_ROWS * 4), J.split);
    const float v[4] = {s.x * f[0].a * f[0].b, s.y * f[1].a * f[1].b, s.z * f[2].a * f[2].b, s.w * f[3].a * f[3].b};
    const long long at = (long long)(t.row0 + c) * J.y_stride + row;
    if (J.y_wide && row + 4 <= J.m) {
      uint32_t h[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (J.y_dtype == GLQB_DT_BF16) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
          h[i] = *reinterpret_cast<const uint32_t*>(&b);
        } else {
          const __half2 b = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
          h[i] = *reinterpret_cast<const uint32_t*>(&b);
        }
      }
      *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(J.y) + at) = make_uint2(h[0], h[1]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (row + i < J.m) mx4_put(J, at + i, v[i]);
    }
  }
}

// ---- 16-bit activations ---------------------------------------------------------------------------
// Weights come as they lie, 17 KiB per 128 x 256 (bulk copies), are decoded by sixteen warps straight into tensor memory as
// the A operand (thread = row, 64 values = 32 columns), activations by TMA as 64-value boxes with the 128-byte swizzle.  A step
// is 128 values, eight MMAs; two groups of eight warps decode the steps in turn.  Warp 0 issues MMAs, warp 1 loads
// activations, warp 2 weights, warps 4-7 drain, 8-23 decode.
//
// With wide tiles what bounds one CTA is shared memory: of 128 bytes a clock, writing and reading the activations of 192 rows takes
// 125 (2048 tokens of 14336 x 4096 317 us; without the loads 202).  Two CTAs therefore share a tile of 256 weight rows (PAIR): each
// brings half of the activations, the first one's thread issues for both.  What is to arrive at the issuing thread comes from
// both CTAs; what it releases goes to both.  2048 tokens of 14336 x 4096 171 us (1405 TFLOP/s; under the power limit 204), 32768 rows over 128
// experts of 2048 x 768 117 (139).
constexpr int G16_THREADS = 768, G16_W_STAGES = 3, G16_PRODUCERS = 8;

struct Mx4Ring { int x_stages, box_rows, x_half, a_stages, acc_cols; };  // stages of x, rows per box, bytes of 64 values of a CTA's rows

template <int FMT, typename T, bool PAIR>
__global__ void __launch_bounds__(G16_THREADS, 1) mx4_gemm16_kernel(const __grid_constant__ Mx4Job J, const __grid_constant__ CUtensorMap map, Mx4Ring R) {
  constexpr int TILE = mx4_tile_bytes(FMT);
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* w_base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* x_base = w_base + G16_W_STAGES * TILE;
  Bars& B = *reinterpret_cast<Bars*>(x_base + R.x_stages * 2 * R.x_half);
  const Mx4Lists L(reinterpret_cast<int*>(&B + 1), J.experts);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // a CTA's place among those that work on one tile: of a pair (weight rows), or of a split (values)
  const int ranks = PAIR ? 2 : J.split, first = blockIdx.x / ranks, step = gridDim.x / ranks, rank = blockIdx.x % ranks;
  if (threadIdx.x == 0) {
    for (int s = 0; s < G16_W_STAGES; ++s) { mbar_init(&B.full_w[s], 1); mbar_init(&B.empty_w[s], 2 * G16_PRODUCERS); }
    for (int s = 0; s < R.x_stages; ++s) { mbar_init(&B.full_x[s], 1); mbar_init(&B.empty_x[s], 1); }
    for (int s = 0; s < R.a_stages; ++s) { mbar_init(&B.full_a[s], PAIR ? 2 * G16_PRODUCERS : G16_PRODUCERS); mbar_init(&B.empty_a[s], 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(&B.acc_full[s], 1); mbar_init(&B.acc_empty[s], PAIR ? 8 : 4); }
    mbar_init(&B.drain, 1);
    B.abort = 0;
    fence_mbar_init();
  }
  if (warp == 0) alloc_all<PAIR>(&B.tmem);
  if (threadIdx.x == 32) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map)) : "memory");
  tc_fence_before();
  if (J.offsets) pdl_wait();
  mx4_groups(J, L);                         // (ends with a block barrier)
  pdl_trigger();
  if constexpr (PAIR) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = B.tmem, tmem_a = tmem + 2 * R.acc_cols;
  const int m_tiles = PAIR ? (J.m_tiles + 1) / 2 : J.m_tiles;
  const int tiles = min(L.pre[J.experts], J.max_tiles) * m_tiles;
  const int k0 = PAIR ? 0 : rank * J.k_tiles / J.split, k1 = PAIR ? J.k_tiles : (rank + 1) * J.k_tiles / J.split;     // tiles of 256 values
  const int steps = min(2 * k1, (J.n + 127) / 128) - 2 * k0;                                                          // of 128
  // this CTA's row tile (the second CTA of a pair may have none: it computes the one before again and stores nothing)
  auto row_tile = [&](const Mx4Walk& t) { return PAIR ? 2 * t.mt + rank : t.mt; };
  auto cols_of = [&](const Mx4Walk& t) { return PAIR ? (t.rows + 31) & ~31 : (t.rows + 15) & ~15; };
  uint32_t loads_w = 0, loads_x = 0;
  bool ok = true;

  if (warp == 0) {
    if ((!PAIR || rank == 0) && elect_one()) {
      Mx4Pos a, x, acc;
      const uint32_t x0 = smem_u32(x_base);
      for (Mx4Walk t(L, J.experts, first, step, tiles, m_tiles); t.more() && ok; t.next(L), acc.add(1, 2)) {
        const uint32_t idesc = idesc16(__is_same(T, __half) ? 0 : 1, PAIR ? 256 : 128, cols_of(t)), d = tmem + acc.s * R.acc_cols;
        if (!mbar_wait(&B.acc_empty[acc.s], acc.phase ^ 1u, &B.abort)) { ok = false; break; }
        tc_fence_after();
        for (int k = 0; k < steps; ++k, a.add(1, R.a_stages), x.add(1, R.x_stages)) {
          if (!mbar_wait(&B.full_x[x.s], x.phase, &B.abort) || !mbar_wait(&B.full_a[a.s], a.phase, &B.abort)) { ok = false; break; }
          tc_fence_after();
          const uint32_t at = tmem_a + a.s * 64u, b = x0 + x.s * 2u * R.x_half;
          const uint64_t d0 = umma_desc_sw128(b), d1 = umma_desc_sw128(b + R.x_half);
#pragma unroll
          for (int j = 0; j < 4; ++j) umma16<PAIR>(d, at + 8u * j, d0 + 2u * j, idesc, (k > 0 || j > 0) ? 1u : 0u);
#pragma unroll
          for (int j = 0; j < 4; ++j) umma16<PAIR>(d, at + 32u + 8u * j, d1 + 2u * j, idesc, 1u);
          commit<PAIR>(&B.empty_x[x.s]);
          commit<PAIR>(&B.empty_a[a.s]);
          if (k + 1 == steps) commit<PAIR>(&B.acc_full[acc.s]);
        }
      }
      if (!ok) { B.abort = 1; atomicCAS(J.status, 0, (int)ST_GAVE_UP_MMA); }
    }
  } else if (warp == 1) {
    // (a box per lane: one thread that issues them in turn is late among the warps that decode)
    pdl_wait();
    Mx4Pos x;
    for (Mx4Walk t(L, J.experts, first, step, tiles, m_tiles); t.more() && ok; t.next(L)) {
      const int rows = PAIR ? cols_of(t) / 2 : t.rows, row0 = t.row0 + (PAIR ? rank * rows : 0), boxes = (rows + R.box_rows - 1) / R.box_rows;
      const int box = lane >> 1, half = lane & 1, to = half * R.x_half + box * R.box_rows * 128;
      for (int k = 0; k < steps; ++k, ++loads_x, x.add(1, R.x_stages)) {
        ok = mbar_wait_warp(&B.empty_x[x.s], x.phase ^ 1u, &B.abort);
        if (!ok) break;
        if (lane == 0 && (!PAIR || rank == 0)) mbar_expect_tx(&B.full_x[x.s], (uint32_t)((PAIR ? 4 : 2) * boxes * R.box_rows * 128));
        __syncwarp();
        if (box < boxes)
          tma_load_2d<PAIR>(x_base + x.s * 2 * R.x_half + to, &map, k0 * MX4_K + k * 128 + half * 64, row0 + box * R.box_rows, &B.full_x[x.s]);
      }
    }
    if (!ok) { B.abort = 1; if (lane == 0) atomicCAS(J.status, 0, (int)ST_GAVE_UP_LOADER); }
  } else if (warp == 2) {
    if (lane == 0) {
      Mx4Pos w;
      auto weights = [&](const Mx4Walk& t) { return J.image + (((long long)t.expert * J.m_tiles + min(row_tile(t), J.m_tiles - 1)) * J.k_tiles + k0) * TILE; };
      if (!J.offsets) {                            // on their way to L2 while the kernel in front ends (which may write them: none is read)
        const Mx4Walk t(L, J.experts, first, step, tiles, m_tiles);
        if (t.more())
          for (int k = 0; k < min(G16_W_STAGES, k1 - k0); ++k) bulk_prefetch_l2(weights(t) + k * TILE, TILE);
      }
      pdl_wait();
      for (Mx4Walk t(L, J.experts, first, step, tiles, m_tiles); t.more() && ok; t.next(L)) {
        const uint8_t* src = weights(t);
        for (int k = k0; k < k1; ++k, ++loads_w, src += TILE, w.add(1, G16_W_STAGES)) {
          if (!mbar_wait(&B.empty_w[w.s], w.phase ^ 1u, &B.abort)) { ok = false; break; }
          mbar_expect_tx(&B.full_w[w.s], TILE);
          bulk_g2s(w_base + w.s * TILE, src, TILE, &B.full_w[w.s]);
        }
      }
      if (!ok) { B.abort = 1; atomicCAS(J.status, 0, (int)ST_GAVE_UP_LOADER); }
    }
  } else if (warp >= 8) {
    pdl_wait();
    // of a group's eight warps four take the first 64 values of a step, four the others; a warp the 32 rows of its quarter of tensor memory
    const int group = (warp - 8) >> 3, half = (warp >> 2) & 1, r = (warp & 3) * 32 + lane;
    const uint32_t to = tmem_a + ((uint32_t)((warp & 3) * 32) << 16) + half * 32u;
    // (A lane whose wait gave up goes on with what lies there, here and where results are drained, to the last tile: the instructions behind
    // the wait are the whole warp's, and it can leave neither alone nor, without a vote, with the others; a vote per wait took 1.5 % of the time
    // of 32768 rows over 128 experts of 2048 x 768, one per tile 1.  The other waits end at their next look at `abort`.)
    // Groups take the CTA's steps in turn, counted over all its tiles: behind an odd number of them the other group begins.  A wait by parity
    // holds only as long as the barrier is no further behind than the phase in front: a group's steps must not lie more than a_stages, two at
    // least, apart.  (They did, by three, where each tile began with the first group: with two stages group 1 could write a stage
    // that was not read yet.)
    Mx4Pos a, w;
    a.add(group, R.a_stages);
    int mine = group;                              // of a tile's steps the even ones or the odd ones
    for (Mx4Walk t(L, J.experts, first, step, tiles, m_tiles); t.more(); t.next(L)) {
      int top = 0;
      float up = 1.0f;
      if constexpr (FMT == GLQB_MX4_MXFP4) {
        top = J.tops[((long long)t.expert * J.m_tiles + min(row_tile(t), J.m_tiles - 1)) * MX4_ROWS + r] & 0xFF;
        if constexpr (!__is_same(T, __half)) top = mx4_base(top);
      } else if constexpr (!__is_same(T, __half)) {
        up = mx4_pow2(126 + mx4_shift(J.w_scale[t.expert], MX4_BF16_MOST));
      }
      for (int k = mine; k < steps + mine; k += 2, w.add(1, G16_W_STAGES)) {
        if (!mbar_wait(&B.full_w[w.s], w.phase, &B.abort)) { ok = false; B.abort = 1; }
        const uint8_t* tile = w_base + w.s * TILE;
        uint32_t v[32];
        if (k < steps) {
          const int c = mine * 4 + half * 2;       // 16-byte units of a row: two of them
          const uint8_t* codes = tile + (r >> 3) * 1024 + (r & 7) * 128;
          const uint8_t* sc = tile + MX4_CODE_BYTES + (r & 31) * 16 + (r >> 5) * 4;
          uint32_t sw;
          if constexpr (FMT == GLQB_MX4_MXFP4) sw = *reinterpret_cast<const uint32_t*>(sc + (c >> 2) * 512) >> (8 * (c & 3));
          else sw = *reinterpret_cast<const uint32_t*>(sc + (c >> 1) * 512);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint4 q = *reinterpret_cast<const uint4*>(codes + (((c + u) ^ (r & 7)) << 4));
            const uint32_t words[4] = {q.x, q.y, q.z, q.w};
            uint32_t m0, m1;
            if constexpr (FMT == GLQB_MX4_MXFP4) m0 = m1 = mx4_multiplier<T>((sw >> (8 * u)) & 0xFFu, top);
            else mx4_multipliers<T>((sw >> (16 * u)) & 0xFFFFu, up, m0, m1);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t p[4];
              mx4_pairs<T>(words[j], p);
#pragma unroll
              for (int e = 0; e < 4; ++e) v[u * 16 + j * 4 + e] = mx4_mul2<T>(p[e], j < 2 ? m0 : m1);
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.empty_w[w.s]);
        if (k < steps) {
          if (!mbar_wait(&B.empty_a[a.s], a.phase ^ 1u, &B.abort)) { ok = false; B.abort = 1; }
          __syncwarp();
          tc_fence_after();
          tmem_st32(to + a.s * 64u, v);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_first<PAIR>(&B.full_a[a.s]);
          a.add(2, R.a_stages);
        }
      }
      mine ^= steps & 1;
    }
    if (!ok) { B.abort = 1; if (lane == 0) atomicCAS(J.status, 0, (int)ST_GAVE_UP_PRODUCER); }
  } else if (warp >= 4) {
    pdl_wait();                                    // (y may still be in use)
    mx4_clear_rest(J, L.eff, threadIdx.x - 128, 128);
    Mx4Pos acc;
    for (Mx4Walk t(L, J.experts, first, step, tiles, m_tiles); t.more(); t.next(L), acc.add(1, 2)) {
      const int mt = row_tile(t), row = mt * MX4_ROWS + (warp & 3) * 32 + lane;
      Mx4Factor f{1.0f, 1.0f};
      if (row < J.m) f = row_factor<FMT, T, false>(J, t.expert, row);
      if (!mbar_wait(&B.acc_full[acc.s], acc.phase, &B.abort)) { B.abort = 1; atomicCAS(J.status, 0, (int)ST_GAVE_UP_EPILOGUE); }
      __syncwarp();
      tc_fence_after();
      if (!PAIR || mt < J.m_tiles)
        drain_tile<FMT, T, false>(J, t, mt, f, tmem + acc.s * R.acc_cols, warp & 3, lane, B.turn[warp & 3], !PAIR && J.split > 1 ? reinterpret_cast<float*>(x_base) : nullptr);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_first<PAIR>(&B.acc_empty[acc.s]);
    }
  }
  // ---- every thread arrives here, also after a wait gave up
  __syncwarp();
  if (!PAIR && J.split > 1) {                      // (one tile per cluster)
    cluster_sync();
    const Mx4Walk t(L, J.experts, first, step, tiles, m_tiles);
    if (t.more()) add_parts<FMT, T, false>(J, t, reinterpret_cast<float*>(x_base), rank);
    cluster_sync();
  }
  tc_fence_before();
  __syncthreads();
  if (B.abort) {
    // what may still be in flight: the copies armed last, and the MMAs issued so far
    if (warp == 2 && lane == 0)
      for (uint32_t n = 0; n < min(loads_w, (uint32_t)G16_W_STAGES); ++n) {
        const uint32_t u = loads_w - 1 - n;
        mbar_wait(&B.full_w[u % G16_W_STAGES], (u / G16_W_STAGES) & 1u);
      }
    if (warp == 1 && lane == 0) {
      if (!PAIR || rank == 0)                      // (a pair's first CTA for both: they end together)
        for (uint32_t n = 0; n < min(loads_x, (uint32_t)R.x_stages); ++n) {
          const uint32_t u = loads_x - 1 - n;
          mbar_wait(&B.full_x[u % R.x_stages], (u / R.x_stages) & 1u);
        }
    }
    if (warp == 0 && (!PAIR || rank == 0) && elect_one()) {
      commit<PAIR>(&B.drain);
      mbar_wait(&B.drain, 0);
    }
    tc_fence_before();
    __syncthreads();
  }
  if constexpr (PAIR) cluster_sync();              // (neither CTA's memory goes while the other still works on it)
  if (warp == 0) {
    tc_fence_after();
    dealloc_all<PAIR>(tmem);
  }
}

// ---- 4-bit activations ----------------------------------------------------------------------------
// Both operands as they lie in their images; a stage is 256 values: four MMAs, whose scales the issuing thread copies to tensor memory
// in front of them.  Warp 0 issues (in a pair's second CTA it reports the stages that have arrived), warp 1 loads, warps 4-7 drain.
//
// What bounds it is shared memory: per stage of 192 columns one CTA writes 43 KiB and the MMAs read 40, where they take 384 clocks at
// 128 bytes each.  Two CTAs that share a tile of 256 weight rows (PAIR) bring and read half of the activations each.  2048 tokens of 14336 x
// 4096 55 us behind 8 for the image of x.
constexpr int G4_THREADS = 256;
template <int FMT> struct G4 {
  static constexpr int ATOMS = mx4_scale_bytes(FMT) / 512;         // 512-byte pieces of scales per 128 rows x 256 values
  static constexpr int MAX_TN = FMT == GLQB_MX4_MXFP4 ? 192 : 160;
  static constexpr int SF_COLS = ATOMS * 12;                       // tensor memory of a stage: weights 4, activations 8 per piece
  static constexpr int STAGES = (512 - 2 * MAX_TN) / SF_COLS;      // MXFP4 5, NVFP4 4: tensor memory, and shared memory
};

template <int FMT, bool PAIR>
__global__ void __launch_bounds__(G4_THREADS, 1) mx4_gemm4_kernel(const __grid_constant__ Mx4Job J, int stages, int x_scales) {
  using C = G4<FMT>;
  constexpr int TILE = mx4_tile_bytes(FMT);
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int own = PAIR ? J.tn / 2 : J.tn, stage_bytes = TILE + (own + 7) / 8 * 1024 + x_scales;      // (a multiple of 1024: whole groups of eight rows)
  Bars& B = *reinterpret_cast<Bars*>(base + stages * stage_bytes);
  const Mx4Lists L(reinterpret_cast<int*>(&B + 1), J.experts);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ranks = PAIR ? 2 : J.split, first = blockIdx.x / ranks, step = gridDim.x / ranks, rank = blockIdx.x % ranks;
  if (threadIdx.x == 0) {
    // (full_w of the first CTA of a pair: the second one's stages)
    for (int s = 0; s < stages; ++s) { mbar_init(&B.full_x[s], 1); mbar_init(&B.empty_x[s], 1); mbar_init(&B.full_w[s], 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(&B.acc_full[s], 1); mbar_init(&B.acc_empty[s], PAIR ? 8 : 4); }
    mbar_init(&B.drain, 1);
    B.abort = 0;
    fence_mbar_init();
  }
  if (warp == 0) alloc_all<PAIR>(&B.tmem);
  tc_fence_before();
  if (J.offsets) pdl_wait();
  mx4_groups(J, L);
  pdl_trigger();
  if constexpr (PAIR) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = B.tmem;
  const int m_tiles = PAIR ? (J.m_tiles + 1) / 2 : J.m_tiles;
  const int tiles = min(L.pre[J.experts], J.max_tiles) * m_tiles;
  const int k0 = PAIR ? 0 : rank * J.k_tiles / J.split, steps = PAIR ? J.k_tiles : (rank + 1) * J.k_tiles / J.split - k0;
  auto row_tile = [&](const Mx4Walk& t) { return PAIR ? 2 * t.mt + rank : t.mt; };
  uint32_t loads = 0;
  bool ok = true;

  if (warp == 0) {
    if (!PAIR || rank == 0) {
      if (elect_one()) {
        Mx4Pos x, acc;
        for (Mx4Walk t(L, J.experts, first, step, tiles, m_tiles); t.more() && ok; t.next(L), acc.add(1, 2)) {
          const int cols = (t.rows + 15) & ~15;
          const uint32_t d = tmem + acc.s * C::MAX_TN;
          if (!mbar_wait(&B.acc_empty[acc.s], acc.phase ^ 1u, &B.abort)) { ok = false; break; }
          tc_fence_after();
          for (int k = 0; k < steps; ++k, x.add(1, stages)) {
            if (!mbar_wait(&B.full_x[x.s], x.phase, &B.abort) || (PAIR && !mbar_wait(&B.full_w[x.s], x.phase, &B.abort))) { ok = false; break; }
            tc_fence_after();
            const uint32_t w = smem_u32(base) + x.s * stage_bytes, xs = w + TILE, sc = xs + (own + 7) / 8 * 1024;
            const uint32_t sa = tmem + 2 * C::MAX_TN + x.s * C::SF_COLS, sb = sa + 4 * C::ATOMS;
            const uint64_t dws = scale_desc(w + MX4_CODE_BYTES), dxs = scale_desc(sc);
            // (copies and MMAs of one thread run in the order they are issued in)
#pragma unroll
            for (int j = 0; j < C::ATOMS; ++j) {
              tmem_copy_scales<PAIR>(sa + 4u * j, dws + 32u * j);
              tmem_copy_scales<PAIR>(sb + 8u * j, dxs + 32u * j);
              if (cols > 128) tmem_copy_scales<PAIR>(sb + 8u * j + 4u, dxs + 32u * (j + C::ATOMS));
            }
            const uint64_t da = umma_desc_sw128(w), db = umma_desc_sw128(xs);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t atom = j * C::ATOMS / 4, sf = C::ATOMS == 2 ? 2u * (j & 1) : 0u;
              umma4<FMT, PAIR>(d, da + 2u * j, db + 2u * j, idesc4<FMT>(PAIR ? 256 : 128, cols, sf), sa + 4u * atom, sb + 8u * atom, (k > 0 || j > 0) ? 1u : 0u);
            }
            commit<PAIR>(&B.empty_x[x.s]);
            if (k + 1 == steps) commit<PAIR>(&B.acc_full[acc.s]);
          }
        }
        if (!ok) { B.abort = 1; atomicCAS(J.status, 0, (int)ST_GAVE_UP_MMA); }
      }
    } else if (lane == 0) {
      Mx4Pos x;
      for (int i = first; i < tiles && ok; i += step)
        for (int k = 0; k < steps; ++k, x.add(1, stages)) {
          if (!mbar_wait(&B.full_x[x.s], x.phase, &B.abort)) { ok = false; break; }
          arrive_first<PAIR>(&B.full_w[x.s]);
        }
      if (!ok) { B.abort = 1; atomicCAS(J.status, 0, (int)ST_GAVE_UP_LOADER); }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const int x_stage = J.tn * 128 + x_scales;
      Mx4Pos x;
      int early = 0;                               // stages whose weights went out before x was there (x's kernel began behind all that may write them)
      for (Mx4Walk t(L, J.experts, first, step, tiles, m_tiles); t.more() && ok; t.next(L)) {
        const uint32_t x_codes = (uint32_t)((t.rows + 15) & ~15) * (PAIR ? 64u : 128u);
        const uint8_t* wsrc = J.image + (((long long)t.expert * J.m_tiles + min(row_tile(t), J.m_tiles - 1)) * J.k_tiles + k0) * TILE;
        const uint8_t* xsrc = J.x_image + ((long long)t.tt * J.k_tiles + k0) * x_stage;
        for (int k = 0; k < steps; ++k, ++loads, x.add(1, stages), wsrc += TILE, xsrc += x_stage) {
          if (!mbar_wait(&B.empty_x[x.s], x.phase ^ 1u, &B.abort)) { ok = false; break; }
          if (loads == 0) {
            for (; early < min(stages, steps); ++early) {
              mbar_expect_tx(&B.full_x[early], TILE + x_codes + x_scales);
              bulk_g2s(base + early * stage_bytes, wsrc + (long long)early * TILE, TILE, &B.full_x[early]);
            }
            pdl_wait();
          }
          uint8_t* w = base + x.s * stage_bytes;
          if (loads >= early) {
            mbar_expect_tx(&B.full_x[x.s], TILE + x_codes + x_scales);
            bulk_g2s(w, wsrc, TILE, &B.full_x[x.s]);
          }
          bulk_g2s(w + TILE, xsrc + (PAIR ? rank * x_codes : 0u), x_codes, &B.full_x[x.s]);
          bulk_g2s(w + TILE + (own + 7) / 8 * 1024, xsrc + J.tn * 128, x_scales, &B.full_x[x.s]);
        }
      }
      loads = max(loads, (uint32_t)early);
      if (!ok) { B.abort = 1; atomicCAS(J.status, 0, (int)ST_GAVE_UP_LOADER); }
    }
  } else if (warp >= 4) {
    pdl_wait();                                    // (y may still be in use)
    mx4_clear_rest(J, L.eff, threadIdx.x - 128, 128);
    Mx4Pos acc;
    for (Mx4Walk t(L, J.experts, first, step, tiles, m_tiles); t.more(); t.next(L), acc.add(1, 2)) {
      const int mt = row_tile(t), row = mt * MX4_ROWS + (warp & 3) * 32 + lane;
      Mx4Factor f{1.0f, 1.0f};
      if (row < J.m) f = row_factor<FMT, __half, true>(J, t.expert, row);
      if (!mbar_wait(&B.acc_full[acc.s], acc.phase, &B.abort)) { B.abort = 1; atomicCAS(J.status, 0, (int)ST_GAVE_UP_EPILOGUE); }
      __syncwarp();
      tc_fence_after();
      if (!PAIR || mt < J.m_tiles)
        drain_tile<FMT, __half, true>(J, t, mt, f, tmem + acc.s * C::MAX_TN, warp & 3, lane, B.turn[warp & 3], !PAIR && J.split > 1 ? reinterpret_cast<float*>(base) : nullptr);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_first<PAIR>(&B.acc_empty[acc.s]);
    }
  }
  // ---- every thread arrives here, also after a wait gave up
  __syncwarp();
  if (!PAIR && J.split > 1) {
    cluster_sync();
    const Mx4Walk t(L, J.experts, first, step, tiles, m_tiles);
    if (t.more()) add_parts<FMT, __half, true>(J, t, reinterpret_cast<float*>(base), rank);
    cluster_sync();
  }
  tc_fence_before();
  __syncthreads();
  if (B.abort) {
    if (warp == 1 && lane == 0)
      for (uint32_t n = 0; n < min(loads, (uint32_t)stages); ++n) {
        const uint32_t u = loads - 1 - n;
        mbar_wait(&B.full_x[u % stages], (u / stages) & 1u);
      }
    if (warp == 0 && (!PAIR || rank == 0) && elect_one()) {
      commit<PAIR>(&B.drain);
      mbar_wait(&B.drain, 0);
    }
    tc_fence_before();
    __syncthreads();
  }
  if constexpr (PAIR) cluster_sync();
  if (warp == 0) {
    tc_fence_after();
    dealloc_all<PAIR>(tmem);
  }
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// More than half of an SM's shared memory, whatever a launch needs: two CTAs on an SM would wait for each other's tensor memory,
// and clusters that do so in turn would wait for ever.
constexpr size_t ONE_PER_SM = 120 * 1024;

size_t groups_bytes(const Mx4Job& J) { return sizeof(Bars) + (size_t)(J.experts + 1) * 12; }

}  // namespace

int mx4_gemm_clusters(int split) { return mx4_clusters(mx4_gemm4_kernel<GLQB_MX4_MXFP4, false>, G4_THREADS, ONE_PER_SM, split); }

cudaError_t mx4_gemm16_launch(int format, bool x_bf16, const Mx4Job& J, int sm_count, cudaStream_t stream, const char** what) {
  Mx4Ring R;
  const int own = J.pair ? (J.tn + 31) / 32 * 16 : J.tn;       // rows of x that a CTA brings
  R.box_rows = std::min(own, 32);
  R.x_half = (own + R.box_rows - 1) / R.box_rows * R.box_rows * 128;
  R.acc_cols = (J.tn + 31) / 32 * 32;
  R.a_stages = std::min(4, (512 - 2 * R.acc_cols) / 64);
  const size_t fixed = 1024 + G16_W_STAGES * (size_t)mx4_tile_bytes(format) + groups_bytes(J);
  R.x_stages = (int)std::min<size_t>(8, (227 * 1024 - fixed) / (2 * (size_t)R.x_half));
  const size_t smem = std::max(ONE_PER_SM, fixed + (size_t)R.x_stages * 2 * R.x_half);
  CUtensorMap map;
  const EncodeTiled encode = encode_tiled();
  if (!encode) { *what = "cuTensorMapEncodeTiled not found"; return cudaErrorNotSupported; }
  const cuuint64_t dims[2] = {(cuuint64_t)J.n, (cuuint64_t)J.rows}, strides[1] = {(cuuint64_t)(J.rows == 1 ? (J.n * 2 + 15) / 16 * 16 : J.x_stride * 2)};
  const cuuint32_t box[2] = {64, (cuuint32_t)R.box_rows}, ones[2] = {1, 1};
  const CUresult r = encode(&map, x_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(J.x), dims, strides, box, ones,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { *what = "cuTensorMapEncodeTiled refused the activations"; return cudaErrorInvalidValue; }
  const int ranks = J.pair ? 2 : J.split;
  const long long tiles = (long long)J.max_tiles * (J.pair ? (J.m_tiles + 1) / 2 : J.m_tiles);
  const int grid = J.split > 1 ? (int)(tiles * ranks) : (int)std::min<long long>(tiles, sm_count / ranks) * ranks;
  auto run = [&](auto fmt, auto type, auto pair) {
    constexpr auto K = mx4_gemm16_kernel<decltype(fmt)::value, decltype(type), decltype(pair)::value>;
    return mx4_launch<K>(K, grid, G16_THREADS, smem, ranks, stream, J, map, R);
  };
  using M = std::integral_constant<int, GLQB_MX4_MXFP4>;
  using N = std::integral_constant<int, GLQB_MX4_NVFP4>;
  auto of = [&](auto pair) {
    if (format == GLQB_MX4_MXFP4) return x_bf16 ? run(M(), __nv_bfloat16(), pair) : run(M(), __half(), pair);
    return x_bf16 ? run(N(), __nv_bfloat16(), pair) : run(N(), __half(), pair);
  };
  return J.pair ? of(std::true_type()) : of(std::false_type());
}

cudaError_t mx4_gemm4_launch(int format, const Mx4Job& J, int sm_count, cudaStream_t stream) {
  const int x_scales = mx4_x_scale_bytes(format, J.tn), most = format == GLQB_MX4_MXFP4 ? G4<GLQB_MX4_MXFP4>::STAGES : G4<GLQB_MX4_NVFP4>::STAGES;
  const int ranks = J.pair ? 2 : J.split, own = J.pair ? J.tn / 2 : J.tn;
  const size_t fixed = 1024 + groups_bytes(J), stage = (size_t)mx4_tile_bytes(format) + (own + 7) / 8 * 1024 + x_scales;
  const int stages = (int)std::min<size_t>(most, (227 * 1024 - fixed) / stage);
  const long long tiles = (long long)J.max_tiles * (J.pair ? (J.m_tiles + 1) / 2 : J.m_tiles);
  const int grid = J.split > 1 ? (int)(tiles * ranks) : (int)std::min<long long>(tiles, sm_count / ranks) * ranks;
  const size_t smem = std::max(ONE_PER_SM, fixed + stages * stage);
  auto run = [&](auto fmt, auto pair) {
    constexpr auto K = mx4_gemm4_kernel<decltype(fmt)::value, decltype(pair)::value>;
    return mx4_launch<K>(K, grid, G4_THREADS, smem, ranks, stream, J, stages, x_scales);
  };
  auto of = [&](auto fmt) { return J.pair ? run(fmt, std::true_type()) : run(fmt, std::false_type()); };
  return format == GLQB_MX4_MXFP4 ? of(std::integral_constant<int, GLQB_MX4_MXFP4>()) : of(std::integral_constant<int, GLQB_MX4_NVFP4>());
}

}  // namespace glqb
