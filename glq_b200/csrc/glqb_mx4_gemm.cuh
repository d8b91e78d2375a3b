// What the products of microscaled 4-bit weights share: the job, the token tiles of experts, the results.
#pragma once
#include "glqb_mx4.cuh"
#include "glqb_ptx.cuh"
#include "glqb_launch.h"
#include <atomic>

namespace glqb {

constexpr int MX4_MAX_EXPERTS = 1024;

struct Mx4Job {
  const uint8_t* image;
  const uint16_t* tops;       // MXFP4: of every row (experts x m_tiles * 128) the largest scale byte, + 256: see mx4_row_top_kernel
  const float* w_scale;       // NVFP4: fp32 scale per expert
  const float* x_scale;       // 4-bit activations, NVFP4: theirs
  const void* offsets;        // null: one matrix, all rows
  int wide, experts, rows, m, n, m_tiles, k_tiles;
  int tn;                     // most rows of x per token tile: a multiple of 16, or 8
  int max_tiles;              // bound of the token tiles
  int split;                  // CTAs of a cluster that share a tile's sum
  int pair;                   // two CTAs share a tile of 256 weight rows (split 1)
  void* y;
  long long y_stride;
  int y_dtype, accumulate;
  int clear;                  // rows of no expert are zeroed
  bool y_wide;                // 16-bit results whose rows lie on 16 bytes, nothing to add
  const void* x;              // 16-bit activations
  long long x_stride;
  uint8_t* x_image;           // 4-bit activations: per token tile, per 256 values: tn rows of 128 bytes, then the scales
  int* status;
};

#ifdef __CUDACC__
// (Each .aligned instruction wants all lanes of its warp: whoever comes here from loops of different lengths is gathered first.)
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_arrive() {      // (hands over nothing)
  __syncwarp();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr, int rank) {
  uint32_t a;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}

__device__ __forceinline__ void st_cluster(uint32_t addr, int rank, float v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
}
// four values of every CTA of the cluster, added in rank order (all loads before the first sum)
__device__ __forceinline__ float4 sum_cluster4(uint32_t addr, int ranks) {
  float4 v[8];
#pragma unroll
  for (int s = 0; s < 8; ++s) v[s] = s < ranks ? ld_cluster4(addr, s) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float4 sum = v[0];
#pragma unroll
  for (int s = 1; s < 8; ++s) sum = make_float4(sum.x + v[s].x, sum.y + v[s].y, sum.z + v[s].z, sum.w + v[s].w);
  return sum;
}
// Rows of every expert and the token tiles in front of it.  offsets are held to 0 .. rows and to ascend (each at least
// the largest before it), so that whatever they hold, experts do not overlap and the tiles are no more than max_tiles.
// Called by all threads; the lists have experts + 1 entries each, in shared memory.
struct Mx4Lists {
  int *eff, *pre, *per;       // an expert's first row, the token tiles in front of it, the rows of its tiles
  __device__ __forceinline__ Mx4Lists(int* at, int experts) : eff(at), pre(at + experts + 1), per(at + 2 * (experts + 1)) {}
};
__device__ __forceinline__ void mx4_groups(const Mx4Job& J, const Mx4Lists& L) {
  int *eff = L.eff, *pre = L.pre;
  if (J.offsets) {
    for (int e = threadIdx.x; e <= J.experts; e += blockDim.x) {
      const long long o = J.wide ? reinterpret_cast<const long long*>(J.offsets)[e] : reinterpret_cast<const int*>(J.offsets)[e];
      eff[e] = (int)max(0ll, min((long long)J.rows, o));
    }
    __syncthreads();
  }
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    if (!J.offsets) {
      if (lane == 0) { eff[0] = 0; eff[1] = J.rows; pre[0] = 0; pre[1] = (J.rows + J.tn - 1) / J.tn; }
    } else {
      int top = 0, tiles = 0;
      for (int b = 0; b <= J.experts; b += 32) {
        const int e = min(b + lane, J.experts);
        int v = eff[e];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int u = __shfl_up_sync(0xFFFFFFFFu, v, d);
          if (lane >= d) v = max(v, u);
        }
        v = max(v, top);
        int before = __shfl_up_sync(0xFFFFFFFFu, v, 1);
        if (lane == 0) before = b == 0 ? v : top;
        int t = (v - before + J.tn - 1) / J.tn;        // tiles of expert e - 1
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int u = __shfl_up_sync(0xFFFFFFFFu, t, d);
          if (lane >= d) t += u;
        }
        t += tiles;
        if (b + lane <= J.experts) { eff[e] = v; pre[e] = t; }
        top = __shfl_sync(0xFFFFFFFFu, v, 31);
        tiles = __shfl_sync(0xFFFFFFFFu, t, 31);
      }
    }
  }
  __syncthreads();
  // An expert's rows are split evenly over as few tiles as they need, in steps of 16 (no tile is empty: the tiles before the last
  // hold fewer than the expert has).
  for (int e = threadIdx.x; e < J.experts; e += blockDim.x) {
    const int rows = eff[e + 1] - eff[e], tiles = max(pre[e + 1] - pre[e], 1);
    L.per[e] = J.tn <= 16 ? J.tn : ((rows + tiles - 1) / tiles + 15) & ~15;
  }
  __syncthreads();
}
// the last e with list[e] <= v (list ascends, list[0] <= v < list[experts]): the expert that has tile, or row, v
__device__ __forceinline__ int mx4_find(const int* list, int experts, int v) {
  int lo = 0, hi = experts;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (list[mid] <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}
// The tiles of a CTA, one after the other: number `i` of (token tile, row tile), rows first.  (A search and three divisions per tile and
// role took 1550 clocks among the warps that decode.)
struct Mx4Walk {
  int i, mt, expert, row0, rows;
  int tt, tiles, m_tiles, step, dt, dm;
  __device__ __forceinline__ Mx4Walk(const Mx4Lists& L, int experts, int first, int step, int tiles, int m_tiles)
      : i(first), tt(first / m_tiles), tiles(tiles), m_tiles(m_tiles), step(step) {
    mt = first - tt * m_tiles;
    dt = step / m_tiles;
    dm = step - dt * m_tiles;
    expert = row0 = rows = 0;
    if (!more()) return;
    if (experts > 1) expert = mx4_find(L.pre, experts, tt);
    place(L);
  }
  __device__ __forceinline__ bool more() const { return i < tiles; }
  __device__ __forceinline__ void place(const Mx4Lists& L) {
    const int per = L.per[expert], at = (tt - L.pre[expert]) * per;
    row0 = L.eff[expert] + at;
    rows = min(per, L.eff[expert + 1] - row0);
  }
  __device__ __forceinline__ void next(const Mx4Lists& L) {
    i += step;
    tt += dt;
    mt += dm;
    if (mt >= m_tiles) { mt -= m_tiles; ++tt; }
    if (!more()) return;
    while (L.pre[expert + 1] <= tt) ++expert;
    place(L);
  }
};

struct Mx4Pos {                   // a place in a ring, and the parity of its round
  uint32_t s = 0, phase = 0;
  __device__ __forceinline__ void add(uint32_t d, uint32_t n) {
    s += d;
    while (s >= n) { s -= n; phase ^= 1u; }
  }
};

__device__ __forceinline__ void mx4_put(const Mx4Job& J, long long at, float v) {
  if (J.y_dtype == GLQB_DT_BF16) {
    __nv_bfloat16* p = reinterpret_cast<__nv_bfloat16*>(J.y) + at;
    *p = __float2bfloat16_rn(J.accumulate ? __bfloat162float(*p) + v : v);
  } else if (J.y_dtype == GLQB_DT_F16) {
    __half* p = reinterpret_cast<__half*>(J.y) + at;
    *p = __float2half_rn(J.accumulate ? __half2float(*p) + v : v);
  } else {
    float* p = reinterpret_cast<float*>(J.y) + at;
    *p = J.accumulate ? *p + v : v;
  }
}

// Rows of no expert (the experts' rows are one range: mx4_groups) are zeroed: by `threads` threads of each CTA.
__device__ __forceinline__ void mx4_clear_rest(const Mx4Job& J, const int* eff, int thread, int threads) {
  if (!J.clear) return;
  const int first = eff[0], last = eff[J.experts], rest = J.rows - (last - first), size = J.y_dtype == GLQB_DT_F32 ? 4 : 2;
  for (int i = blockIdx.x; i < rest; i += gridDim.x) {
    uint8_t* p = reinterpret_cast<uint8_t*>(J.y) + (long long)(i < first ? i : i + (last - first)) * J.y_stride * size;
    if (J.y_wide && J.m % 8 == 0) {
      for (int c = thread; c < J.m / 8; c += threads) reinterpret_cast<uint4*>(p)[c] = make_uint4(0, 0, 0, 0);
    } else {
      for (int c = thread; c < J.m; c += threads) {
        if (size == 4) reinterpret_cast<uint32_t*>(p)[c] = 0u;
        else reinterpret_cast<uint16_t*>(p)[c] = 0;
      }
    }
  }
}

// ---- 4-bit weights as 16-bit operands -------------------------------------------------------------
// fp16: cvt takes two codes of a byte to fp16.  bf16 has no such instruction: the bits of a code are moved to sign, exponent and
// first mantissa bit of a 16-bit number, where they read as the value times 2^-126, subnormals included.  One multiplication by
// the scale then gives the operand exactly.  So that multiplier and operand stay in range, operands are
//   MXFP4  value * 2^(s - top + 13) (fp16), value * 2^(s - base) (bf16), top the largest scale byte of the row, base mx4_base(top)
//   NVFP4  value * s (fp16), value * s * 2^k (bf16), k mx4_shift(t)
// and mx4_row_factor is what the sums are multiplied by.  bf16 activations may be near the end of fp32's range: a sum must not leave it where the
// result does not.  Operands are therefore no larger than the weights, down to where they are so small (6 * 2^-24, 2688 * 2^-31) that sums of 2^19
// products stay in range whatever the activations are.
//
// bf16: the four pairs of a word, unscaled, r[i] holds values 2i and 2i + 1.  Logic and right shifts issue at half an instruction a
// clock, and so do integer products (left shifts), on a pipe of their own.  Two of the pairs are therefore brought to bits 9:6 of
// each half and copied to 15:12 by a product with 65, the others masked at 15:12 and shifted down: ten instructions on the one
// pipe and four on the other per word, where all pairs the second way are twelve and three.
__device__ __forceinline__ void mx4_pairs_bf16(uint32_t w, uint32_t (&r)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < 2) {
      r[i] = (((w << (6 - 4 * i)) & 0x03C003C0u) * 65u) & 0x81C081C0u;
    } else {
      const uint32_t x = (i == 3 ? w : w << 4) & 0xF000F000u;
      r[i] = (x | x >> 6) & 0x81C081C0u;
    }
  }
}
// fp16: the bytes of a word, two values each
__device__ __forceinline__ void mx4_bytes_f16(uint32_t w, uint32_t (&r)[4]) {
  asm("{ .reg .b8 a, b, c, d; mov.b32 {a, b, c, d}, %4; cvt.rn.f16x2.e2m1x2 %0, a; cvt.rn.f16x2.e2m1x2 %1, b; cvt.rn.f16x2.e2m1x2 %2, c; "
      "cvt.rn.f16x2.e2m1x2 %3, d; }" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(w));
}
// the pairs of a word in the order of the values
template <typename T>
__device__ __forceinline__ void mx4_pairs(uint32_t w, uint32_t (&r)[4]) {
  if constexpr (__is_same(T, __half)) {
    // nibbles 0 2 4 6 1 3 5 7 -> bytes (0 1) (2 3) (4 5) (6 7)
    const uint32_t v = w >> 16, a = (w & 0x0F0Fu) | ((v & 0x0F0Fu) << 4), b = ((w >> 4) & 0x0F0Fu) | (v & 0xF0F0u);
    mx4_bytes_f16(__byte_perm(a, b, 0x5140), r);
  } else {
    mx4_pairs_bf16(w, r);
  }
}
// MXFP4: the scale byte that bf16 operands of a row are held relative to
__device__ __forceinline__ int mx4_base(int top) { return top + min(24, max(0, 127 - top)); }
// NVFP4: the power of two that a matrix's bf16 operands (or the sums of few rows) are multiplied by: that of t, between 2^-31 and 2^most
__device__ __forceinline__ int mx4_shift(float t, int most) { return max(-31, min(most, (int)(__float_as_uint(t) >> 23 & 0xFFu) - 127)); }
constexpr int MX4_BF16_MOST = -7;                              // (operands of up to 21: the multiplier, 448 * 2^(126 + k), is a bf16 number)
__device__ __forceinline__ float mx4_pow2(int p) { return __uint_as_float((uint32_t)(p + 127) << 23); }      // -126 .. 127
// MXFP4: what a block's codes are multiplied by, in both halves; `top`: what its row's operands are relative to
template <typename T>
__device__ __forceinline__ uint32_t mx4_multiplier(uint32_t s, int top) {
  const int d = (int)s - top;
  uint32_t h;
  if constexpr (__is_same(T, __half)) h = s == 255u ? 0x7E00u : d > -28 ? (uint32_t)(d + 28) << 10 : d >= -37 ? 1u << (d + 37) : 0u;
  else h = s == 255u ? 0x7FC0u : (uint32_t)max(d + 253, 0) << 7;
  return h | h << 16;
}
// NVFP4: the same of two neighbouring blocks, from their bytes; `up` (bf16): 2^(126 + shift)
template <typename T>
__device__ __forceinline__ void mx4_multipliers(uint32_t two, float up, uint32_t& m0, uint32_t& m1) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
  if constexpr (__is_same(T, __half)) {
    const uint32_t b = (uint32_t)h.x | (uint32_t)h.y << 16;
    m0 = __byte_perm(b, 0, 0x1010);
    m1 = __byte_perm(b, 0, 0x3232);
  } else {
    const float2 f = __half22float2(__half2(h));
    float a = f.x, b = f.y;
    mx4_mul_f32x2(a, b, up, up);
    m0 = __byte_perm(__float_as_uint(a), 0, 0x3232);
    m1 = __byte_perm(__float_as_uint(b), 0, 0x3232);
  }
}
template <typename T>
__device__ __forceinline__ uint32_t mx4_mul2(uint32_t a, uint32_t b) {
  if constexpr (__is_same(T, __half)) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}
struct Mx4Factor { float a, b; };     // two factors: 2^-127 and 2^127 have no single one
template <typename T>
__device__ __forceinline__ Mx4Factor mx4_power(uint32_t top) {          // MXFP4, from a row's entry in `tops`
  const int s = (int)(top & 0xFFu), p = __is_same(T, __half) ? s - 140 : mx4_base(s) - 127, h = p >> 1;
  return Mx4Factor{__uint_as_float((uint32_t)(h + 127) << 23), __uint_as_float((uint32_t)(p - h + 127) << 23)};
}
// NVFP4, sums that are held smaller by a power of two p: times p t, in an order that does not leave fp32's range on the way
__device__ __forceinline__ Mx4Factor mx4_factor(float t, float p) { return t < 1.0f ? Mx4Factor{1.0f, t * p} : Mx4Factor{p, t}; }
template <int FMT, typename T>
__device__ __forceinline__ Mx4Factor mx4_row_factor(const Mx4Job& J, int expert, int row) {
  if constexpr (FMT == GLQB_MX4_MXFP4) return mx4_power<T>(J.tops[(long long)expert * J.m_tiles * MX4_ROWS + row]);
  else if constexpr (__is_same(T, __half)) return Mx4Factor{1.0f, J.w_scale[expert]};
  else return mx4_factor(J.w_scale[expert], mx4_pow2(-mx4_shift(J.w_scale[expert], MX4_BF16_MOST)));
}
#endif  // __CUDACC__

inline int mx4_device() {       // the current one, 0..63
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64 ? dev : 0;
}
// Chained to the kernel in front (launch_chained), `cluster` CTAs per cluster.
template <auto K, typename... P, typename... A>
inline cudaError_t mx4_launch(void (*kernel)(P...), int grid, int threads, size_t smem, int cluster, cudaStream_t stream, A... args) {
  static std::atomic<int> limit[64];     // per device: the shared memory the kernel may have (raised, never lowered)
  std::atomic<int>& most = limit[mx4_device()];
  if (most.load(std::memory_order_relaxed) < (int)smem) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e != cudaSuccess) return e;
    most.store(227 * 1024, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled();
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// Clusters of `cluster` CTAs that the device holds at once (SMs come in groups whose size no cluster divides: 132 CTAs of 148 in clusters
// of four, 120 of eight; a launch of more takes twice as long).
template <typename... P>
inline int mx4_clusters(void (*kernel)(P...), int threads, size_t smem, int cluster) {
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)cluster);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  return cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) == cudaSuccess ? n : 0;
}
int mx4_mv_clusters(int split);
int mx4_gemm_clusters(int split);
// ---- glqb_mx4_mv.cu
// Few rows of x (tn 8 or 16), which start on 16 bytes and end on whole eights of values.
cudaError_t mx4_mv_launch(int format, bool x_bf16, const Mx4Job& job, int sm_count, cudaStream_t stream);
// ---- glqb_mx4_gemm.cu
// `x_bf16`: type of 16-bit activations.  Rows of x start on 16 bytes.
cudaError_t mx4_gemm16_launch(int format, bool x_bf16, const Mx4Job& job, int sm_count, cudaStream_t stream, const char** what);
cudaError_t mx4_gemm4_launch(int format, const Mx4Job& job, int sm_count, cudaStream_t stream);
// scales of a token tile per 256 values, in bytes
inline int mx4_x_scale_bytes(int format, int tn) { return mx4_scale_bytes(format) * ((tn + 127) / 128); }

}  // namespace glqb
