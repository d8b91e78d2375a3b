// Products of microscaled 4-bit weights with few rows of x: decode steps, experts of few tokens.
//
// What bounds these is the weights' way from HBM and, close behind, the instructions that make 16-bit operands of them.  A warp
// streams 16 rows x 256 values at a time (four 16-byte loads per lane, the next four under way), turns them into fragments of
// mma.sync.m16n8k16 in registers (five instructions per two weights) and multiplies them with 8 NB rows of x.  The MMA's order
// of values is free as long as both operands have it: lane t of a quad takes the 16-byte unit t of a weight row, 32 values, and
// of each row of x the same 32 values, so nothing is exchanged.  The eight warps of a CTA share out the values of a strip of 16
// rows; their sums are added in warp order.  A CTA takes strips in turn, its loads running ahead over the strips' borders.
#include "glqb_mx4_gemm.cuh"
#include "glqb_launch.h"
#include <algorithm>

namespace glqb {
namespace {

constexpr int MV4_WARPS = 8, MV4_THREADS = MV4_WARPS * 32, MV4_ROWS = 16;

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (__is_same(T, __half))
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 ld_stream(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// The token tile of a CTA: an expert and up to tn of its rows.  All threads; a range that ends before it begins is empty.
__device__ __forceinline__ bool mv4_tile(const Mx4Job& J, int tile, Mx4Tile& t) {
  if (!J.offsets) {
    t = Mx4Tile{0, tile * J.tn, min(J.tn, J.rows - tile * J.tn)};
    return t.rows > 0;
  }
  __shared__ int sums[MV4_WARPS], found[3];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int begin[4], rows[4], mine = 0;                       // four experts per thread: MX4_MAX_EXPERTS
  const int e0 = threadIdx.x * 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    begin[i] = rows[i] = 0;
    const int e = e0 + i;
    if (e < J.experts) {
      const long long b = J.wide ? reinterpret_cast<const long long*>(J.offsets)[e] : reinterpret_cast<const int*>(J.offsets)[e];
      const long long f = J.wide ? reinterpret_cast<const long long*>(J.offsets)[e + 1] : reinterpret_cast<const int*>(J.offsets)[e + 1];
      begin[i] = (int)max(0ll, min((long long)J.rows, b));
      rows[i] = (int)max(0ll, min((long long)J.rows, f)) - begin[i];
    }
    mine += (max(rows[i], 0) + J.tn - 1) / J.tn;
  }
  int upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int u = __shfl_up_sync(0xFFFFFFFFu, upto, d);
    if (lane >= d) upto += u;
  }
  if (lane == 31) sums[warp] = upto;
  if (threadIdx.x == 0) found[2] = 0;
  __syncthreads();
  for (int w = 0; w < warp; ++w) upto += sums[w];
  int at = tile - (upto - mine);
  if (at >= 0 && at < mine) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = (max(rows[i], 0) + J.tn - 1) / J.tn;
      if (at >= 0 && at < n) {
        found[0] = e0 + i;
        found[1] = begin[i] + at * J.tn;
        found[2] = min(J.tn, rows[i] - at * J.tn);
      }
      at -= n;
    }
  }
  __syncthreads();
  t = Mx4Tile{found[0], found[1], found[2]};
  return t.rows > 0;
}

template <int FMT>
struct Mv4Item {               // 16 rows x 256 values: rows g and g + 8, 16-byte units t and t + 4, and their scales
  uint4 w[2][2];
  uint32_t s[2][2];
  __device__ __forceinline__ void load(const uint8_t* tile, int r, int t) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = r + 8 * h;
      const uint8_t* codes = tile + (row >> 3) * 1024 + (row & 7) * 128;
      const uint8_t* scales = tile + MX4_CODE_BYTES + (row & 31) * 16 + (row >> 5) * 4;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        w[h][u] = ld_stream(codes + (((t + 4 * u) ^ (row & 7)) << 4));
        if constexpr (FMT == GLQB_MX4_MXFP4) s[h][u] = __ldg(scales + u * 512 + t);
        else s[h][u] = __ldg(reinterpret_cast<const uint16_t*>(scales + (2 * u + (t >> 1)) * 512 + (t & 1) * 2));
      }
    }
  }
};

template <int FMT, typename T, int NB>
__global__ void __launch_bounds__(MV4_THREADS, NB == 1 ? 3 : 2) mx4_mv_kernel(const __grid_constant__ Mx4Job J, int strips) {
  __shared__ float red[2][MV4_WARPS][8 * NB][MV4_ROWS];
  Mx4Tile tile;
  if (!mv4_tile(J, blockIdx.y, tile)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint8_t* image = J.image + (long long)tile.expert * J.m_tiles * J.k_tiles * mx4_tile_bytes(FMT);
  const T* x = reinterpret_cast<const T*>(J.x) + (long long)tile.row0 * J.x_stride;
  auto tile_of = [&](int strip, int k) -> const uint8_t* { return image + ((long long)(strip >> 3) * J.k_tiles + k) * mx4_tile_bytes(FMT); };

  int strip = blockIdx.x, k = warp;
  Mv4Item<FMT> next;
  if (k < J.k_tiles) next.load(tile_of(strip, k), (strip & 7) * MV4_ROWS + g, t);
  for (int turn = 0; strip < strips; ++turn) {
    float acc[NB][4] = {};
    int top[2] = {0, 0};
    if constexpr (FMT == GLQB_MX4_MXFP4) {
      const uint8_t* p = J.tops + ((long long)tile.expert * J.m_tiles * MX4_ROWS) + strip * MV4_ROWS + g;
      top[0] = p[0];
      top[1] = p[8];
    }
    const int after = strip + gridDim.x;
#pragma unroll 1
    for (; k < J.k_tiles; ) {
      Mv4Item<FMT> it = next;
      const int kt = k;
      k += MV4_WARPS;
      if (k < J.k_tiles) next.load(tile_of(strip, k), (strip & 7) * MV4_ROWS + g, t);
      else if (after < strips) next.load(tile_of(after, warp), (after & 7) * MV4_ROWS + g, t);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int col = kt * MX4_K + (t + 4 * u) * 32;
        uint32_t m[2][2];                                // multipliers of rows g and g + 8, of the first and last 16 values
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (FMT == GLQB_MX4_MXFP4) m[h][0] = m[h][1] = mx4_multiplier<FMT, T>(it.s[h][u], top[h]);
          else {
            m[h][0] = mx4_multiplier<FMT, T>(it.s[h][u] & 0xFFu, 0);
            m[h][1] = mx4_multiplier<FMT, T>(it.s[h][u] >> 8, 0);
          }
        }
        const uint32_t w[2][4] = {{it.w[0][u].x, it.w[0][u].y, it.w[0][u].z, it.w[0][u].w}, {it.w[1][u].x, it.w[1][u].y, it.w[1][u].z, it.w[1][u].w}};
#pragma unroll
        for (int j = 0; j < 4; ++j) {                    // eight values: two MMAs
          uint4 b[NB];
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            b[i] = make_uint4(0, 0, 0, 0);
            if (i * 8 + g < tile.rows && col + j * 8 < J.n) b[i] = *reinterpret_cast<const uint4*>(x + (long long)(i * 8 + g) * J.x_stride + col + j * 8);
          }
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            uint32_t a[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) a[q] = mx4_mul2<T>(mx4_pair<T>(w[q & 1][j], 2 * p + (q >> 1)), m[q & 1][j >> 1]);
#pragma unroll
            for (int i = 0; i < NB; ++i) mma16816<T>(acc[i], a, p ? b[i].z : b[i].x, p ? b[i].w : b[i].y);
          }
        }
      }
    }
    // (two buffers in turn: a strip's sums are read before the barrier of the next one's)
    auto& mine = red[turn & 1];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) mine[warp][i * 8 + 2 * t + (q & 1)][g + 8 * (q >> 1)] = acc[i][q];
    __syncthreads();
    for (int o = threadIdx.x; o < tile.rows * MV4_ROWS; o += MV4_THREADS) {
      const int r = o % MV4_ROWS, c = o / MV4_ROWS, row = strip * MV4_ROWS + r;
      float v = 0.0f;
#pragma unroll
      for (int s = 0; s < MV4_WARPS; ++s) v += mine[s][c][r];
      if (row < J.m) {
        const Mx4Factor f = mx4_row_factor<FMT, T>(J, tile.expert, row);
        mx4_put(J, (long long)(tile.row0 + c) * J.y_stride + row, v * f.a * f.b);
      }
    }
    strip = after;
    k = warp;
  }
}

}  // namespace

cudaError_t mx4_mv_launch(int format, bool x_bf16, const Mx4Job& J, int sm_count, cudaStream_t stream) {
  const int strips = (J.m + MV4_ROWS - 1) / MV4_ROWS, nb = J.tn / 8;
  // as many CTAs as the SMs hold, each with the same number of strips
  const long long room = std::max<long long>(1, (long long)sm_count * (nb == 1 ? 3 : 2) / J.max_tiles), turns = (strips + room - 1) / room;
  const dim3 grid((unsigned)((strips + turns - 1) / turns), (unsigned)J.max_tiles);
  auto run = [&](auto* kernel) { kernel<<<grid, MV4_THREADS, 0, stream>>>(J, strips); return cudaGetLastError(); };
  auto of = [&](auto fmt, auto type) {
    using T = decltype(type);
    constexpr int F = decltype(fmt)::value;
    return nb == 1 ? run(mx4_mv_kernel<F, T, 1>) : run(mx4_mv_kernel<F, T, 2>);
  };
  using M = std::integral_constant<int, GLQB_MX4_MXFP4>;
  using N = std::integral_constant<int, GLQB_MX4_NVFP4>;
  if (format == GLQB_MX4_MXFP4) return x_bf16 ? of(M(), __nv_bfloat16()) : of(M(), __half());
  return x_bf16 ? of(N(), __nv_bfloat16()) : of(N(), __half());
}

}  // namespace glqb
