// Microscaled 4-bit floating point: quantisation and back, the weight image, and the C entry points (include/glq_b200.h).
#include "glqb_mx4_gemm.cuh"
#include <algorithm>
#include <atomic>
#include <cstdarg>
#include <cstdio>

namespace glqb {
namespace {

int mx4_fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  set_error_message(buf);
  return code;
}
int mx4_launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? GLQB_OK : mx4_fail(GLQB_E_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

constexpr int QT_THREADS = 256;

__device__ int g_mx4_status;   // 0, or what gave up (ST_GAVE_UP_*): products have no plan to keep it in

// Rows and columns of a call.  Rows that follow one another without a gap and end on whole blocks are one long row: their
// codes and scales do too.
struct Mx4Rows {
  long long rows, stride;     // elements between rows
  long long cols;
  int chunks;                 // eights of values per row, whole blocks
  bool vec;
};

// Rows offsets[0] .. offsets[experts] - 1, held to those there are.
struct Mx4Range {
  const void* offsets;        // null: all
  int wide, experts;
  __device__ void get(long long rows, long long& first, long long& last) const {
    first = 0;
    last = rows;
    if (!offsets) return;
    first = wide ? reinterpret_cast<const long long*>(offsets)[0] : reinterpret_cast<const int*>(offsets)[0];
    last = wide ? reinterpret_cast<const long long*>(offsets)[experts] : reinterpret_cast<const int*>(offsets)[experts];
    first = max(0ll, min(rows, first));
    last = max(0ll, min(rows, last));
  }
};

// ---- largest finite magnitude ---------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(QT_THREADS) mx4_amax_kernel(const T* __restrict__ x, Mx4Rows q, Mx4Range range, float* amax) {
  uint32_t top = 0;
  const long long chunks = (q.cols + 7) / 8;
  long long first, last;
  range.get(q.rows, first, last);
  const long long total = last * chunks;
  for (long long i = first * chunks + (long long)blockIdx.x * QT_THREADS + threadIdx.x; i < total; i += (long long)gridDim.x * QT_THREADS) {
    const long long row = q.rows == 1 ? 0 : i / chunks, c = i - row * chunks;
    const long long left = q.cols - c * 8;
    float v[8];
    mx4_load8(x + row * q.stride + c * 8, 0, (int)min(left, 8ll), q.vec, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t b = __float_as_uint(v[j]) & 0x7FFFFFFFu;
      top = b < 0x7F800000u ? max(top, b) : top;
    }
  }
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  // (non-negative floats order as their bits do; the largest does not depend on the order)
  if ((threadIdx.x & 31) == 0 && top) atomicMax(reinterpret_cast<unsigned*>(amax), top);
}

// ---- quantisation ---------------------------------------------------------------------------------
template <typename T, int FMT>
__global__ void __launch_bounds__(QT_THREADS)
mx4_quantize_kernel(const T* __restrict__ x, Mx4Rows q, long long total, const float* tensor_scale, const float* amax, float* own_scale,
                    uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  constexpr int PER = Mx4Fmt<FMT>::BLOCK / 8;
  float t = 1.0f;
  if constexpr (FMT == GLQB_MX4_NVFP4) {
    t = tensor_scale ? *tensor_scale : mx4_tensor_scale(*amax);
    if (!tensor_scale && blockIdx.x == 0 && threadIdx.x == 0) *own_scale = t;
  }
  const long long code_row = (q.cols + 1) / 2, scale_row = q.chunks / PER;
  // (whole warps: the threads of a block exchange their largest value)
  const long long first = (long long)blockIdx.x * QT_THREADS + threadIdx.x, warp_first = first - (threadIdx.x & 31);
  for (long long w = warp_first, i = first; w < total; w += (long long)gridDim.x * QT_THREADS, i += (long long)gridDim.x * QT_THREADS) {
    float v[8];
    const bool live = i < total;
    const long long row = q.rows == 1 ? 0 : live ? i / q.chunks : 0, c = live ? i - row * q.chunks : 0;
    const long long left = live ? q.cols - c * 8 : 0;
    if (left > 0) mx4_load8(x + row * q.stride + c * 8, 0, (int)min(left, 8ll), q.vec, v);
    else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    }
    uint32_t s;
    const uint32_t word = mx4_quantize8<FMT, false>(v, t, s);
    if (!live) continue;
    uint8_t* p = codes + row * code_row + c * 4;
    if (left >= 8 && (code_row & 3) == 0) *reinterpret_cast<uint32_t*>(p) = word;
    else {
      for (int j = 0; j < 4; ++j)
        if (2 * j < left) p[j] = (uint8_t)(word >> (8 * j));
    }
    if (c % PER == 0) scales[row * scale_row + c / PER] = (uint8_t)s;
  }
}

template <int FMT>
__global__ void __launch_bounds__(QT_THREADS)
mx4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, const float* __restrict__ tensor_scale,
                      long long rows_per_scale, Mx4Rows q, long long total, void* __restrict__ out, int out_dtype) {
  constexpr int PER = Mx4Fmt<FMT>::BLOCK / 8;
  const long long code_row = (q.cols + 1) / 2, scale_row = q.chunks / PER;
  for (long long i = (long long)blockIdx.x * QT_THREADS + threadIdx.x; i < total; i += (long long)gridDim.x * QT_THREADS) {
    const long long row = q.rows == 1 ? 0 : i / q.chunks, c = i - row * q.chunks;
    const long long left = q.cols - c * 8;
    if (left <= 0) continue;
    const uint8_t* p = codes + row * code_row + c * 4;
    uint32_t word = 0;
    if (left >= 8 && (code_row & 3) == 0) word = *reinterpret_cast<const uint32_t*>(p);
    else {
      for (int j = 0; j < 4; ++j)
        if (2 * j < left) word |= (uint32_t)p[j] << (8 * j);
    }
    const float s = mx4_scale_value<FMT>(scales[row * scale_row + c / PER]);
    float t = 1.0f;
    if constexpr (FMT == GLQB_MX4_NVFP4) t = tensor_scale[row / rows_per_scale];
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = mx4_value((word >> (4 * j)) & 15u) * s * t;
    const long long at = row * q.cols + c * 8;
    const bool whole = left >= 8 && q.vec;
    if (out_dtype == GLQB_DT_F32) {
      float* o = reinterpret_cast<float*>(out) + at;
      if (whole) {
        reinterpret_cast<float4*>(o)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(o)[1] = make_float4(v[4], v[5], v[6], v[7]);
      } else
        for (int j = 0; j < 8; ++j)
          if (j < left) o[j] = v[j];
    } else {
      uint16_t h[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        h[j] = out_dtype == GLQB_DT_F16 ? __half_as_ushort(__float2half_rn(v[j])) : __bfloat16_as_ushort(__float2bfloat16_rn(v[j]));
      uint16_t* o = reinterpret_cast<uint16_t*>(out) + at;
      if (whole)
        *reinterpret_cast<uint4*>(o) = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | (uint32_t)h[7] << 16);
      else
        for (int j = 0; j < 8; ++j)
          if (j < left) o[j] = h[j];
    }
  }
}

// ---- the weight image -----------------------------------------------------------------------------
// One thread per 32-bit word of a tile's codes, then one per scale byte; rows and values past the matrix are zeros.
template <int FMT>
__global__ void __launch_bounds__(256) mx4_pack_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int m, int n,
                                                       int k_tiles, int m_tiles, uint8_t* __restrict__ image, const uint16_t* __restrict__ tops) {
  constexpr int BLOCK = Mx4Fmt<FMT>::BLOCK, PER = MX4_K / BLOCK;
  const int kt = blockIdx.x % k_tiles;
  const long long at = blockIdx.x / k_tiles;                  // (expert, row tile)
  const int mt = (int)(at % m_tiles);
  const long long e = at / m_tiles;
  uint8_t* tile = image + (long long)blockIdx.x * mx4_tile_bytes(FMT);
  const long long code_row = (n + 1) / 2, scale_row = (n + BLOCK - 1) / BLOCK;
  for (int i = threadIdx.x; i < MX4_CODE_BYTES / 4; i += blockDim.x) {
    const int r = i / (MX4_K / 8), k = i % (MX4_K / 8) * 8, row = mt * MX4_ROWS + r, col = kt * MX4_K + k;
    uint32_t w = 0;
    if (row < m && col < n) {
      const uint8_t* p = codes + (e * m + row) * code_row + col / 2;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col + 2 * j < n) w |= (uint32_t)p[j] << (8 * j);
      if (col + 8 > n) w &= 0xFFFFFFFFu >> (4 * (col + 8 - n));
    }
    *reinterpret_cast<uint32_t*>(tile + mx4_word_offset(r, k)) = mx4_interleave(w);
  }
  for (int i = threadIdx.x; i < mx4_scale_bytes(FMT); i += blockDim.x) {
    const int r = i / PER, b = i % PER, row = mt * MX4_ROWS + r;
    const long long col = (long long)kt * PER + b;
    const bool in = row < m && col < scale_row;
    uint32_t byte = in ? scales[(e * m + row) * scale_row + col] : 0u;
    if constexpr (FMT == GLQB_MX4_MXFP4) {
      // A block of zeros (past the matrix, or of a quantised zero, whose byte is 0) gets the row's largest scale: it stays zero, and
      // the operands' scales lie close together.
      uint32_t any = 0;
      if (in) {
        const int first = kt * (MX4_K / 2) + b * (BLOCK / 2);
        const uint8_t* p = codes + (e * m + row) * code_row;
        for (int j = first; j < min(first + BLOCK / 2, (int)code_row); ++j) any |= p[j] & (2 * j + 1 < n ? 0x77u : 0x07u);
      }
      if (byte != 255u && !any) byte = row < m ? tops[(e * m_tiles + mt) * MX4_ROWS + r] & 0xFFu : 0u;
    }
    tile[MX4_CODE_BYTES + mx4_scale_offset(r, b)] = (uint8_t)byte;
  }
}
// MXFP4: the largest scale byte of every row's blocks that are numbers and not zero; + 256 for rows that have a block that is no number,
// or one so far below the largest that 2^(s - largest + 13) is no normal fp16 number.
__global__ void __launch_bounds__(256) mx4_row_top_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, long long rows, int m,
                                                          int m_pad, int n, uint16_t* __restrict__ tops) {
  const long long row = (long long)blockIdx.x * 8 + threadIdx.x / 32;          // of experts x m_pad
  if (row >= rows) return;
  const int r = (int)(row % m_pad), scale_row = (n + 31) / 32, code_row = (n + 1) / 2;
  uint32_t top = 0, low = 255, nan = 0;
  if (r < m) {
    const long long at = row / m_pad * m + r;
    for (int c = threadIdx.x % 32; c < scale_row; c += 32) {
      const uint32_t s = scales[at * scale_row + c];
      uint32_t any = 0;
      for (int j = c * 16; j < min(c * 16 + 16, code_row); ++j) any |= codes[at * code_row + j] & (2 * j + 1 < n ? 0x77u : 0x07u);
      if (s == 255u) nan = 1u;
      else if (any) { top = max(top, s); low = min(low, s); }
    }
  }
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  low = __reduce_min_sync(0xFFFFFFFFu, low);
  nan = __any_sync(0xFFFFFFFFu, nan);
  if (threadIdx.x % 32 == 0) tops[row] = (uint16_t)(top | (nan || top > low + 27u ? 256u : 0u));
}

// ---- activations of the products ------------------------------------------------------------------
// Rows that TMA cannot read (not on 16 bytes) are copied, to rows of a multiple of eight values.
__global__ void __launch_bounds__(256) mx4_align_kernel(const uint16_t* __restrict__ x, long long x_stride, long long rows, int n, int n_pad,
                                                        uint16_t* __restrict__ out) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < rows * n_pad; i += (long long)gridDim.x * 256) {
    const long long r = i / n_pad;
    const int c = (int)(i - r * n_pad);
    out[i] = c < n ? x[r * x_stride + c] : (uint16_t)0;
  }
}

// Rows of x in 4 bits, as the tiles the 4-bit product fetches (per token tile, per 256 values: tn rows of 128 bytes with the
// 128-byte swizzle, then the scales, 128 rows at a time as in the weight image).  A warp takes a row, 256 values at a time;
// values past the row are zeros, rows past a tile's are left out (their columns are not stored).
template <typename T, int FMT>
__global__ void __launch_bounds__(256) mx4_x_image_kernel(const __grid_constant__ Mx4Job J, const float* x_scale, const float* amax, float* own_scale,
                                                          int x_scales, bool vec) {
  extern __shared__ int lists[];
  int* eff = lists;
  int* pre = lists + J.experts + 1;
  mx4_groups(J, eff, pre);
  constexpr int PER = Mx4Fmt<FMT>::BLOCK / 8;
  float t = 1.0f;
  if constexpr (FMT == GLQB_MX4_NVFP4) {
    t = x_scale ? *x_scale : mx4_tensor_scale(*amax);
    if (!x_scale && blockIdx.x == 0 && threadIdx.x == 0) *own_scale = t;
  }
  const int lane = threadIdx.x & 31, end = eff[J.experts];
  const long long stage = (long long)J.tn * 128 + x_scales;
  for (int row = eff[0] + blockIdx.x * 8 + (threadIdx.x >> 5); row < end; row += gridDim.x * 8) {
    const int e = J.experts == 1 ? 0 : mx4_find(eff, J.experts, row), in = row - eff[e];
    const int per = mx4_per_tile(J.tn, eff[e + 1] - eff[e], pre[e + 1] - pre[e]), tile = pre[e] + in / per, r = in % per;
    if (tile >= J.max_tiles) continue;
    uint8_t* at = J.x_image + (long long)tile * J.k_tiles * stage;
    uint8_t* codes = at + (r >> 3) * 1024 + (r & 7) * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4;
    uint8_t* scales = at + J.tn * 128 + (r >> 7) * mx4_scale_bytes(FMT) + mx4_scale_offset(r & 127, lane / PER);
    const T* src = reinterpret_cast<const T*>(J.x) + row * J.x_stride;
    for (int k = 0; k < J.k_tiles; ++k, codes += stage, scales += stage) {
      float v[8];
      mx4_load8(src, k * MX4_K + lane * 8, J.n, vec, v);
      uint32_t s;
      *reinterpret_cast<uint32_t*>(codes) = mx4_quantize8<FMT, true>(v, t, s);
      if (lane % PER == 0) *scales = (uint8_t)s;
    }
  }
}

// Rows of no expert are zeroed.  (Offsets as mx4_groups takes them: the experts' rows are one range.)
__global__ void __launch_bounds__(256) mx4_clear_kernel(const __grid_constant__ Mx4Job J) {
  extern __shared__ int lists[];
  int* eff = lists;
  mx4_groups(J, eff, lists + J.experts + 1);
  const int first = eff[0], last = eff[J.experts], size = J.y_dtype == GLQB_DT_F32 ? 4 : 2;
  for (int row = blockIdx.x; row < J.rows; row += gridDim.x) {
    if (row >= first && row < last) {
      // (to the next row of this CTA behind the experts')
      row += (last - row - 1) / (int)gridDim.x * (int)gridDim.x;
      continue;
    }
    uint8_t* p = reinterpret_cast<uint8_t*>(J.y) + row * J.y_stride * size;
    for (int i = threadIdx.x; i < J.m; i += 256) {
      if (size == 4) reinterpret_cast<uint32_t*>(p)[i] = 0u;
      else reinterpret_cast<uint16_t*>(p)[i] = 0;
    }
  }
}

Mx4Rows rows_of(long long rows, int cols, long long stride, int format, const void* base, int elem) {
  const int block = mx4_block(format);
  Mx4Rows q;
  q.rows = rows;
  q.cols = cols;
  q.stride = stride;
  q.chunks = (cols + block - 1) / block * (block / 8);
  q.vec = reinterpret_cast<uintptr_t>(base) % 16 == 0 && (stride * elem % 16 == 0 || rows == 1);
  return q;
}
// Whole blocks, no gaps: one row (of up to 2^31 eights: what a row's count of them holds).
bool one_row(long long rows, int cols, long long stride, int format) {
  return stride == cols && cols % mx4_block(format) == 0 && rows * (cols / 8) < (1ll << 31);
}
int grid_for(long long total) { return (int)std::min<long long>((total + QT_THREADS - 1) / QT_THREADS, 148 * 64); }

// the largest finite |x| of the range's rows
int amax_launch(const void* x, int x_dtype, const Mx4Rows& q, const Mx4Range& range, float* amax, cudaStream_t stream) {
  const cudaError_t e = cudaMemsetAsync(amax, 0, 4, stream);
  if (e != cudaSuccess) return mx4_fail(GLQB_E_CUDA, "mx4 amax: %s", cudaGetErrorString(e));
  const long long n = q.rows * ((q.cols + 7) / 8);
  const int grid = (int)std::min<long long>((n + QT_THREADS - 1) / QT_THREADS, 148 * 8);
  if (x_dtype == GLQB_DT_F16) mx4_amax_kernel<__half><<<grid, QT_THREADS, 0, stream>>>((const __half*)x, q, range, amax);
  else if (x_dtype == GLQB_DT_BF16) mx4_amax_kernel<__nv_bfloat16><<<grid, QT_THREADS, 0, stream>>>((const __nv_bfloat16*)x, q, range, amax);
  else mx4_amax_kernel<float><<<grid, QT_THREADS, 0, stream>>>((const float*)x, q, range, amax);
  return GLQB_OK;
}
template <int FMT>
int quantize_launch(const void* x, int x_dtype, const Mx4Rows& q, const float* tensor_scale, float* own_scale, uint8_t* codes, uint8_t* scales,
                    cudaStream_t stream) {
  const long long total = q.rows * q.chunks;
  if (FMT == GLQB_MX4_NVFP4 && !tensor_scale) {
    const int rc = amax_launch(x, x_dtype, q, Mx4Range{nullptr, 0, 0}, own_scale + 1, stream);
    if (rc) return rc;
  }
  const int grid = grid_for(total);
  if (x_dtype == GLQB_DT_F16)
    mx4_quantize_kernel<__half, FMT><<<grid, QT_THREADS, 0, stream>>>((const __half*)x, q, total, tensor_scale, own_scale + 1, own_scale, codes, scales);
  else if (x_dtype == GLQB_DT_BF16)
    mx4_quantize_kernel<__nv_bfloat16, FMT><<<grid, QT_THREADS, 0, stream>>>((const __nv_bfloat16*)x, q, total, tensor_scale, own_scale + 1, own_scale, codes, scales);
  else
    mx4_quantize_kernel<float, FMT><<<grid, QT_THREADS, 0, stream>>>((const float*)x, q, total, tensor_scale, own_scale + 1, own_scale, codes, scales);
  return mx4_launched("mx4_quantize");
}

bool dtype_ok(int d) { return d == GLQB_DT_F16 || d == GLQB_DT_BF16 || d == GLQB_DT_F32; }
bool format_ok(int f) { return f == GLQB_MX4_MXFP4 || f == GLQB_MX4_NVFP4; }
int size_of(int dtype) { return dtype == GLQB_DT_F32 ? 4 : 2; }

}  // namespace
}  // namespace glqb

using namespace glqb;

extern "C" {

int glqb_mx4_quantize(const void* x, int32_t x_dtype, int64_t x_stride, int64_t rows, int32_t cols, int32_t format,
                      const float* tensor_scale, float* own_scale, void* codes, void* scales, void* stream_) {
  if (!format_ok(format)) return mx4_fail(GLQB_E_INVALID, "mx4_quantize: format %d", format);
  if (!dtype_ok(x_dtype)) return mx4_fail(GLQB_E_INVALID, "mx4_quantize: dtype %d", x_dtype);
  if (rows < 0 || cols < 0) return mx4_fail(GLQB_E_INVALID, "mx4_quantize: %lld x %d", (long long)rows, cols);
  if (format == GLQB_MX4_NVFP4 && !tensor_scale && !own_scale) return mx4_fail(GLQB_E_INVALID, "mx4_quantize: nvfp4 needs tensor_scale or own_scale");
  if (rows == 0 || cols == 0) return GLQB_OK;
  if (!x || !codes || !scales) return mx4_fail(GLQB_E_INVALID, "mx4_quantize: null argument");
  if (x_stride < cols && rows > 1) return mx4_fail(GLQB_E_INVALID, "mx4_quantize: rows of %d values %lld apart", cols, (long long)x_stride);
  Mx4Rows q = rows_of(rows, cols, x_stride, format, x, size_of(x_dtype));
  if (one_row(rows, cols, x_stride, format)) { q.cols = rows * cols; q.chunks = (int)(q.cols / 8); q.rows = 1; q.vec = reinterpret_cast<uintptr_t>(x) % 16 == 0; }
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  if (format == GLQB_MX4_MXFP4)
    return quantize_launch<GLQB_MX4_MXFP4>(x, x_dtype, q, tensor_scale, own_scale, (uint8_t*)codes, (uint8_t*)scales, stream);
  return quantize_launch<GLQB_MX4_NVFP4>(x, x_dtype, q, tensor_scale, own_scale, (uint8_t*)codes, (uint8_t*)scales, stream);
}

int glqb_mx4_dequantize(const void* codes, const void* scales, const float* tensor_scale, int64_t rows_per_scale, int64_t rows,
                        int32_t cols, int32_t format, void* out, int32_t out_dtype, void* stream_) {
  if (!format_ok(format)) return mx4_fail(GLQB_E_INVALID, "mx4_dequantize: format %d", format);
  if (!dtype_ok(out_dtype)) return mx4_fail(GLQB_E_INVALID, "mx4_dequantize: dtype %d", out_dtype);
  if (rows < 0 || cols < 0) return mx4_fail(GLQB_E_INVALID, "mx4_dequantize: %lld x %d", (long long)rows, cols);
  if (format == GLQB_MX4_NVFP4 && (!tensor_scale || rows_per_scale < 1)) return mx4_fail(GLQB_E_INVALID, "mx4_dequantize: nvfp4 needs tensor_scale");
  if (rows == 0 || cols == 0) return GLQB_OK;
  if (!codes || !scales || !out) return mx4_fail(GLQB_E_INVALID, "mx4_dequantize: null argument");
  Mx4Rows q = rows_of(rows, cols, cols, format, out, size_of(out_dtype));
  if (one_row(rows, cols, cols, format) && (format == GLQB_MX4_MXFP4 || rows_per_scale >= rows)) {
    q.cols = rows * cols;
    q.chunks = (int)(q.cols / 8);
    q.rows = 1;
    q.vec = reinterpret_cast<uintptr_t>(out) % 16 == 0;
  }
  const long long total = q.rows * q.chunks;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  if (format == GLQB_MX4_MXFP4)
    mx4_dequantize_kernel<GLQB_MX4_MXFP4><<<grid_for(total), QT_THREADS, 0, stream>>>((const uint8_t*)codes, (const uint8_t*)scales, nullptr, 1, q, total, out, out_dtype);
  else
    mx4_dequantize_kernel<GLQB_MX4_NVFP4><<<grid_for(total), QT_THREADS, 0, stream>>>((const uint8_t*)codes, (const uint8_t*)scales, tensor_scale, rows_per_scale, q, total, out, out_dtype);
  return mx4_launched("mx4_dequantize");
}

size_t glqb_mx4_image_bytes(int32_t format, int32_t experts, int32_t m, int32_t n) {
  if (!format_ok(format) || experts < 1 || m < 1 || n < 1) return 0;
  const size_t mt = ((size_t)m + MX4_ROWS - 1) / MX4_ROWS, kt = ((size_t)n + MX4_K - 1) / MX4_K;
  return (size_t)experts * mt * (kt * mx4_tile_bytes(format) + (format == GLQB_MX4_MXFP4 ? 2 * MX4_ROWS : 0));
}

int glqb_mx4_pack(const void* codes, const void* scales, int32_t format, int32_t experts, int32_t m, int32_t n, void* image,
                  void* stream_) {
  if (!format_ok(format)) return mx4_fail(GLQB_E_INVALID, "mx4_pack: format %d", format);
  if (experts < 1 || m < 1 || n < 1) return mx4_fail(GLQB_E_INVALID, "mx4_pack: %d x %d x %d", experts, m, n);
  if (!codes || !scales || !image) return mx4_fail(GLQB_E_INVALID, "mx4_pack: null argument");
  if (reinterpret_cast<uintptr_t>(image) % 128) return mx4_fail(GLQB_E_INVALID, "mx4_pack: the image must be 128-byte aligned");
  const int mt = (m + MX4_ROWS - 1) / MX4_ROWS, kt = (n + MX4_K - 1) / MX4_K;
  const long long tiles = (long long)experts * mt * kt;
  if (tiles >= (1ll << 31)) return mx4_fail(GLQB_E_INVALID, "mx4_pack: %d x %d x %d is more than 2^31 tiles", experts, m, n);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  if (format == GLQB_MX4_MXFP4) {
    const long long rows = (long long)experts * mt * MX4_ROWS;
    uint16_t* tops = (uint16_t*)((uint8_t*)image + tiles * mx4_tile_bytes(format));
    mx4_row_top_kernel<<<(unsigned)(rows / 8), 256, 0, stream>>>((const uint8_t*)codes, (const uint8_t*)scales, rows, m, mt * MX4_ROWS, n, tops);
    mx4_pack_kernel<GLQB_MX4_MXFP4><<<(unsigned)tiles, 256, 0, stream>>>((const uint8_t*)codes, (const uint8_t*)scales, m, n, kt, mt, (uint8_t*)image, tops);
  } else {
    mx4_pack_kernel<GLQB_MX4_NVFP4><<<(unsigned)tiles, 256, 0, stream>>>((const uint8_t*)codes, (const uint8_t*)scales, m, n, kt, mt, (uint8_t*)image, nullptr);
  }
  return mx4_launched("mx4_pack");
}

// What a call launches, by its sizes alone.
struct Form {
  int tn, max_tiles, split, pair, x_scales, n_pad;
  bool align, mv;
  size_t image, bytes;        // of the workspace: x in 4 bits or aligned, then two floats
};
struct Device { std::atomic<int> sms; std::atomic<int*> status; };
static Device* device() {
  static Device known[64];
  Device& d = known[mx4_device()];
  if (d.sms.load(std::memory_order_acquire) == 0) {
    int n = 0;
    int* p = nullptr;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, mx4_device()) != cudaSuccess || n < 1 ||
        cudaGetSymbolAddress(reinterpret_cast<void**>(&p), g_mx4_status) != cudaSuccess)
      return nullptr;
    d.status.store(p, std::memory_order_relaxed);
    d.sms.store(n, std::memory_order_release);
  }
  return &d;
}
constexpr int MV_MAX_ROWS = 16;     // rows (an expert's, on average) up to which the streaming kernel runs
static Form form_of(const GlqbMx4Weight* w, long long rows, long long x_stride, const void* x, int quantize, int sms) {
  Form f = {};
  const int avg = (int)((rows + w->experts - 1) / w->experts);
  f.mv = !quantize && avg <= MV_MAX_ROWS;
  const int most = quantize ? (w->format == GLQB_MX4_MXFP4 ? 192 : 160) : 192;
  // token tiles: a matrix's rows split evenly; of experts up to twice their average, so that most have one tile
  if (f.mv) f.tn = avg > (w->experts == 1 ? 8 : 4) ? 16 : 8;
  else if (w->experts == 1) f.tn = (int)(((rows + (rows + most - 1) / most - 1) / ((rows + most - 1) / most) + 15) / 16 * 16);
  else f.tn = std::min(most, (2 * avg + 15) / 16 * 16);
  f.max_tiles = w->experts == 1 ? (int)((rows + f.tn - 1) / f.tn) : (int)(rows / f.tn + std::min<long long>(w->experts, rows));
  const long long mt = (w->m + MX4_ROWS - 1) / MX4_ROWS, kt = (w->n + MX4_K - 1) / MX4_K, tiles = f.max_tiles * mt;
  // CTAs that share a tile's sum: as many as the SMs hold at once
  f.split = (int)std::max<long long>(1, std::min<long long>(std::min<long long>(8, kt), (f.mv ? 2 : 1) * sms / std::max<long long>(1, tiles)));
  f.pair = !quantize && !f.mv && f.split == 1 && f.tn >= 96 && mt > 1;
  if (quantize) {
    f.x_scales = mx4_x_scale_bytes(w->format, f.tn);
    f.image = (size_t)f.max_tiles * kt * ((size_t)f.tn * 128 + f.x_scales);
    f.bytes = f.image + 256;
  } else if (reinterpret_cast<uintptr_t>(x) % 16 || (rows > 1 && x_stride % 8) || (f.mv && w->n % 8)) {
    f.align = true;
    f.n_pad = (w->n + 7) / 8 * 8;
    f.bytes = (size_t)rows * f.n_pad * 2;
  }
  return f;
}

size_t glqb_mx4_workspace_bytes(const GlqbMx4Weight* w, int64_t rows, int64_t x_stride, const void* x, int32_t quantize) {
  if (!w || !format_ok(w->format) || rows <= 0 || rows >= (1ll << 31) || w->experts < 1 || w->m < 1 || w->n < 1) return 0;
  return form_of(w, rows, x_stride, x, quantize, 1).bytes;      // (what a call needs does not depend on the SMs)
}

int glqb_mx4_product(const GlqbMx4Weight* w, const void* x, int32_t x_dtype, int64_t x_stride, int64_t rows,
                     const void* offsets, int32_t offsets_are_int64, int32_t quantize, const float* x_scale,
                     void* y, int32_t y_dtype, int64_t y_stride, int32_t accumulate, int32_t clear_rest,
                     void* workspace, size_t workspace_bytes, void* stream_) {
  if (!w || !format_ok(w->format)) return mx4_fail(GLQB_E_INVALID, "mx4_product: format");
  if (w->experts < 1 || w->experts > MX4_MAX_EXPERTS || w->m < 1 || w->n < 1)
    return mx4_fail(GLQB_E_INVALID, "mx4_product: %d x %d x %d (at most %d experts)", w->experts, w->m, w->n, MX4_MAX_EXPERTS);
  if (!offsets && w->experts != 1) return mx4_fail(GLQB_E_INVALID, "mx4_product: %d experts need offsets", w->experts);
  if (!dtype_ok(x_dtype) || !dtype_ok(y_dtype)) return mx4_fail(GLQB_E_INVALID, "mx4_product: dtype");
  if (!quantize && x_dtype == GLQB_DT_F32) return mx4_fail(GLQB_E_INVALID, "mx4_product: fp32 activations are served quantised only");
  if (rows < 0 || rows >= (1ll << 31)) return mx4_fail(GLQB_E_INVALID, "mx4_product: %lld rows", (long long)rows);
  if (rows == 0) return GLQB_OK;
  if (!w->image || !x || !y || (w->format == GLQB_MX4_NVFP4 && !w->tensor_scale)) return mx4_fail(GLQB_E_INVALID, "mx4_product: null argument");
  if (rows > 1 && (x_stride < w->n || y_stride < w->m)) return mx4_fail(GLQB_E_INVALID, "mx4_product: rows overlap");
  const Device* d = device();
  const int sms = d ? d->sms.load(std::memory_order_relaxed) : 1;      // (the workspace does not depend on it)
  const Form f = form_of(w, rows, x_stride, x, quantize, sms);
  if (workspace_bytes < f.bytes || (f.bytes && !workspace))
    return mx4_fail(GLQB_E_WORKSPACE, "mx4_product: workspace of %zu bytes, %zu needed", workspace_bytes, f.bytes);
  if (!d) return mx4_fail(GLQB_E_CUDA, "mx4_product: no device");
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  cudaError_t e = cudaSuccess;
  Mx4Job J = {};
  J.m = w->m;
  J.n = w->n;
  J.m_tiles = (w->m + MX4_ROWS - 1) / MX4_ROWS;
  J.k_tiles = (w->n + MX4_K - 1) / MX4_K;
  J.image = (const uint8_t*)w->image;
  J.tops = (const uint16_t*)(J.image + (size_t)w->experts * J.m_tiles * J.k_tiles * mx4_tile_bytes(w->format));
  J.w_scale = w->tensor_scale;
  J.offsets = offsets;
  J.wide = offsets_are_int64;
  J.experts = w->experts;
  J.rows = (int)rows;
  J.tn = f.tn;
  J.max_tiles = f.max_tiles;
  J.split = f.split;
  J.pair = f.pair;
  J.y = y;
  J.y_stride = y_stride;
  J.y_dtype = y_dtype;
  J.accumulate = accumulate;
  J.y_wide = y_dtype != GLQB_DT_F32 && !accumulate && reinterpret_cast<uintptr_t>(y) % 16 == 0 && (rows == 1 || y_stride % 8 == 0);
  J.x = x;
  J.x_stride = x_stride;
  J.status = d->status.load(std::memory_order_relaxed);
  const size_t lists = (size_t)(J.experts + 1) * 8;
  if (offsets && clear_rest) mx4_clear_kernel<<<(unsigned)std::min<long long>(rows, 148), 256, lists, stream>>>(J);
  if (!quantize) {
    if (f.align) {
      mx4_align_kernel<<<grid_for(rows * f.n_pad), 256, 0, stream>>>((const uint16_t*)x, x_stride, rows, w->n, f.n_pad, (uint16_t*)workspace);
      J.x = workspace;
      J.x_stride = f.n_pad;
    }
    if (f.mv) {
      if (f.align) J.n = f.n_pad;
      e = mx4_mv_launch(w->format, x_dtype == GLQB_DT_BF16, J, sms, stream);
      return e == cudaSuccess ? GLQB_OK : mx4_fail(GLQB_E_CUDA, "mx4_product: %s", cudaGetErrorString(e));
    }
    const char* what = nullptr;
    e = mx4_gemm16_launch(w->format, x_dtype == GLQB_DT_BF16, J, sms, stream, &what);
    if (e != cudaSuccess) return mx4_fail(GLQB_E_CUDA, "mx4_product: %s", what ? what : cudaGetErrorString(e));
    return mx4_launched("mx4_product");
  }
  J.x_image = (uint8_t*)workspace;
  float* own = (float*)((uint8_t*)workspace + f.image);
  J.x_scale = x_scale ? x_scale : own;
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (rows == 1 || x_stride * size_of(x_dtype) % 16 == 0);
  if (w->format == GLQB_MX4_NVFP4 && !x_scale) {
    const Mx4Rows q = rows_of(rows, w->n, x_stride, w->format, x, size_of(x_dtype));
    const int rc = amax_launch(x, x_dtype, q, Mx4Range{offsets, offsets_are_int64, w->experts}, own + 1, stream);
    if (rc) return rc;
  }
  const int grid = (int)std::min<long long>((rows + 7) / 8, 148 * 8);
  auto image = [&](auto fmt) {
    constexpr int FMT = decltype(fmt)::value;
    if (x_dtype == GLQB_DT_F16) mx4_x_image_kernel<__half, FMT><<<grid, 256, lists, stream>>>(J, x_scale, own + 1, own, f.x_scales, vec);
    else if (x_dtype == GLQB_DT_BF16) mx4_x_image_kernel<__nv_bfloat16, FMT><<<grid, 256, lists, stream>>>(J, x_scale, own + 1, own, f.x_scales, vec);
    else mx4_x_image_kernel<float, FMT><<<grid, 256, lists, stream>>>(J, x_scale, own + 1, own, f.x_scales, vec);
  };
  if (w->format == GLQB_MX4_MXFP4) image(std::integral_constant<int, GLQB_MX4_MXFP4>());
  else image(std::integral_constant<int, GLQB_MX4_NVFP4>());
  e = mx4_gemm4_launch(w->format, J, sms, stream);
  if (e != cudaSuccess) return mx4_fail(GLQB_E_CUDA, "mx4_product: %s", cudaGetErrorString(e));
  return mx4_launched("mx4_product");
}

int glqb_mx4_status(int32_t* status_out) {
  int code = 0;
  const int zero = 0;
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&code, g_mx4_status, sizeof code);
  if (e == cudaSuccess && code) e = cudaMemcpyToSymbol(g_mx4_status, &zero, sizeof zero);
  if (e != cudaSuccess) return mx4_fail(GLQB_E_CUDA, "mx4_status: %s", cudaGetErrorString(e));
  if (status_out) *status_out = code;
  return code ? mx4_fail(GLQB_E_DEVICE, "a bounded wait in a 4-bit product gave up (status %d): results are invalid", code) : GLQB_OK;
}

}  // extern "C"
