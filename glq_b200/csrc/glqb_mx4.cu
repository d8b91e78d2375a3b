// Microscaled 4-bit floating point: quantisation and back, the weight image, and the C entry points (include/glq_b200.h).
#include "glqb_mx4.cuh"
#include <algorithm>
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

// Rows and columns of a call.  Rows that follow one another without a gap and end on whole blocks are one long row: their
// codes and scales do too.
struct Mx4Rows {
  long long rows, stride;     // elements between rows
  long long cols;
  int chunks;                 // eights of values per row, whole blocks
  bool vec;
};

// The rows that belong to an expert: offsets[0] .. offsets[experts] - 1, held to those there are.
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
                                                       int k_tiles, int m_tiles, uint8_t* __restrict__ image) {
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
    tile[MX4_CODE_BYTES + mx4_scale_offset(r, b)] = row < m && col < scale_row ? scales[(e * m + row) * scale_row + col] : 0;
  }
}
// MXFP4: the largest scale byte of every row that is a number
__global__ void __launch_bounds__(256) mx4_row_top_kernel(const uint8_t* __restrict__ scales, long long rows, int m, int m_pad, int scale_row,
                                                          uint8_t* __restrict__ tops) {
  const long long row = (long long)blockIdx.x * 8 + threadIdx.x / 32;          // of experts x m_pad
  if (row >= rows) return;
  const int r = (int)(row % m_pad);
  uint32_t top = 0;
  if (r < m)
    for (int c = threadIdx.x % 32; c < scale_row; c += 32) {
      const uint32_t s = scales[(row / m_pad * m + r) * scale_row + c];
      top = s < 255u ? max(top, s) : top;
    }
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  if (threadIdx.x % 32 == 0) tops[row] = (uint8_t)top;
}

// ---- the product, plainly: a warp sums eight rows of x against one row of the matrix in fp32 -------
template <int FMT, typename T>
__global__ void __launch_bounds__(256)
mx4_plain_kernel(const uint8_t* __restrict__ image, const float* __restrict__ tensor_scale, int m, int n, int k_tiles, int m_tiles,
                 const T* __restrict__ x, long long x_stride, long long rows, const void* offsets, int wide, const float* x_scale,
                 uint8_t* y, int y_dtype, long long y_stride, int accumulate) {
  constexpr int BLOCK = Mx4Fmt<FMT>::BLOCK;
  const int row = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x % 32, e = blockIdx.z;
  if (row >= m) return;
  long long begin = 0, end = rows;
  if (offsets) {
    begin = wide ? reinterpret_cast<const long long*>(offsets)[e] : reinterpret_cast<const int*>(offsets)[e];
    end = wide ? reinterpret_cast<const long long*>(offsets)[e + 1] : reinterpret_cast<const int*>(offsets)[e + 1];
    begin = max(0ll, min(rows, begin));
    end = max(0ll, min(rows, end));
  }
  const uint8_t* tiles = image + ((long long)e * m_tiles + row / MX4_ROWS) * k_tiles * mx4_tile_bytes(FMT);
  const int r = row % MX4_ROWS;
  float scale = 1.0f;
  if constexpr (FMT == GLQB_MX4_NVFP4) scale = tensor_scale[e] * (x_scale ? *x_scale : 1.0f);
  for (long long t0 = begin + blockIdx.y * 8ll; t0 < end; t0 += gridDim.y * 8ll) {
    float acc[8] = {};
    for (int k = lane * 8; k < n; k += 256) {
      const uint8_t* tile = tiles + (long long)(k / MX4_K) * mx4_tile_bytes(FMT);
      const int kk = k % MX4_K;
      const uint32_t w = *reinterpret_cast<const uint32_t*>(tile + mx4_word_offset(r, kk));
      const float s = mx4_scale_value<FMT>(tile[MX4_CODE_BYTES + mx4_scale_offset(r, kk / BLOCK)]);
      for (int j = 0; j < 8 && k + j < n; ++j) {
        const float v = mx4_value(w >> (4 * ((j >> 1) + 4 * (j & 1))) & 15u) * s;
        for (int t = 0; t < 8; ++t)
          if (t0 + t < end) acc[t] += v * (float)x[(t0 + t) * x_stride + k + j];
      }
    }
    for (int t = 0; t < 8; ++t) {
      float a = acc[t];
      for (int d = 16; d; d >>= 1) a += __shfl_xor_sync(0xFFFFFFFFu, a, d);
      if (lane || t0 + t >= end) continue;
      a *= scale;
      const long long at = (t0 + t) * y_stride + row;
      if (y_dtype == GLQB_DT_F32) {
        float* o = reinterpret_cast<float*>(y) + at;
        *o = accumulate ? *o + a : a;
      } else if (y_dtype == GLQB_DT_F16) {
        __half* o = reinterpret_cast<__half*>(y) + at;
        *o = __float2half_rn(accumulate ? __half2float(*o) + a : a);
      } else {
        __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(y) + at;
        *o = __float2bfloat16_rn(accumulate ? __bfloat162float(*o) + a : a);
      }
    }
  }
}

// rows of no expert
__global__ void __launch_bounds__(256) mx4_clear_kernel(const void* offsets, int wide, int experts, long long rows, int m, uint8_t* y, int size,
                                                        long long y_stride) {
  const long long row = blockIdx.x;
  __shared__ int owned;
  if (threadIdx.x == 0) owned = 0;
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += blockDim.x) {
    const long long b = wide ? reinterpret_cast<const long long*>(offsets)[e] : reinterpret_cast<const int*>(offsets)[e];
    const long long f = wide ? reinterpret_cast<const long long*>(offsets)[e + 1] : reinterpret_cast<const int*>(offsets)[e + 1];
    if (row >= b && row < f) owned = 1;
  }
  __syncthreads();
  if (owned) return;
  for (int i = threadIdx.x; i < m * size; i += blockDim.x) y[row * y_stride * size + i] = 0;
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

template <int FMT>
int quantize_launch(const void* x, int x_dtype, const Mx4Rows& q, const Mx4Range& range, const float* tensor_scale, float* own_scale, uint8_t* codes,
                    uint8_t* scales, cudaStream_t stream) {
  const long long total = q.rows * q.chunks;
  if (FMT == GLQB_MX4_NVFP4 && !tensor_scale) {
    const cudaError_t e = cudaMemsetAsync(own_scale + 1, 0, 4, stream);
    if (e != cudaSuccess) return mx4_fail(GLQB_E_CUDA, "mx4_quantize: %s", cudaGetErrorString(e));
    const long long n = q.rows * ((q.cols + 7) / 8);
    const int grid = (int)std::min<long long>((n + QT_THREADS - 1) / QT_THREADS, 148 * 8);
    if (x_dtype == GLQB_DT_F16) mx4_amax_kernel<__half><<<grid, QT_THREADS, 0, stream>>>((const __half*)x, q, range, own_scale + 1);
    else if (x_dtype == GLQB_DT_BF16) mx4_amax_kernel<__nv_bfloat16><<<grid, QT_THREADS, 0, stream>>>((const __nv_bfloat16*)x, q, range, own_scale + 1);
    else mx4_amax_kernel<float><<<grid, QT_THREADS, 0, stream>>>((const float*)x, q, range, own_scale + 1);
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

static int quantize_rows(const void* x, int32_t x_dtype, int64_t x_stride, int64_t rows, int32_t cols, int32_t format, const Mx4Range& range,
                         const float* tensor_scale, float* own_scale, void* codes, void* scales, void* stream_) {
  if (!format_ok(format)) return mx4_fail(GLQB_E_INVALID, "mx4_quantize: format %d", format);
  if (!dtype_ok(x_dtype)) return mx4_fail(GLQB_E_INVALID, "mx4_quantize: dtype %d", x_dtype);
  if (rows < 0 || cols < 0) return mx4_fail(GLQB_E_INVALID, "mx4_quantize: %lld x %d", (long long)rows, cols);
  if (format == GLQB_MX4_NVFP4 && !tensor_scale && !own_scale) return mx4_fail(GLQB_E_INVALID, "mx4_quantize: nvfp4 needs tensor_scale or own_scale");
  if (rows == 0 || cols == 0) return GLQB_OK;
  if (!x || !codes || !scales) return mx4_fail(GLQB_E_INVALID, "mx4_quantize: null argument");
  if (x_stride < cols && rows > 1) return mx4_fail(GLQB_E_INVALID, "mx4_quantize: rows of %d values %lld apart", cols, (long long)x_stride);
  Mx4Rows q = rows_of(rows, cols, x_stride, format, x, size_of(x_dtype));
  if (!range.offsets && one_row(rows, cols, x_stride, format)) { q.cols = rows * cols; q.chunks = (int)(q.cols / 8); q.rows = 1; q.vec = reinterpret_cast<uintptr_t>(x) % 16 == 0; }
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  if (format == GLQB_MX4_MXFP4)
    return quantize_launch<GLQB_MX4_MXFP4>(x, x_dtype, q, range, tensor_scale, own_scale, (uint8_t*)codes, (uint8_t*)scales, stream);
  return quantize_launch<GLQB_MX4_NVFP4>(x, x_dtype, q, range, tensor_scale, own_scale, (uint8_t*)codes, (uint8_t*)scales, stream);
}

int glqb_mx4_quantize(const void* x, int32_t x_dtype, int64_t x_stride, int64_t rows, int32_t cols, int32_t format,
                      const float* tensor_scale, float* own_scale, void* codes, void* scales, void* stream_) {
  return quantize_rows(x, x_dtype, x_stride, rows, cols, format, Mx4Range{nullptr, 0, 0}, tensor_scale, own_scale, codes, scales, stream_);
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
  return (size_t)experts * mt * (kt * mx4_tile_bytes(format) + (format == GLQB_MX4_MXFP4 ? MX4_ROWS : 0));
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
    mx4_pack_kernel<GLQB_MX4_MXFP4><<<(unsigned)tiles, 256, 0, stream>>>((const uint8_t*)codes, (const uint8_t*)scales, m, n, kt, mt, (uint8_t*)image);
    const long long rows = (long long)experts * mt * MX4_ROWS;
    mx4_row_top_kernel<<<(unsigned)(rows / 8), 256, 0, stream>>>((const uint8_t*)scales, rows, m, mt * MX4_ROWS, (n + 31) / 32,
                                                                 (uint8_t*)image + tiles * mx4_tile_bytes(format));
  } else {
    mx4_pack_kernel<GLQB_MX4_NVFP4><<<(unsigned)tiles, 256, 0, stream>>>((const uint8_t*)codes, (const uint8_t*)scales, m, n, kt, mt, (uint8_t*)image);
  }
  return mx4_launched("mx4_pack");
}

// quantised activations: codes, scales, the tensor's scale
static size_t x_bytes(const GlqbMx4Weight* w, int64_t rows, size_t* scales_at, size_t* own_at, size_t* back_at) {
  const size_t codes = ((size_t)rows * ((w->n + 1) / 2) + 255) / 256 * 256;
  const size_t scales = ((size_t)rows * ((w->n + mx4_block(w->format) - 1) / mx4_block(w->format)) + 255) / 256 * 256;
  *scales_at = codes;
  *own_at = codes + scales;
  *back_at = codes + scales + 256;
  return *back_at + (size_t)rows * w->n * 4;
}

size_t glqb_mx4_workspace_bytes(const GlqbMx4Weight* w, int64_t rows, int64_t x_stride, const void* x, int32_t quantize) {
  if (!w || !format_ok(w->format) || rows < 0 || !quantize) return 0;
  size_t a, b, c;
  return x_bytes(w, rows, &a, &b, &c);
}

int glqb_mx4_product(const GlqbMx4Weight* w, const void* x, int32_t x_dtype, int64_t x_stride, int64_t rows,
                     const void* offsets, int32_t offsets_are_int64, int32_t quantize, const float* x_scale,
                     void* y, int32_t y_dtype, int64_t y_stride, int32_t accumulate, int32_t clear_rest,
                     void* workspace, size_t workspace_bytes, void* stream_) {
  if (!w || !format_ok(w->format)) return mx4_fail(GLQB_E_INVALID, "mx4_product: format");
  if (w->experts < 1 || w->m < 1 || w->n < 1) return mx4_fail(GLQB_E_INVALID, "mx4_product: %d x %d x %d", w->experts, w->m, w->n);
  if (!offsets && w->experts != 1) return mx4_fail(GLQB_E_INVALID, "mx4_product: %d experts need offsets", w->experts);
  if (!dtype_ok(x_dtype) || !dtype_ok(y_dtype)) return mx4_fail(GLQB_E_INVALID, "mx4_product: dtype");
  if (!quantize && x_dtype == GLQB_DT_F32) return mx4_fail(GLQB_E_INVALID, "mx4_product: fp32 activations are served quantised only");
  if (rows < 0 || rows >= (1ll << 31)) return mx4_fail(GLQB_E_INVALID, "mx4_product: %lld rows", (long long)rows);
  if (rows == 0) return GLQB_OK;
  if (!w->image || !x || !y || (w->format == GLQB_MX4_NVFP4 && !w->tensor_scale)) return mx4_fail(GLQB_E_INVALID, "mx4_product: null argument");
  if (rows > 1 && (x_stride < w->n || y_stride < w->m)) return mx4_fail(GLQB_E_INVALID, "mx4_product: rows overlap");
  if (workspace_bytes < glqb_mx4_workspace_bytes(w, rows, x_stride, x, quantize) || (quantize && !workspace))
    return mx4_fail(GLQB_E_WORKSPACE, "mx4_product: workspace of %zu bytes, %zu needed", workspace_bytes, glqb_mx4_workspace_bytes(w, rows, x_stride, x, quantize));
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const int mt = (w->m + MX4_ROWS - 1) / MX4_ROWS, kt = (w->n + MX4_K - 1) / MX4_K;
  if (offsets && clear_rest)
    mx4_clear_kernel<<<(unsigned)rows, 256, 0, stream>>>(offsets, offsets_are_int64, w->experts, rows, w->m, (uint8_t*)y, size_of(y_dtype), y_stride);
  const float* xs = nullptr;
  if (quantize) {
    size_t scales_at, own_at, back_at;
    x_bytes(w, rows, &scales_at, &own_at, &back_at);
    uint8_t* ws = (uint8_t*)workspace;
    float* own = (float*)(ws + own_at);
    int rc = quantize_rows(x, x_dtype, x_stride, rows, w->n, w->format, Mx4Range{offsets, offsets_are_int64, w->experts}, x_scale, own, ws, ws + scales_at, stream_);
    if (rc) return rc;
    xs = x_scale ? x_scale : own;
    rc = glqb_mx4_dequantize(ws, ws + scales_at, xs, rows, rows, w->n, w->format, ws + back_at, GLQB_DT_F32, stream_);
    if (rc) return rc;
    x = ws + back_at;
    x_stride = w->n;
    x_dtype = GLQB_DT_F32;
  }
  const dim3 grid((unsigned)((w->m + 7) / 8), (unsigned)std::min<long long>((rows + 7) / 8, 1024), (unsigned)w->experts);
  auto launch = [&](auto fmt) {
    constexpr int FMT = decltype(fmt)::value;
    if (x_dtype == GLQB_DT_F16)
      mx4_plain_kernel<FMT, __half><<<grid, 256, 0, stream>>>((const uint8_t*)w->image, w->tensor_scale, w->m, w->n, kt, mt, (const __half*)x, x_stride, rows, offsets,
                                                              offsets_are_int64, nullptr, (uint8_t*)y, y_dtype, y_stride, accumulate);
    else if (x_dtype == GLQB_DT_BF16)
      mx4_plain_kernel<FMT, __nv_bfloat16><<<grid, 256, 0, stream>>>((const uint8_t*)w->image, w->tensor_scale, w->m, w->n, kt, mt, (const __nv_bfloat16*)x, x_stride, rows,
                                                                     offsets, offsets_are_int64, nullptr, (uint8_t*)y, y_dtype, y_stride, accumulate);
    else
      mx4_plain_kernel<FMT, float><<<grid, 256, 0, stream>>>((const uint8_t*)w->image, w->tensor_scale, w->m, w->n, kt, mt, (const float*)x, x_stride, rows, offsets,
                                                             offsets_are_int64, nullptr, (uint8_t*)y, y_dtype, y_stride, accumulate);
  };
  if (w->format == GLQB_MX4_MXFP4) launch(std::integral_constant<int, GLQB_MX4_MXFP4>());
  else launch(std::integral_constant<int, GLQB_MX4_NVFP4>());
  return mx4_launched("mx4_product");
}

int glqb_mx4_status(int32_t* status_out) {
  if (status_out) *status_out = 0;
  return GLQB_OK;
}

}  // extern "C"
