// Microscaled 4-bit floating point: quantisation and back, the weight image, and the C entry points (include/glq_b200.h).
#include "glqb_mx4_gemm.cuh"
#include <algorithm>
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <mutex>

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
constexpr int MX4_MAX_SIZE = 1 << 30, MX4_MAX_ROWS = 0x7FFF0000;   // (sums with a tile's size stay 32-bit)

__device__ int g_mx4_status;   // 0, or what gave up (ST_GAVE_UP_*): products have no plan to keep it in

// Rows and columns of a call.  Rows that follow one another without a gap and end on whole blocks are one long row: their
// codes and scales do too.
struct Mx4Rows {
  long long rows, stride;     // elements between rows
  long long cols;
  long long chunks;           // sixteens of values per row, whole blocks
  long long full;             // those that have all sixteen
  uint32_t magic;             // i / chunks = i * magic / 2^(32 + shift) for i < 2^31 (see rows_of)
  int rest, shift;            // values behind the full ones
};

// The rows of the experts: from offsets[0] up to the largest offset, held to those there are.  (mx4_groups counts an offset below one before
// it as that one: its experts end at the largest, wherever that stands.)
struct Mx4Range {
  const void* offsets;        // null: all
  int wide, experts;
  __device__ long long at(int e, long long rows) const {
    const long long o = wide ? reinterpret_cast<const long long*>(offsets)[e] : reinterpret_cast<const int*>(offsets)[e];
    return max(0ll, min(rows, o));
  }
  // By all threads of a block; tops: a word per warp.  (rows < 2^31)
  __device__ void get(long long rows, long long& first, long long& last, uint32_t* tops) const {
    first = 0;
    last = rows;
    if (!offsets) return;
    uint32_t top = 0;
    for (int e = threadIdx.x; e <= experts; e += blockDim.x) top = max(top, (uint32_t)at(e, rows));
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    last = __reduce_max_sync(0xFFFFFFFFu, (threadIdx.x & 31) < blockDim.x / 32 ? tops[threadIdx.x & 31] : 0u);
    first = at(0, rows);
    __syncthreads();          // (tops is used again)
  }
};

// Sixteens of values that a thread takes at once, their loads in front of everything else.  I: the type of a sixteenth's index (64-bit
// divisions only where there are more than 2^31).  What bounds these kernels next to HBM is the instructions around the values
// (by eights 112 per warp and eight for MXFP4, half of them addresses and scales): sixteens share them out further.
constexpr int QT_BATCH = 2;
template <typename I>
__device__ __forceinline__ void place(const Mx4Rows& q, I i, I& row, I& c) {
  if constexpr (sizeof(I) == 4) row = q.chunks == 1 ? i : __umulhi(i, q.magic) >> q.shift;
  else row = q.rows == 1 ? (I)0 : i / (I)q.chunks;
  c = i - row * (I)q.chunks;
}
// values of a row from its sixteen c on, at most sixteen
template <typename I>
__device__ __forceinline__ int values_at(const Mx4Rows& q, I c) { return c < (I)q.full ? 16 : c == (I)q.full ? q.rest : 0; }

// ---- largest finite magnitude ---------------------------------------------------------------------
// A part per CTA; those who need the whole reduce the parts (no atomics, nothing to clear beforehand).  HBM bound: 88 MB of fp32 in 20 us.
constexpr int AMAX_PARTS = 296, AMAX_THREADS = 1024;      // (two for each of 148 SMs)
static_assert(AMAX_PARTS + 1 == GLQB_MX4_SCALE_FLOATS, "");
template <typename T, typename I>
__global__ void __launch_bounds__(AMAX_THREADS) mx4_amax_kernel(const T* x, Mx4Rows q, Mx4Range range, float* parts) {
  pdl_wait();
  pdl_trigger();
  __shared__ uint32_t tops[AMAX_THREADS / 32];
  uint32_t top = 0;
  long long first, last;
  range.get(q.rows, first, last, tops);
  const I end = (I)(last * q.chunks), step = (I)gridDim.x * AMAX_THREADS;
  for (I b = (I)(first * q.chunks) + (I)blockIdx.x * AMAX_THREADS + threadIdx.x; b < end; b += step * QT_BATCH) {
    Mx4Raw<T> raw[QT_BATCH];
#pragma unroll
    for (int j = 0; j < QT_BATCH; ++j) {
      const I i = b + j * step;
      I row, c;
      place(q, i, row, c);
      raw[j].load(x + (long long)row * q.stride + (long long)c * 16, i < end ? values_at(q, c) : 0);
    }
#pragma unroll
    for (int j = 0; j < QT_BATCH; ++j) {
      const uint32_t all = raw[j].top();
      if (all < 0x7F800000u) top = max(top, all);
      else {                                                        // the finite ones among them
        float v[16];
        raw[j].get(v);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t w = __float_as_uint(v[e]) & 0x7FFFFFFFu;
          top = w < 0x7F800000u ? max(top, w) : top;
        }
      }
    }
  }
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x < 32) {
    top = __reduce_max_sync(0xFFFFFFFFu, threadIdx.x < AMAX_THREADS / 32 ? tops[threadIdx.x] : 0u);
    if (threadIdx.x == 0) parts[blockIdx.x] = __uint_as_float(top);
  }
}
// The tensor's scale for all threads of a block of 256: given, or from the parts; the first block leaves it in own_scale[0].
__device__ __forceinline__ float whole_scale(const float* given, float* own_scale, int parts) {
  if (given) return *given;
  uint32_t top = 0;
  for (int i = threadIdx.x; i < parts; i += QT_THREADS) top = max(top, __float_as_uint(own_scale[1 + i]));      // (non-negative: ordered as their bits)
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  __shared__ uint32_t tops[QT_THREADS / 32];
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < QT_THREADS / 32; ++i) top = max(top, tops[i]);
  const float t = mx4_tensor_scale(__uint_as_float(top));
  if (blockIdx.x == 0 && threadIdx.x == 0) *own_scale = t;
  return t;
}

// ---- quantisation ---------------------------------------------------------------------------------
// 2 or 4 bytes in and 0.53 or 0.56 out per value: 2048 x 14336 bf16 to MXFP4 and back 24.9 us = 6.0 TB/s; to NVFP4 the instructions of
// the scales and of two conversions per value count as well (5376 x 4100 fp32 25 us of 101 MB).
template <typename T, int FMT, typename I>
__global__ void __launch_bounds__(QT_THREADS)
mx4_quantize_kernel(const T* x, Mx4Rows q, const float* tensor_scale, float* own_scale, int parts, uint8_t* codes,
                    uint8_t* scales) {
  constexpr int PER = Mx4Fmt<FMT>::BLOCK / 16;
  pdl_wait();
  pdl_trigger();
  const long long code_row = (q.cols + 1) / 2, scale_row = q.chunks / PER;
  const I total = (I)(q.rows * q.chunks);
  Mx4Raw<T> raw[QT_BATCH];
  I row[QT_BATCH], c[QT_BATCH];
  int left[QT_BATCH];                                                // -1: behind the last row
#pragma unroll
  for (int j = 0; j < QT_BATCH; ++j) {
    const I i = (I)blockIdx.x * (QT_THREADS * QT_BATCH) + j * QT_THREADS + threadIdx.x;
    place(q, i, row[j], c[j]);
    left[j] = i < total ? values_at(q, c[j]) : -1;
    raw[j].load(x + (long long)row[j] * q.stride + (long long)c[j] * 16, left[j]);
  }
  float t = 1.0f;
  if constexpr (FMT == GLQB_MX4_NVFP4) t = whole_scale(tensor_scale, own_scale, parts);       // (while the values are on their way)
#pragma unroll
  for (int j = 0; j < QT_BATCH; ++j) {
    uint32_t s;
    float v[16];
    raw[j].get(v);
    const uint2 word = mx4_quantize16<FMT, false>(v, raw[j].top(), t, s);     // (all lanes: the threads of a block exchange their largest value)
    if (left[j] < 0) continue;
    uint8_t* p = codes + (long long)row[j] * code_row + (long long)c[j] * 8;
    const uint32_t at = left[j] == 16 ? (uint32_t)reinterpret_cast<uintptr_t>(p) : 1u;
    if ((at & 7u) == 0) *reinterpret_cast<uint2*>(p) = word;
    else if ((at & 3u) == 0) {
      reinterpret_cast<uint32_t*>(p)[0] = word.x;
      reinterpret_cast<uint32_t*>(p)[1] = word.y;
    } else if ((at & 1u) == 0) {
      *reinterpret_cast<uint16_t*>(p) = (uint16_t)word.x;
      *reinterpret_cast<uint32_t*>(p + 2) = __funnelshift_r(word.x, word.y, 16);
      *reinterpret_cast<uint16_t*>(p + 6) = (uint16_t)(word.y >> 16);
    } else {
#pragma unroll
      for (int b = 0; b < 8; ++b)
        if (2 * b < left[j]) p[b] = (uint8_t)((b < 4 ? word.x : word.y) >> (8 * (b & 3)));
    }
    if (c[j] % PER == 0) scales[(long long)row[j] * scale_row + (long long)(c[j] / PER)] = (uint8_t)s;
  }
}

template <int FMT, typename I>
__global__ void __launch_bounds__(QT_THREADS)
mx4_dequantize_kernel(const uint8_t* codes, const uint8_t* scales, const float* tensor_scale, long long rows_per_scale, Mx4Rows q, void* out,
                      int out_dtype) {
  constexpr int PER = Mx4Fmt<FMT>::BLOCK / 16;
  pdl_wait();
  pdl_trigger();
  const long long code_row = (q.cols + 1) / 2, scale_row = q.chunks / PER;
  const I total = (I)(q.rows * q.chunks);
  const bool one_scale = FMT != GLQB_MX4_NVFP4 || rows_per_scale >= q.rows;
  float t0 = 1.0f;
  if (FMT == GLQB_MX4_NVFP4 && one_scale) t0 = *tensor_scale;
  uint32_t part[QT_BATCH][4], byte[QT_BATCH];                        // (parts of codes as they are loaded: nothing waits for them here)
  I row[QT_BATCH], c[QT_BATCH];
  int left[QT_BATCH];
#pragma unroll
  for (int j = 0; j < QT_BATCH; ++j) {
    const I i = (I)blockIdx.x * (QT_THREADS * QT_BATCH) + j * QT_THREADS + threadIdx.x;
    place(q, i, row[j], c[j]);
    left[j] = i < total ? values_at(q, c[j]) : 0;
    byte[j] = part[j][0] = part[j][1] = part[j][2] = part[j][3] = 0;
    if (left[j] <= 0) continue;
    const uint8_t* p = codes + (long long)row[j] * code_row + (long long)c[j] * 8;
    const uint32_t at = left[j] == 16 ? (uint32_t)reinterpret_cast<uintptr_t>(p) : 1u;
    if ((at & 7u) == 0) {
      const uint2 w = *reinterpret_cast<const uint2*>(p);
      part[j][0] = w.x;
      part[j][2] = w.y;
    } else if ((at & 3u) == 0) {
      part[j][0] = reinterpret_cast<const uint32_t*>(p)[0];
      part[j][2] = reinterpret_cast<const uint32_t*>(p)[1];
    } else if ((at & 1u) == 0) {
      part[j][0] = *reinterpret_cast<const uint16_t*>(p);
      part[j][1] = *reinterpret_cast<const uint32_t*>(p + 2);
      part[j][3] = *reinterpret_cast<const uint16_t*>(p + 6);
    } else {
#pragma unroll
      for (int b = 0; b < 8; ++b)
        if (2 * b < left[j]) part[j][b >> 2 << 1] |= (uint32_t)p[b] << (8 * (b & 3));
    }
    byte[j] = scales[(long long)row[j] * scale_row + (long long)(c[j] / PER)];
  }
#pragma unroll
  for (int j = 0; j < QT_BATCH; ++j) {
    if (left[j] <= 0) continue;
    const float s = mx4_scale_value<FMT>(byte[j]);
    const float t = one_scale ? t0 : tensor_scale[(long long)row[j] / rows_per_scale];
    const uint32_t words[2] = {part[j][0] | part[j][1] << 16, part[j][2] | part[j][1] >> 16 | part[j][3] << 16};
    float v[16];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      float u[8];
      mx4_values8(words[w], u);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        mx4_mul_f32x2(u[e], u[e + 1], s, s);
        if constexpr (FMT == GLQB_MX4_NVFP4) mx4_mul_f32x2(u[e], u[e + 1], t, t);
        v[8 * w + e] = u[e];
        v[8 * w + e + 1] = u[e + 1];
      }
    }
    const long long at = (long long)row[j] * q.cols + (long long)c[j] * 16;
    if (out_dtype == GLQB_DT_F32) {
      float* o = reinterpret_cast<float*>(out) + at;
      uint32_t h[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) h[e] = __float_as_uint(v[e]);
      if (left[j] == 16) mx4_put_words(o, h);
      else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (e < left[j]) o[e] = v[e];
      }
    } else {
      uint32_t h[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (out_dtype == GLQB_DT_F16) {
          const __half2 r = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
          h[e] = *reinterpret_cast<const uint32_t*>(&r);
        } else {
          const __nv_bfloat162 r = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
          h[e] = *reinterpret_cast<const uint32_t*>(&r);
        }
      }
      uint16_t* o = reinterpret_cast<uint16_t*>(out) + at;
      if (left[j] == 16) mx4_put_words(o, h);
      else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (e < left[j]) o[e] = (uint16_t)(h[e >> 1] >> (16 * (e & 1)));
      }
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
__global__ void __launch_bounds__(256) mx4_align_kernel(const uint16_t* x, long long x_stride, long long rows, int n, int n_pad, uint16_t* out) {
  pdl_wait();
  pdl_trigger();
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < rows * n_pad; i += (long long)gridDim.x * 256) {
    const long long r = i / n_pad;
    const int c = (int)(i - r * n_pad);
    out[i] = c < n ? x[r * x_stride + c] : (uint16_t)0;
  }
}

// Rows of x in 4 bits, as the tiles the 4-bit product fetches (per token tile, per 256 values: tn rows of 128 bytes with the
// 128-byte swizzle, then the scales, 128 rows at a time as in the weight image).  A warp takes `batches` times 1024 values of a row
// (with many rows all of a row: finding its tile takes as long as a thousand values); values past the row are zeros, rows past a
// tile's are left out (their columns are not stored).  32768 rows of 2048 bf16 values to MXFP4 38 us (170 MB): the instructions around the
// values bound it, 88 per warp for eight of a lane.  (The next step's values in registers meanwhile: three CTAs per SM for four, 44 us.)
constexpr int X_TILES = 2 * QT_BATCH;              // of 256 values: what a warp takes at once
template <typename T, int FMT>
__global__ void __launch_bounds__(QT_THREADS, 4) mx4_x_image_kernel(const __grid_constant__ Mx4Job J, const float* x_scale, float* own_scale, int parts,
                                                                 int x_scales, int batches) {
  extern __shared__ int lists[];
  const Mx4Lists L(lists, J.experts);
  pdl_wait();
  pdl_trigger();
  mx4_groups(J, L);
  constexpr int PER = Mx4Fmt<FMT>::BLOCK / 16;
  float t = 1.0f;
  if constexpr (FMT == GLQB_MX4_NVFP4) t = whole_scale(x_scale, own_scale, parts);
  const int lane = threadIdx.x & 31, first = L.eff[0], end = L.eff[J.experts], per_row = (J.k_tiles + X_TILES * batches - 1) / (X_TILES * batches);
  const int half = lane >> 4, c = lane & 15;                // a step's second tile, sixteen of a tile
  const long long stage = (long long)J.tn * 128 + x_scales, items = (long long)(end - first) * per_row;
  const long long warps = (long long)gridDim.x * (QT_THREADS / 32), w = (long long)blockIdx.x * (QT_THREADS / 32) + (threadIdx.x >> 5);
  const long long i0 = w * items / warps, i1 = (w + 1) * items / warps;
  if (i0 == i1) return;
  // a warp's items follow one another: the expert and the tile of a row come from those of the row before
  int row = first + (int)(i0 / per_row), part = (int)(i0 % per_row);
  int e = J.experts == 1 ? 0 : mx4_find(L.eff, J.experts, row), per = L.per[e];
  int tile = L.pre[e] + (row - L.eff[e]) / per, r = (row - L.eff[e]) % per;
  for (long long i = i0; i < i1; ++i) {
    if (i > i0 && ++part == per_row) {
      part = 0;
      ++row;
      if (row >= L.eff[e + 1]) {
        while (row >= L.eff[e + 1]) ++e;
        per = L.per[e];
        tile = L.pre[e];
        r = 0;
      } else if (++r == per) {
        ++tile;
        r = 0;
      }
    }
    if (tile >= J.max_tiles) continue;
    int k0 = part * X_TILES * batches;
    const T* src = reinterpret_cast<const T*>(J.x) + row * J.x_stride;
    uint8_t* at = J.x_image + ((long long)tile * J.k_tiles + k0 + half) * stage;
    uint8_t* codes = at + (r >> 3) * 1024 + (r & 7) * 128 + (((c >> 1) ^ (r & 7)) << 4) + (c & 1) * 8;
    uint8_t* scales = at + J.tn * 128 + (r >> 7) * mx4_scale_bytes(FMT) + mx4_scale_offset(r & 127, c / PER);
    for (const int k1 = min(J.k_tiles, k0 + X_TILES * batches); k0 < k1; k0 += X_TILES) {
      Mx4Raw<T> raw[QT_BATCH];
#pragma unroll
      for (int j = 0; j < QT_BATCH; ++j) {
        const int col = (k0 + 2 * j + half) * MX4_K + c * 16;
        raw[j].load(src + col, max(0, min(16, J.n - col)));
      }
#pragma unroll
      for (int j = 0; j < QT_BATCH; ++j, codes += 2 * stage, scales += 2 * stage) {
        uint32_t s;
        float v[16];
        raw[j].get(v);
        const uint2 word = mx4_quantize16<FMT, true>(v, raw[j].top(), t, s);
        // four blocks' scales lie together: one store (a store per byte took a sixth of the kernel's time)
        s |= __shfl_down_sync(0xFFFFFFFFu, s, PER) << 8;
        s |= __shfl_down_sync(0xFFFFFFFFu, s, 2 * PER) << 16;
        if (k0 + 2 * j + half >= k1) continue;
        *reinterpret_cast<uint2*>(codes) = word;
        if (c % (4 * PER) == 0) *reinterpret_cast<uint32_t*>(scales) = s;
      }
    }
  }
}

Mx4Rows rows_of(long long rows, int cols, long long stride, int format, bool join) {
  const int block = mx4_block(format);
  Mx4Rows q;
  q.rows = rows;
  q.cols = cols;
  q.stride = stride;
  q.chunks = ((long long)cols + block - 1) / block * (block / 16);
  if (join && stride == cols && cols % block == 0) {       // whole blocks, no gaps: one row
    q.cols = rows * cols;
    q.chunks = q.cols / 16;
    q.rows = 1;
  }
  q.full = q.cols / 16;
  q.rest = (int)(q.cols % 16);
  // Division by a multiplication: with 2^(l - 1) < chunks <= 2^l and magic = ceil(2^(31 + l) / chunks), less than
  // 2^32, magic * chunks is above 2^(31 + l) by less than 2^l, so that i * magic / 2^(31 + l) is off by less than 1 / chunks for i < 2^31.
  q.magic = 0;
  q.shift = 0;
  if (q.chunks < 2 || q.chunks >= 1ll << 31) return q;
  int l = 1;
  while ((1ll << l) < q.chunks) ++l;
  q.magic = (uint32_t)(((1ull << (31 + l)) + (uint64_t)q.chunks - 1) / (uint64_t)q.chunks);
  q.shift = l - 1;
  return q;
}
bool small(const Mx4Rows& q) { return q.rows * q.chunks < (1ll << 31) - QT_THREADS * QT_BATCH; }
unsigned grid_for(const Mx4Rows& q) { return (unsigned)((q.rows * q.chunks + QT_THREADS * QT_BATCH - 1) / (QT_THREADS * QT_BATCH)); }

// the largest finite |x| of the range's rows, in parts; their number
int amax_launch(const void* x, int x_dtype, const Mx4Rows& q, const Mx4Range& range, float* parts, cudaStream_t stream) {
  const int grid = (int)std::min<long long>((q.rows * q.chunks + AMAX_THREADS - 1) / AMAX_THREADS, AMAX_PARTS);
  auto run = [&](auto type, auto index) {
    using T = decltype(type);
    launch_chained(true, mx4_amax_kernel<T, decltype(index)>, grid, AMAX_THREADS, 0, stream, (const T*)x, q, range, parts);
  };
  auto of = [&](auto type) { q.rows * q.chunks < (1ll << 31) - (long long)AMAX_PARTS * AMAX_THREADS * QT_BATCH ? run(type, (uint32_t)0) : run(type, (uint64_t)0); };
  if (x_dtype == GLQB_DT_F16) of(__half());
  else if (x_dtype == GLQB_DT_BF16) of(__nv_bfloat16());
  else of(float());
  return grid;
}
template <int FMT>
int quantize_launch(const void* x, int x_dtype, const Mx4Rows& q, const float* tensor_scale, float* own_scale, uint8_t* codes, uint8_t* scales,
                    cudaStream_t stream) {
  int parts = 0;
  if (FMT == GLQB_MX4_NVFP4 && !tensor_scale) parts = amax_launch(x, x_dtype, q, Mx4Range{nullptr, 0, 0}, own_scale + 1, stream);
  auto run = [&](auto type, auto index) {
    using T = decltype(type);
    launch_chained(true, mx4_quantize_kernel<T, FMT, decltype(index)>, (int)grid_for(q), QT_THREADS, 0, stream, (const T*)x, q, tensor_scale, own_scale, parts, codes,
                   scales);
  };
  auto of = [&](auto type) { small(q) ? run(type, (uint32_t)0) : run(type, (uint64_t)0); };
  if (x_dtype == GLQB_DT_F16) of(__half());
  else if (x_dtype == GLQB_DT_BF16) of(__nv_bfloat16());
  else of(float());
  return mx4_launched("mx4_quantize");
}
template <int FMT>
int dequantize_launch(const uint8_t* codes, const uint8_t* scales, const float* tensor_scale, long long rows_per_scale, const Mx4Rows& q, void* out,
                      int out_dtype, cudaStream_t stream) {
  auto* kernel = small(q) ? mx4_dequantize_kernel<FMT, uint32_t> : mx4_dequantize_kernel<FMT, uint64_t>;
  launch_chained(true, kernel, (int)grid_for(q), QT_THREADS, 0, stream, codes, scales, tensor_scale, rows_per_scale, q, out, out_dtype);
  return mx4_launched("mx4_dequantize");
}

// Is an address a multiple of `bytes`?  (Kernels access values whole, and the images' bulk copies 16 bytes at a time: elsewhere they fault.)
bool lies_on(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
size_t size_of(int dtype) { return dtype == GLQB_DT_F32 ? 4 : 2; }
bool dtype_ok(int d) { return d == GLQB_DT_F16 || d == GLQB_DT_BF16 || d == GLQB_DT_F32; }
bool format_ok(int f) { return f == GLQB_MX4_MXFP4 || f == GLQB_MX4_NVFP4; }

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
  if (!lies_on(x, size_of(x_dtype)) || !lies_on(tensor_scale, 4) || !lies_on(own_scale, 4)) return mx4_fail(GLQB_E_INVALID, "mx4_quantize: values that are not aligned");
  const Mx4Rows q = rows_of(rows, cols, x_stride, format, true);
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
  if (!lies_on(out, size_of(out_dtype)) || !lies_on(tensor_scale, 4)) return mx4_fail(GLQB_E_INVALID, "mx4_dequantize: values that are not aligned");
  const Mx4Rows q = rows_of(rows, cols, cols, format, format == GLQB_MX4_MXFP4 || rows_per_scale >= rows);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  if (format == GLQB_MX4_MXFP4)
    return dequantize_launch<GLQB_MX4_MXFP4>((const uint8_t*)codes, (const uint8_t*)scales, nullptr, rows, q, out, out_dtype, stream);
  return dequantize_launch<GLQB_MX4_NVFP4>((const uint8_t*)codes, (const uint8_t*)scales, tensor_scale, rows_per_scale, q, out, out_dtype, stream);
}

size_t glqb_mx4_image_bytes(int32_t format, int32_t experts, int32_t m, int32_t n) {
  if (!format_ok(format) || experts < 1 || m < 1 || n < 1) return 0;
  const size_t mt = ((size_t)m + MX4_ROWS - 1) / MX4_ROWS, kt = ((size_t)n + MX4_K - 1) / MX4_K;
  return (size_t)experts * mt * (kt * mx4_tile_bytes(format) + (format == GLQB_MX4_MXFP4 ? 2 * MX4_ROWS : 0));
}

int glqb_mx4_pack(const void* codes, const void* scales, int32_t format, int32_t experts, int32_t m, int32_t n, void* image,
                  void* stream_) {
  if (!format_ok(format)) return mx4_fail(GLQB_E_INVALID, "mx4_pack: format %d", format);
  if (experts < 1 || m < 1 || n < 1 || m > MX4_MAX_SIZE || n > MX4_MAX_SIZE) return mx4_fail(GLQB_E_INVALID, "mx4_pack: %d x %d x %d", experts, m, n);
  if (!codes || !scales || !image) return mx4_fail(GLQB_E_INVALID, "mx4_pack: null argument");
  if (!lies_on(image, 128)) return mx4_fail(GLQB_E_INVALID, "mx4_pack: the image must be 128-byte aligned");
  const int mt = (m + MX4_ROWS - 1) / MX4_ROWS, kt = (n + MX4_K - 1) / MX4_K;
  const long long tiles = (long long)experts * mt * kt;
  if (tiles >= (1ll << 31) || experts > MX4_MAX_EXPERTS || (long long)experts * mt >= 1ll << 27)
    return mx4_fail(GLQB_E_INVALID, "mx4_pack: %d x %d x %d: too many tiles (at most %d experts)", experts, m, n, MX4_MAX_EXPERTS);
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
  size_t image, bytes;        // of the workspace: x in 4 bits, then the floats of its scale; or x on 16 bytes
};
struct Device {
  std::atomic<int> sms{0};
  int* status = nullptr;
  int mv[9] = {}, gemm[9] = {};       // clusters that are there at once, by their CTAs
};
static const Device* device() {
  static Device known[64];
  static std::mutex building;
  Device& d = known[mx4_device()];
  if (d.sms.load(std::memory_order_acquire) == 0) {
    std::lock_guard<std::mutex> lock(building);
    int n = 0;
    if (d.sms.load(std::memory_order_relaxed) == 0) {
      if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, mx4_device()) != cudaSuccess || n < 1 ||
          cudaGetSymbolAddress(reinterpret_cast<void**>(&d.status), g_mx4_status) != cudaSuccess)
        return nullptr;
      for (int s = 2; s <= 8; ++s) { d.mv[s] = mx4_mv_clusters(s); d.gemm[s] = mx4_gemm_clusters(s); }
      d.sms.store(n, std::memory_order_release);
    }
  }
  return &d;
}
// Rows (an expert's, on average) up to which the streaming kernel runs; of small layers twice as many: its passes over the weights cost
// less than the tensor-core form's start.  Streaming / tensor cores in a graph, us: 16 tokens of 4096 x 14336 17.2 / 19.4, of 2048 x 2048
// 5.5 / 7.8, of 14336 x 4096 18.9 / 18.9, 24 30.6 / 19.4; 32 tokens of 2048 x 2048 6.3 / 8.3, of 2048 x 4096 8.1 / 9.6, of 8192 x 1024 8.3 / 8.7,
// but of 1024 x 8192 11.0 / 9.9 and of 4096 x 4096 11.7 / 11.1; 128 experts of 1536 x 2048, 600 rows 80 / 94, 1000 82 / 94, 1400 93 / 94; of
// 2048 x 768, 2000 rows 63 / 56.
constexpr int MV_MAX_ROWS = 16, MV_MAX_EXPERT_ROWS = 8, MV_SMALL_TILES = 256, MV_SMALL_K = 16;
static Form form_of(const GlqbMx4Weight* w, long long rows, long long x_stride, const void* x, int quantize, const Device* d) {
  Form f = {};
  const int avg = (int)((rows + w->experts - 1) / w->experts);          // (below 2^30: countable)
  const long long mt = (w->m + MX4_ROWS - 1) / MX4_ROWS, kt = (w->n + MX4_K - 1) / MX4_K;
  const bool small = kt <= MV_SMALL_K && mt * kt <= MV_SMALL_TILES;
  f.mv = !quantize && avg <= (w->experts != 1 ? MV_MAX_EXPERT_ROWS : small ? 2 * MV_MAX_ROWS : MV_MAX_ROWS);
  const int most = quantize ? (w->format == GLQB_MX4_MXFP4 ? 192 : 160) : 192;
  // token tiles: a matrix's rows split evenly; of experts up to twice their average, so that most have one tile
  if (f.mv) f.tn = avg > (w->experts == 1 ? 8 : 4) ? 16 : 8;
  else if (w->experts == 1) f.tn = (int)(((rows + (rows + most - 1) / most - 1) / ((rows + most - 1) / most) + 15) / 16 * 16);
  else f.tn = std::min(most, (2 * avg + 15) / 16 * 16);
  f.max_tiles = w->experts == 1 ? (int)((rows + f.tn - 1) / f.tn) : (int)(rows / f.tn + std::min<long long>(w->experts, rows));
  const long long tiles = f.max_tiles * mt;
  // CTAs that share a tile's sum: as many as leave all tiles there at once
  f.split = 1;
  for (int s = 2; d && s <= std::min<long long>(8, kt); ++s)
    if (tiles <= (f.mv ? d->mv : d->gemm)[s]) f.split = s;
  f.pair = !f.mv && f.split == 1 && f.tn >= 96 && mt > 1;
  if (quantize) {
    f.x_scales = mx4_x_scale_bytes(w->format, f.tn);
    f.image = (size_t)f.max_tiles * kt * ((size_t)f.tn * 128 + f.x_scales);
    f.bytes = f.image + GLQB_MX4_SCALE_FLOATS * 4;
  } else if (reinterpret_cast<uintptr_t>(x) % 16 || (rows > 1 && x_stride % 8) || (f.mv && w->n % 8)) {
    f.align = true;
    f.n_pad = (w->n + 7) / 8 * 8;
    f.bytes = (size_t)rows * f.n_pad * 2;
  }
  return f;
}

// (token tiles are counted in 31 bits)
static bool countable(const GlqbMx4Weight* w, long long rows) { return (rows + w->experts) * ((w->m + MX4_ROWS - 1) / MX4_ROWS) < 1ll << 30; }

size_t glqb_mx4_workspace_bytes(const GlqbMx4Weight* w, int64_t rows, int64_t x_stride, const void* x, int32_t quantize) {
  if (!w || !format_ok(w->format) || rows <= 0 || rows > MX4_MAX_ROWS || w->experts < 1 || w->experts > MX4_MAX_EXPERTS || w->m < 1 ||
      w->m > MX4_MAX_SIZE || w->n < 1 || w->n > MX4_MAX_SIZE || !countable(w, rows))
    return 0;
  return form_of(w, rows, x_stride, x, quantize, nullptr).bytes;      // (what a call needs does not depend on the device)
}

int glqb_mx4_product(const GlqbMx4Weight* w, const void* x, int32_t x_dtype, int64_t x_stride, int64_t rows,
                     const void* offsets, int32_t offsets_are_int64, int32_t quantize, const float* x_scale,
                     void* y, int32_t y_dtype, int64_t y_stride, int32_t accumulate, int32_t clear_rest,
                     void* workspace, size_t workspace_bytes, void* stream_) {
  if (!w || !format_ok(w->format)) return mx4_fail(GLQB_E_INVALID, "mx4_product: format");
  if (w->experts < 1 || w->experts > MX4_MAX_EXPERTS || w->m < 1 || w->n < 1)
    return mx4_fail(GLQB_E_INVALID, "mx4_product: %d x %d x %d (at most %d experts)", w->experts, w->m, w->n, MX4_MAX_EXPERTS);
  if (w->m > MX4_MAX_SIZE || w->n > MX4_MAX_SIZE) return mx4_fail(GLQB_E_INVALID, "mx4_product: %d x %d", w->m, w->n);
  if (!offsets && w->experts != 1) return mx4_fail(GLQB_E_INVALID, "mx4_product: %d experts need offsets", w->experts);
  if (!dtype_ok(x_dtype) || !dtype_ok(y_dtype)) return mx4_fail(GLQB_E_INVALID, "mx4_product: dtype");
  if (!quantize && x_dtype == GLQB_DT_F32) return mx4_fail(GLQB_E_INVALID, "mx4_product: fp32 activations are served quantised only");
  if (rows < 0 || rows > MX4_MAX_ROWS) return mx4_fail(GLQB_E_INVALID, "mx4_product: %lld rows", (long long)rows);
  if (rows == 0) return GLQB_OK;
  if (!countable(w, rows))
    return mx4_fail(GLQB_E_INVALID, "mx4_product: %lld rows of %d results are too many for one call", (long long)rows, w->m);
  if (!w->image || !x || !y || (w->format == GLQB_MX4_NVFP4 && !w->tensor_scale)) return mx4_fail(GLQB_E_INVALID, "mx4_product: null argument");
  if (rows > 1 && (x_stride < w->n || y_stride < w->m)) return mx4_fail(GLQB_E_INVALID, "mx4_product: rows overlap");
  if (!lies_on(w->image, 128)) return mx4_fail(GLQB_E_INVALID, "mx4_product: the image must be 128-byte aligned");
  if (!lies_on(workspace, 16)) return mx4_fail(GLQB_E_INVALID, "mx4_product: the workspace must be 16-byte aligned");
  if (!lies_on(x, size_of(x_dtype)) || !lies_on(y, size_of(y_dtype)) || !lies_on(offsets, offsets_are_int64 ? 8 : 4) || !lies_on(w->tensor_scale, 4) || !lies_on(x_scale, 4))
    return mx4_fail(GLQB_E_INVALID, "mx4_product: values that are not aligned");
  const Device* d = device();
  const Form f = form_of(w, rows, x_stride, x, quantize, d);
  if (workspace_bytes < f.bytes || (f.bytes && !workspace))
    return mx4_fail(GLQB_E_WORKSPACE, "mx4_product: workspace of %zu bytes, %zu needed", workspace_bytes, f.bytes);
  if (!d) return mx4_fail(GLQB_E_CUDA, "mx4_product: no device");
  const int sms = d->sms.load(std::memory_order_relaxed);
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
  J.status = d->status;
  const size_t lists = (size_t)(J.experts + 1) * 12;
  J.clear = offsets && clear_rest;
  if (!quantize) {
    if (f.align) {
      launch_chained(true, mx4_align_kernel, (int)std::min<long long>((rows * f.n_pad + 255) / 256, 148 * 32), 256, 0, stream, (const uint16_t*)x, x_stride, rows, w->n,
                     f.n_pad, (uint16_t*)workspace);
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
  int parts = 0;
  if (w->format == GLQB_MX4_NVFP4 && !x_scale) {
    const Mx4Rows q = rows_of(rows, w->n, x_stride, w->format, !offsets);
    parts = amax_launch(x, x_dtype, q, Mx4Range{offsets, offsets_are_int64, w->experts}, own + 1, stream);
  }
  const long long warps = (long long)sms * 32, batches = (J.k_tiles + X_TILES - 1) / X_TILES;
  const int at_once = (int)std::max<long long>(1, std::min(batches, rows * batches / warps));
  const int grid = (int)std::min<long long>((rows * ((batches + at_once - 1) / at_once) + 7) / 8, (long long)sms * 4);
  auto image = [&](auto fmt) {
    constexpr int FMT = decltype(fmt)::value;
    if (x_dtype == GLQB_DT_F16) launch_chained(true, mx4_x_image_kernel<__half, FMT>, grid, QT_THREADS, lists, stream, J, x_scale, own, parts, f.x_scales, at_once);
    else if (x_dtype == GLQB_DT_BF16) launch_chained(true, mx4_x_image_kernel<__nv_bfloat16, FMT>, grid, QT_THREADS, lists, stream, J, x_scale, own, parts, f.x_scales, at_once);
    else launch_chained(true, mx4_x_image_kernel<float, FMT>, grid, QT_THREADS, lists, stream, J, x_scale, own, parts, f.x_scales, at_once);
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
