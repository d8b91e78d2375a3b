// Microscaled 4-bit floating point: formats, the weight image, and the conversions every kernel of glqb_mx4*.cu shares.
//
// A value is e2m1 (sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6) times the scale of its block:
//   MXFP4  32 values share 2^(s - 127), s one byte (255: not a number)
//   NVFP4  16 values share an e4m3 number, and a tensor (or expert) one fp32 number
// Rows are stored as checkpoints store them: two codes to a byte, the even value in the low nibble, and one byte per block.
//
// The image of a weight matrix is those bytes in the order the products read them: tiles of 128 rows x 256 values,
// [row tile][value tile], each 16 KiB of codes as a K-major tile with the 128-byte swizzle of the tensor core (so one bulk copy
// brings what tcgen05.mma reads), then the scales of the tile, 512 bytes per four blocks: byte (r % 32) * 16 + (r / 32) * 4 + i
// is block i of row r, which is how tcgen05.cp hands scales to tensor memory.  The eight codes of a 32-bit word lie in the order
// 0 2 4 6 1 3 5 7: values 2i and 2i + 1 are nibbles i and i + 4, so that one shift and mask bring a pair to the halves of
// a register.  (The 4-bit products do not see it: both operands have that order, and a word never leaves its block.)
// Behind the tiles: for MXFP4 two bytes per row, the largest scale of the row, which 16-bit operands are held relative to.
#pragma once
#include "glqb_internal.h"
#include <cuda_fp8.h>
#include <type_traits>

namespace glqb {

constexpr int MX4_ROWS = 128, MX4_K = 256;                    // a tile
constexpr int MX4_CODE_BYTES = MX4_ROWS * MX4_K / 2;          // 16 KiB

template <int FMT> struct Mx4Fmt;
template <> struct Mx4Fmt<GLQB_MX4_MXFP4> { static constexpr int BLOCK = 32; };
template <> struct Mx4Fmt<GLQB_MX4_NVFP4> { static constexpr int BLOCK = 16; };
__host__ __device__ constexpr int mx4_block(int fmt) { return fmt == GLQB_MX4_MXFP4 ? 32 : 16; }
__host__ __device__ constexpr int mx4_scale_bytes(int fmt) { return MX4_ROWS * (MX4_K / mx4_block(fmt)); }   // of a tile
__host__ __device__ constexpr int mx4_tile_bytes(int fmt) { return MX4_CODE_BYTES + mx4_scale_bytes(fmt); }

// byte of the 32-bit word that holds value k (0..255) of row r of a tile
__host__ __device__ __forceinline__ int mx4_word_offset(int r, int k) {
  return (r >> 3) * 1024 + (r & 7) * 128 + (((k >> 5) ^ (r & 7)) << 4) + ((k >> 3) & 3) * 4;
}
// byte of the scale of block b (of a tile) of row r, behind the codes
__host__ __device__ __forceinline__ int mx4_scale_offset(int r, int b) {
  return (b >> 2) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (b & 3);
}

#ifdef __CUDACC__
// 0 1 2 3 4 5 6 7 -> 0 2 4 6 1 3 5 7
__device__ __forceinline__ uint32_t mx4_interleave(uint32_t w) {
  uint32_t lo = w & 0x0F0F0F0Fu, hi = (w >> 4) & 0x0F0F0F0Fu;            // even values, odd values, a byte each
  lo = (lo | (lo >> 4)) & 0x00FF00FFu;
  hi = (hi | (hi >> 4)) & 0x00FF00FFu;
  return (lo | (lo >> 8)) & 0xFFFFu | ((hi | (hi >> 8)) << 16);
}
// Eight floats to e2m1, round to nearest even, saturating; `image`: in the image's order of nibbles.
template <bool IMAGE>
__device__ __forceinline__ uint32_t mx4_codes8(const float (&v)[8]) {
  uint32_t r;
  // (the first source of the conversion is the high nibble)
  if constexpr (IMAGE)
    asm("{ .reg .b8 a, b, c, d; cvt.rn.satfinite.e2m1x2.f32 a, %3, %1; cvt.rn.satfinite.e2m1x2.f32 b, %7, %5; "
        "cvt.rn.satfinite.e2m1x2.f32 c, %4, %2; cvt.rn.satfinite.e2m1x2.f32 d, %8, %6; mov.b32 %0, {a, b, c, d}; }"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  else
    asm("{ .reg .b8 a, b, c, d; cvt.rn.satfinite.e2m1x2.f32 a, %2, %1; cvt.rn.satfinite.e2m1x2.f32 b, %4, %3; "
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5; cvt.rn.satfinite.e2m1x2.f32 d, %8, %7; mov.b32 %0, {a, b, c, d}; }"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// the eight values of a stored word
__device__ __forceinline__ void mx4_values8(uint32_t w, float (&v)[8]) {
  uint32_t r[4];
  asm("{ .reg .b8 a, b, c, d; mov.b32 {a, b, c, d}, %4; cvt.rn.f16x2.e2m1x2 %0, a; cvt.rn.f16x2.e2m1x2 %1, b; cvt.rn.f16x2.e2m1x2 %2, c; "
      "cvt.rn.f16x2.e2m1x2 %3, d; }" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ float mx4_e4m3(uint32_t byte) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
}
__device__ __forceinline__ float mx4_e8m0(uint32_t byte) {                // 2^(byte - 127)
  return byte == 255u ? __uint_as_float(0x7FC00000u) : byte ? __uint_as_float(byte << 23) : __uint_as_float(0x00400000u);
}
template <int FMT>
__device__ __forceinline__ float mx4_scale_value(uint32_t byte) {
  if constexpr (FMT == GLQB_MX4_MXFP4) return mx4_e8m0(byte);
  else return mx4_e4m3(byte);
}

// Two products at once: (a x, b y).
__device__ __forceinline__ void mx4_mul_f32x2(float& a, float& b, float x, float y) {
  asm("{ .reg .b64 u, v; mov.b64 u, {%0, %1}; mov.b64 v, {%2, %3}; mul.rn.f32x2 u, u, v; mov.b64 {%0, %1}, u; }" : "+f"(a), "+f"(b) : "f"(x), "f"(y));
}

// ---- quantisation ---------------------------------------------------------------------------------
// The definition is in real numbers: the scale of an NVFP4 block is the e4m3 number nearest to amax / (6 t), a code the e2m1
// number nearest to x / (s t), ties to even.  fp32 quotients can land on the wrong side of a border, so the conversion is done
// for the quotient a little smaller and a little larger (its error is below 1.5 * 2^-22, the margin 2^-21); where the two disagree
// the side is taken from an exact comparison: border * s and border * 6 have at most eight bits, so fma(-p, t, x) has the
// sign of x - border * s * t.  (MXFP4 divides by powers of two: nothing to decide.)
constexpr float MX4_BELOW = 1.0f - 0x1p-21f, MX4_ABOVE = 1.0f + 0x1p-21f;
// Steps below 2^-100 would lose bits in that product, and their reciprocal's range ends: 64 bits there.
constexpr float MX4_TINY = 0x1p-100f;

__device__ __forceinline__ uint32_t mx4_nv_scale(float amax, float t) {
  const float q = __fdividef(amax, 6.0f * t);
  uint16_t both;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(both) : "f"(q * MX4_ABOVE), "f"(q * MX4_BELOW));
  const uint32_t lo = both & 0xFFu, hi = both >> 8;
  const bool tiny = t < MX4_TINY || t > 0x1p100f;
  if (lo == hi && !tiny) return lo;
  if (tiny) {
    // amax / (6 t) to the nearest, by its distance to the neighbours of the value that fp32 arithmetic of 64 bits gives
    const double d = fmin((double)amax / (6.0 * (double)t), 448.0);
    uint32_t s = __nv_cvt_double_to_fp8(d, __NV_SATFINITE, __NV_E4M3) & 0x7Fu;
    while (s < 126u && 2.0 * d > (double)mx4_e4m3(s) + (double)mx4_e4m3(s + 1u)) ++s;
    while (s > 0u && 2.0 * d < (double)mx4_e4m3(s) + (double)mx4_e4m3(s - 1u)) --s;
    if (s < 126u && (s & 1u) && 2.0 * d == (double)mx4_e4m3(s) + (double)mx4_e4m3(s + 1u)) ++s;
    else if (s > 0u && (s & 1u) && 2.0 * d == (double)mx4_e4m3(s) + (double)mx4_e4m3(s - 1u)) --s;
    return s;
  }
  const float middle = 0.5f * (mx4_e4m3(lo) + mx4_e4m3(hi)), rest = fmaf(-(middle * 6.0f), t, amax);
  return rest > 0.0f ? hi : rest < 0.0f ? lo : (lo & 1u) ? hi : lo;
}
// Eight codes of |x| / (s t), from those of slightly smaller quotients: where the slightly larger ones differ (by one), the border between
// decides.  One at a time: bf16 values meet borders exactly in every few blocks (2688 = 2^7 * 21, borders of 7/4 and scales of 3/2), most
// of a block's others never.  (All eight side by side: 32768 bf16 rows of 2048 with their product 192 us, so 163.)
template <bool IMAGE>
__device__ __forceinline__ uint32_t mx4_decide8(uint32_t a, uint32_t b, const float* v, float s, float t) {
  uint32_t c = a;
  for (uint32_t differ = a ^ b; differ;) {
    const int at = (31 - __clz(differ)) >> 2, i = IMAGE ? 2 * (at & 3) + (at >> 2) : at;
    differ &= ~(15u << (4 * at));
    const float x0 = i & 1 ? v[1] : v[0], x1 = i & 1 ? v[3] : v[2], x2 = i & 1 ? v[5] : v[4], x3 = i & 1 ? v[7] : v[6];
    const float x = fabsf(i & 4 ? (i & 2 ? x3 : x2) : (i & 2 ? x1 : x0));
    const uint32_t lo = (a >> (4 * at)) & 7u;
    const float border = 0.25f * (float)(__byte_perm(0x07050301u, 0x00140E0Au, lo) & 0xFFu);      // 1 3 5 7 10 14 20 quarters
    const float rest = fmaf(-(border * s), t, x);
    if (rest > 0.0f || (rest == 0.0f && (lo & 1u))) c += 1u << (4 * at);
  }
  return c;
}
static __device__ __noinline__ uint32_t mx4_decide_tiny(float x, float s, float t) {
  const double d = (double)s * (double)t, a = (double)x;      // (31 bits: products with the borders are exact)
  return (uint32_t)((a > 0.25 * d) + (a >= 0.75 * d) + (a > 1.25 * d) + (a >= 1.75 * d) + (a > 2.5 * d) + (a >= 3.5 * d) + (a > 5.0 * d));
}

// Sixteen consecutive values of a row per thread, `top` the bits of their largest magnitude; the BLOCK / 16 threads of a block are
// neighbours in a warp (all 32 lanes take part).  Returns the codes; `scale`: the block's byte, the same in its threads.  A
// block with an infinity or NaN gets the scale NaN and codes of zero.
template <int FMT, bool IMAGE>
__device__ __forceinline__ uint2 mx4_quantize16(const float (&v)[16], uint32_t top, float t, uint32_t& scale) {
#pragma unroll
  for (int d = 1; d < Mx4Fmt<FMT>::BLOCK / 16; d <<= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
  const bool broken = top >= 0x7F800000u;
  uint32_t c[2];
  if constexpr (FMT == GLQB_MX4_MXFP4) {
    const uint32_t e = top >> 23;
    scale = broken ? 255u : e > 2u ? e - 2u : 0u;
    if (broken) return make_uint2(0u, 0u);
    const float r = __uint_as_float((254u - scale) << 23);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      float q[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = v[8 * w + i];
#pragma unroll
      for (int i = 0; i < 8; i += 2) mx4_mul_f32x2(q[i], q[i + 1], r, r);
      c[w] = mx4_codes8<IMAGE>(q);
    }
  } else {
    scale = broken ? 0x7Fu : mx4_nv_scale(__uint_as_float(top), t);
    if (broken) return make_uint2(0u, 0u);
    const float s = mx4_e4m3(scale), step = s * t;
    if (step >= MX4_TINY) {
      const float r = __frcp_rn(step), rl = r * MX4_BELOW, rh = r * MX4_ABOVE;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        float lo[8], hi[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) lo[i] = hi[i] = v[8 * w + i];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          mx4_mul_f32x2(lo[i], lo[i + 1], rl, rl);
          mx4_mul_f32x2(hi[i], hi[i + 1], rh, rh);
        }
        const uint32_t a = mx4_codes8<IMAGE>(lo), b = mx4_codes8<IMAGE>(hi);
        c[w] = mx4_decide8<IMAGE>(a, b, v + 8 * w, s, t);
      }
    } else {
      c[0] = c[1] = 0u;
      if (scale != 0u) {
#pragma unroll 1
        for (int i = 0; i < 16; ++i) {
          const int at = IMAGE ? ((i & 7) >> 1) + 4 * (i & 1) : i & 7;
          float x = v[0];
#pragma unroll
          for (int j = 1; j < 16; ++j) x = i == j ? v[j] : x;
          const uint32_t code = (mx4_decide_tiny(fabsf(x), s, t) | (x < 0.0f ? 8u : 0u)) << (4 * at);
          c[0] |= i < 8 ? code : 0u;
          c[1] |= i < 8 ? 0u : code;
        }
      }
    }
  }
  return make_uint2(c[0], c[1]);
}

// The fp32 scale of a tensor whose largest finite value is `amax`: the top of both levels, 448 * 6, by its fp32 reciprocal.
__device__ __forceinline__ float mx4_tensor_scale(float amax) { return fmaxf(amax * (1.0f / 2688.0f), 0x1p-126f); }

// ---- loads of activations -------------------------------------------------------------------------
// 32 bytes at once, from and to addresses on 32 bytes.
__device__ __forceinline__ void mx4_load32(const void* p, uint4& a, uint4& b) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w) : "l"(p) : "memory");
}
__device__ __forceinline__ void mx4_store32(void* p, const uint4& a, const uint4& b) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w) : "memory");
}
// 32-bit words to any address that the values allow, in the widest stores that lie on their size.  (A sector that is written in two
// halves costs as much as two: where 64 bytes start in the middle of a sector, its other half comes from the neighbour.)
template <int WORDS>
__device__ __forceinline__ void mx4_put_words(void* p, const uint32_t (&h)[WORDS]) {
  const uint32_t at = (uint32_t)reinterpret_cast<uintptr_t>(p);
  auto four = [&](int i) { return make_uint4(h[i], h[i + 1], h[i + 2], h[i + 3]); };
  uint4* p4 = reinterpret_cast<uint4*>(p);
  if ((at & 31u) == 0) {
#pragma unroll
    for (int i = 0; i < WORDS; i += 8) mx4_store32(p4 + i / 4, four(i), four(i + 4));
  } else if ((at & 15u) == 0) {
    p4[0] = four(0);
#pragma unroll
    for (int i = 4; i + 8 < WORDS; i += 8) mx4_store32(p4 + i / 4, four(i), four(i + 4));
    p4[WORDS / 4 - 1] = four(WORDS - 4);
  } else if ((at & 3u) == 0) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) reinterpret_cast<uint32_t*>(p)[i] = h[i];
  } else {
#pragma unroll
    for (int i = 0; i < 2 * WORDS; ++i) reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(h[i >> 1] >> (16 * (i & 1)));
  }
}
// Sixteen values of a row as they lie, zeros from the `left`-th on, and as fp32.
template <typename T>
struct Mx4Raw {
  uint4 w[sizeof(T)];
  __device__ __forceinline__ void load(const T* p, int left) {
    constexpr int N = sizeof(T);
    const uint32_t at = (uint32_t)reinterpret_cast<uintptr_t>(p);
    const uint4* p4 = reinterpret_cast<const uint4*>(p);
    if (left >= 16 && (at & 31u) == 0) {
#pragma unroll
      for (int i = 0; i < N; i += 2) mx4_load32(p4 + i, w[i], w[i + 1]);
    } else if (left >= 16 && (at & 15u) == 0) {
      w[0] = p4[0];
      if constexpr (N == 4) mx4_load32(p4 + 1, w[1], w[2]);
      w[N - 1] = p4[N - 1];
    } else if (left >= 16 && (at & 7u) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint2 a = reinterpret_cast<const uint2*>(p)[2 * i], b = reinterpret_cast<const uint2*>(p)[2 * i + 1];
        w[i] = make_uint4(a.x, a.y, b.x, b.y);
      }
    } else if (left >= 16 && (at & 3u) == 0) {
      const uint32_t* u = reinterpret_cast<const uint32_t*>(p);
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = make_uint4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
    } else {
      using U = std::conditional_t<N == 4, uint32_t, uint16_t>;
      const U* u = reinterpret_cast<const U*>(p);
      uint32_t e[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) e[i] = i < left ? (uint32_t)u[i] : 0u;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if constexpr (N == 4) w[i] = make_uint4(e[4 * i], e[4 * i + 1], e[4 * i + 2], e[4 * i + 3]);
        else w[i] = make_uint4(e[8 * i] | e[8 * i + 1] << 16, e[8 * i + 2] | e[8 * i + 3] << 16, e[8 * i + 4] | e[8 * i + 5] << 16, e[8 * i + 6] | e[8 * i + 7] << 16);
      }
    }
  }
  // bits, as fp32, of the largest magnitude (16-bit types: two at a time, their bits without the sign are ordered as they are)
  __device__ __forceinline__ uint32_t top() const {
    if constexpr (sizeof(T) == 4) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        m = max(max(m, max(w[i].x & 0x7FFFFFFFu, w[i].y & 0x7FFFFFFFu)), max(w[i].z & 0x7FFFFFFFu, w[i].w & 0x7FFFFFFFu));
      return m;
    } else {
      constexpr uint32_t M = 0x7FFF7FFFu;
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 2; ++i) m = __vmaxu2(__vmaxu2(m, __vmaxu2(w[i].x & M, w[i].y & M)), __vmaxu2(w[i].z & M, w[i].w & M));
      if constexpr (__is_same(T, __half)) return __float_as_uint(__half2float(__ushort_as_half((unsigned short)max(m & 0xFFFFu, m >> 16))));
      else return max(m << 16, m & 0xFFFF0000u);
    }
  }
  __device__ __forceinline__ void get(float (&v)[16]) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) {
      const uint32_t h[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) v[4 * i + j] = __uint_as_float(h[j]);
        else if constexpr (__is_same(T, __half)) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
          v[8 * i + 2 * j] = f.x;
          v[8 * i + 2 * j + 1] = f.y;
        } else {
          v[8 * i + 2 * j] = __uint_as_float(h[j] << 16);
          v[8 * i + 2 * j + 1] = __uint_as_float(h[j] & 0xFFFF0000u);
        }
      }
    }
  }
};
#endif  // __CUDACC__

}  // namespace glqb
