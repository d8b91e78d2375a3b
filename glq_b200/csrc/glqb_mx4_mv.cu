// Products of microscaled 4-bit weights with few rows of x: decode steps, experts of few tokens.
//
// What bounds these is the weights' way from HBM and, close behind, the instructions that make 16-bit operands of them.  A CTA
// takes 128 weight rows x 8 NB rows of x; one warp brings tiles of 128 x 256 weights into a ring of stages (bulk copies), two or four bring the
// values of x that belong to them, and they run ahead over the borders of the CTA's work.  Eight warps take 16 weight rows each, turn a tile into fragments of mma.sync.m16n8k16 in
// registers and multiply.  The MMA's order of values is free as long as both operands have it: lane t of a quad takes word t of a
// 16-byte unit, eight values, and of x the same eight, so nothing is exchanged and every shared-memory access is free of
// conflicts.  Where there are few tiles the CTAs of a cluster share out the values and add their parts in rank order.
//
// The scale of an MXFP4 block multiplies the block's sum instead of its codes: a 16-byte unit is a block, two MMAs, and four products per
// eight columns take the place of eight of pairs (256 rows over 128 experts of 1536 x 2048 60.9 -> 58.1 us, one token of 14336 x 4096 13.3 ->
// 12.1).  An NVFP4 unit has two blocks, whose lanes meet in every MMA: there the codes are multiplied.
//
// Operands are fp16, because two codes become fp16 in one instruction and bf16 in four (as bf16: 505 instructions per warp
// for 16 rows x 256 values, 256 rows over 128 experts of 1536 x 2048 70 us).  bf16 rows of x are brought to
// fp16 on their way to shared memory, 256 values at a time, by the power of two that takes the largest finite one to 2^15 .. 2^16; the sums of a tile are multiplied back in
// fp32.  (The largest bf16 number below 2^16 is 65280, which fp16 has.)  fp16 steps by 2^-24: values of at least 2^-32 of the largest are exact,
// smaller ones off by at most 2^-25, 2^-40 of it.  Where the largest is below 2^-94 the power is 2^109, and every bf16 number exact.
//
// A sum must not leave fp32's range where the result does not.  MXFP4 sums are relative to mx4_base; NVFP4 sums are multiplied, with the power that
// brings a row of x back, by that of the matrix's scale (mx4_shift).  Nothing waits for the scale before a tile's first sums are there (eight
// tokens of 14336 x 4096 14.9 us, without the power 14.7, with a wait at the start 15.5).
#include "glqb_mx4_gemm.cuh"
#include "glqb_launch.h"
#include <algorithm>

namespace glqb {
namespace {

constexpr int MV4_WARPS = 8;
constexpr int MV4_X_ROW = MX4_K * 2 + 64;        // bytes of a row of x: two rows in different banks
template <int FMT, typename T, int NB> struct Mv4 {
  static constexpr int X = mx4_tile_bytes(FMT) + (FMT == GLQB_MX4_MXFP4 ? 2 * MX4_ROWS : 0);       // of a stage: weights, their rows' largest scales,
  static constexpr int X_SCALE = X + 8 * NB * MV4_X_ROW, STAGE = X_SCALE + 128;                    // x, what its sums are multiplied by
  static constexpr int STAGES = NB == 1 ? 4 : 3;                                                   // two CTAs per SM
  static constexpr int X_WARPS = 2 * NB, THREADS = (MV4_WARPS + 1 + X_WARPS) * 32;
  static constexpr bool SHIFT = FMT == GLQB_MX4_NVFP4 && !__is_same(T, __half);                    // sums times a power of two of the matrix's scale
};
// A tile's factor, from the scale that was loaded at its start (used here first: moved in front of the sums it would be waited for there).
template <bool SHIFT>
__device__ __forceinline__ void settle_factor(Mx4Factor& f) {
  if constexpr (SHIFT) {
    asm volatile("" : "+f"(f.b));
    f = mx4_factor(f.b, mx4_pow2(-mx4_shift(f.b, 0)));
  }
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma16816_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// NVFP4: the scales of a row's blocks that lane t meets in the 16-byte units 2i and 2i + 1, bytes t / 2 and t / 2 + 2 of word i, as pairs of fp16.
__device__ __forceinline__ void multipliers(uint32_t word, uint32_t pick, uint32_t (&m)[2]) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)__byte_perm(word, 0, pick), __NV_E4M3);
  const uint32_t b = (uint32_t)h.x | (uint32_t)h.y << 16;
  m[0] = __byte_perm(b, 0, 0x1010);
  m[1] = __byte_perm(b, 0, 0x3232);
}
// MXFP4: 2^(scale - top) of a row's block j, from its word of scales (top: mx4_base of the row's largest).  PLAIN (all numbers, within 2^27 of
// the largest, which base is no more than 24 above): the word holds scale - top + 127.
template <bool PLAIN>
__device__ __forceinline__ float block_power(uint32_t word, int j, int top) {
  const int b = j & 3;
  if constexpr (PLAIN) return __uint_as_float((b == 3 ? word >> 1 : word << (23 - 8 * b)) & 0x7F800000u);
  const uint32_t s = (word >> (8 * b)) & 0xFFu;
  return s == 255u ? __uint_as_float(0x7FC00000u) : ldexpf(1.0f, (int)s - top);
}

// A row's eight values of a lane to `p` as fp16 in the order 0 2 4 6 1 3 5 7; bf16 times a power of two: returned is what the sums are
// multiplied by, its inverse.
template <typename T>
__device__ __forceinline__ float put8(uint8_t* p, const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (__is_same(T, __half)) {
    *reinterpret_cast<uint4*>(p) = make_uint4(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410), __byte_perm(w[0], w[1], 0x7632),
                                              __byte_perm(w[2], w[3], 0x7632));
    return 1.0f;
  } else {
    constexpr uint32_t M = 0x7FFF7FFFu;
    const uint32_t both = __vmaxu2(__vmaxu2(w[0] & M, w[1] & M), __vmaxu2(w[2] & M, w[3] & M));
    uint32_t top = max(both & 0xFFFFu, both >> 16);
    if (top >= 0x7F80u) {                                // an infinity or NaN: the largest of the others
      top = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = w[i] & 0x7FFFu, hi = (w[i] >> 16) & 0x7FFFu;
        top = max(top, max(lo < 0x7F80u ? lo : 0u, hi < 0x7F80u ? hi : 0u));
      }
    }
    __syncwarp();
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    const int e = max((int)(top >> 7), 33);              // biased exponent of the largest; 2^(142 - e) takes it to 2^15
    const float up = __uint_as_float((uint32_t)(269 - e) << 23);
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      mx4_mul_f32x2(f[2 * i], f[2 * i + 1], up, up);
    }
    auto pack = [](float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); };
    *reinterpret_cast<uint4*>(p) = make_uint4(pack(f[0], f[2]), pack(f[4], f[6]), pack(f[1], f[3]), pack(f[5], f[7]));
    return __uint_as_float((uint32_t)(e - 15) << 23);
  }
}

template <int FMT, typename T, int NB>
__global__ void __launch_bounds__((MV4_WARPS + 1 + 2 * NB) * 32, 2) mx4_mv_kernel(const __grid_constant__ Mx4Job J) {
  using C = Mv4<FMT, T, NB>;
  constexpr int TILE = mx4_tile_bytes(FMT), STAGE = C::STAGE, STAGES = C::STAGES;
  extern __shared__ __align__(128) uint8_t ring[];
  float* red = reinterpret_cast<float*>(ring + STAGES * STAGE);                      // [2][8 NB][128]
  uint64_t* full = reinterpret_cast<uint64_t*>(red + 2 * 8 * NB * MX4_ROWS);
  uint64_t* empty = full + STAGES;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + STAGES);
  const Mx4Lists L(const_cast<int*>(abort_flag) + 2, J.experts);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1 + C::X_WARPS); mbar_init(&empty[s], MV4_WARPS); }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (J.offsets) pdl_wait();
  mx4_groups(J, L);                                      // (ends with a block barrier)
  pdl_trigger();
  const int tiles = min(L.pre[J.experts], J.max_tiles) * J.m_tiles;
  const int first = blockIdx.x / J.split, step = gridDim.x / J.split, rank = blockIdx.x % J.split;
  const int k0 = rank * J.k_tiles / J.split, k1 = (rank + 1) * J.k_tiles / J.split;
  uint32_t loads = 0;
  bool ok = true;
  Mx4Factor factor{1.0f, 1.0f};
  if (J.split > 1) cluster_arrive();

  if (warp == MV4_WARPS) {
    if (lane == 0) {
      Mx4Pos p;
      if (!J.offsets) {                                  // on their way to L2 while the kernel in front ends (which may write them: none is read)
        const Mx4Walk t(L, J.experts, first, step, tiles, J.m_tiles);
        if (t.more())
          for (int k = k0; k < min(k0 + STAGES, k1); ++k) bulk_prefetch_l2(J.image + (((long long)t.expert * J.m_tiles + t.mt) * J.k_tiles + k) * TILE, TILE);
      }
      pdl_wait();
      for (Mx4Walk t(L, J.experts, first, step, tiles, J.m_tiles); t.more() && ok; t.next(L)) {
        const long long at = (long long)t.expert * J.m_tiles + t.mt;
        const uint8_t* src = J.image + (at * J.k_tiles + k0) * TILE;
        for (int k = k0; k < k1; ++k, ++loads, src += TILE, p.add(1, STAGES)) {
          const uint32_t tops = FMT == GLQB_MX4_MXFP4 && k == k0 ? 2 * MX4_ROWS : 0;
          if (!mbar_wait(&empty[p.s], p.phase ^ 1u, abort_flag)) { ok = false; break; }
          mbar_expect_tx(&full[p.s], TILE + tops);
          bulk_g2s(ring + p.s * STAGE, src, TILE, &full[p.s]);
          if (tops) bulk_g2s(ring + p.s * STAGE + TILE, J.tops + at * MX4_ROWS, tops, &full[p.s]);
        }
      }
      if (!ok) { *abort_flag = 1; atomicCAS(J.status, 0, (int)ST_GAVE_UP_LOADER); }
    }
  } else if (warp > MV4_WARPS) {
    // four rows of x each: those of the next tile are on their way while the last ones are written
    pdl_wait();
    constexpr int OWN = 8 * NB / C::X_WARPS;
    const int mine = warp - MV4_WARPS - 1;
    Mx4Walk t(L, J.experts, first, step, tiles, J.m_tiles);
    int k = k0, rows = 0;
    const T* at = nullptr;                               // of row `mine`
    auto place = [&]() {
      rows = t.more() ? t.rows : 0;
      at = reinterpret_cast<const T*>(J.x) + (long long)(t.row0 + mine) * J.x_stride + k0 * MX4_K + lane * 8;
    };
    auto fetch = [&](uint4 (&raw)[OWN]) {
      const bool in = k * MX4_K + lane * 8 < J.n;        // (n is a multiple of eight)
#pragma unroll
      for (int n = 0; n < OWN; ++n) {
        raw[n] = make_uint4(0, 0, 0, 0);
        if (mine + C::X_WARPS * n < rows && in) raw[n] = *reinterpret_cast<const uint4*>(at + C::X_WARPS * n * J.x_stride);
      }
      at += MX4_K;
    };
    auto put = [&](const uint4 (&raw)[OWN], int there, const Mx4Pos& p) -> bool {
      if (!mbar_wait_warp(&empty[p.s], p.phase ^ 1u, abort_flag)) return false;
      uint8_t* stage = ring + p.s * STAGE;
#pragma unroll
      for (int n = 0; n < OWN; ++n) {
        const int row = mine + C::X_WARPS * n;
        if (row >= there) break;
        const float down = put8<T>(stage + C::X + row * MV4_X_ROW + lane * 16, raw[n]);
        if (lane == 0) *reinterpret_cast<float*>(stage + C::X_SCALE + row * 4) = down;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[p.s]);
      return true;
    };
    Mx4Pos p;
    uint4 now[OWN];
    place();
    if (rows) fetch(now);
    while (rows && ok) {
      const int there = rows;
      if (++k == k1) {
        k = k0;
        t.next(L);
        place();
      }
      uint4 next[OWN];
      if (rows) fetch(next);
      ok = put(now, there, p);
#pragma unroll
      for (int n = 0; n < OWN; ++n) now[n] = next[n];
      p.add(1, STAGES);
    }
    if (!ok) { *abort_flag = 1; if (lane == 0) atomicCAS(J.status, 0, (int)ST_GAVE_UP_LOADER); }
  } else {
    pdl_wait();                                          // (y may still be in use)
    mx4_clear_rest(J, L.eff, threadIdx.x, MV4_WARPS * 32);
    const int g = lane >> 2, t = lane & 3, r = warp * 16 + g;
    const uint32_t codes0 = (uint32_t)(warp * 2048 + g * 128 + (g << 4) + t * 4);
    const uint32_t scales0 = (uint32_t)(MX4_CODE_BYTES + (r & 31) * 16 + (r >> 5) * 4), x0 = (uint32_t)(C::X + g * MV4_X_ROW + t * 16);
    const uint32_t pick = (uint32_t)(t >> 1) | (uint32_t)((t >> 1) + 2) << 4;
    constexpr int WORDS = FMT == GLQB_MX4_MXFP4 ? 2 : 4;
    int turn = 0;
    Mx4Pos p;
    // (A lane whose wait gave up goes through the rest without waiting, with what lies there: the others of its warp meet it at votes and
    // matrix instructions, and other warps at the barriers.  A vote per wait took 56.5 -> 57.5 us for 256 rows over 128 experts of 1536 x 2048.)
    for (Mx4Walk tile(L, J.experts, first, step, tiles, J.m_tiles); tile.more(); tile.next(L)) {
      int top[2] = {0, 0};
      bool plain = true;                                 // rows that the short form of the multiplier covers
      Mx4Factor f{1.0f, 1.0f};
      if constexpr (FMT == GLQB_MX4_NVFP4) f.b = J.w_scale[tile.expert];
      float acc[NB][4] = {};
      for (int k = k0; k < k1; ++k, p.add(1, STAGES)) {
        if (ok && !mbar_wait(&full[p.s], p.phase, abort_flag)) { ok = false; *abort_flag = 1; }
        const uint8_t* stage = ring + p.s * STAGE;
        if constexpr (FMT == GLQB_MX4_MXFP4) {
          if (k == k0) {
            const uint16_t* tops = reinterpret_cast<const uint16_t*>(stage + TILE);
            top[0] = tops[r];
            top[1] = tops[r + 8];
            plain = !__any_sync(0xFFFFFFFFu, ((top[0] | top[1]) & 256) != 0);
            top[0] = mx4_base(top[0] & 255);
            top[1] = mx4_base(top[1] & 255);
            f = mx4_power<__nv_bfloat16>(tops[threadIdx.x & 127]);
          }
        }
        uint32_t sw[2][WORDS];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int a = 0; a < WORDS; ++a) sw[h][a] = *reinterpret_cast<const uint32_t*>(stage + scales0 + 128 * h + 512 * a);
        float d[NB][4];                                  // of the tile's values
        auto codes = [&](int j, uint32_t (&w)[2][4]) {   // of unit j, rows g and g + 8
          const uint8_t* c = stage + (codes0 ^ (uint32_t)(j << 4));
          mx4_bytes_f16(*reinterpret_cast<const uint32_t*>(c), w[0]);
          mx4_bytes_f16(*reinterpret_cast<const uint32_t*>(c + 1024), w[1]);
        };
        auto values = [&](int j, uint4 (&b)[NB]) {
#pragma unroll
          for (int n = 0; n < NB; ++n) b[n] = *reinterpret_cast<const uint4*>(stage + x0 + n * 8 * MV4_X_ROW + j * 64);
        };
        if constexpr (FMT == GLQB_MX4_MXFP4) {
          // A unit is a block: codes are multiplied as they are, the sums by the block's power of two.
          auto units = [&](auto is_plain) {
            constexpr bool PLAIN = decltype(is_plain)::value;
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) d[n][e] = 0.0f;
            if constexpr (PLAIN) {
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int a = 0; a < WORDS; ++a) sw[h][a] -= (uint32_t)(top[h] - 127) * 0x01010101u;       // (76 .. 127 in every byte)
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              uint32_t w[2][4];
              uint4 b[NB];
              codes(j, w);
              values(j, b);
              const float p[2] = {block_power<PLAIN>(sw[0][j >> 2], j, top[0]), block_power<PLAIN>(sw[1][j >> 2], j, top[1])};
              const uint32_t a0[4] = {w[0][0], w[1][0], w[0][1], w[1][1]}, a1[4] = {w[0][2], w[1][2], w[0][3], w[1][3]};
#pragma unroll
              for (int n = 0; n < NB; ++n) {
                float part[4];
                mma16816_first(part, a0, b[n].x, b[n].y);
                mma16816(part, a1, b[n].z, b[n].w);
#pragma unroll
                for (int e = 0; e < 4; ++e) d[n][e] = fmaf(part[e], p[e >> 1], d[n][e]);
              }
            }
          };
          if (plain) units(std::true_type());
          else units(std::false_type());
        } else {
          float chain[NB][2][4] = {};                    // two chains of MMAs
#pragma unroll
          for (int i = 0; i < 4; ++i) {                  // two units of 16 bytes
            uint32_t m[2][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) multipliers(sw[h][i], pick, m[h]);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              uint32_t w[2][4];
              uint4 b[NB];
              codes(2 * i + u, w);
              values(2 * i + u, b);
#pragma unroll
              for (int v = 0; v < 2; ++v) {
                uint32_t a[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) a[e] = mx4_mul2<__half>(w[e & 1][2 * v + (e >> 1)], m[e & 1][u]);
#pragma unroll
                for (int n = 0; n < NB; ++n) mma16816(chain[n][v], a, v ? b[n].z : b[n].x, v ? b[n].w : b[n].y);
              }
            }
          }
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) d[n][e] = chain[n][0][e] + chain[n][1][e];
        }
        float shift = 1.0f;
        if constexpr (C::SHIFT) {
          asm volatile("" : "+f"(f.b));
          shift = fminf(fmaxf(__uint_as_float(__float_as_uint(f.b) & 0x7F800000u), 0x1p-31f), 1.0f);      // 2^mx4_shift(f.b, 0)
        }
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          float2 down = make_float2(1.0f, 1.0f);
          if constexpr (!__is_same(T, __half)) down = *reinterpret_cast<const float2*>(stage + C::X_SCALE + (n * 8 + 2 * t) * 4);
          if constexpr (C::SHIFT) { down.x *= shift; down.y *= shift; }       // (at least 2^-140: exact)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][e] = fmaf(d[n][e], e & 1 ? down.y : down.x, acc[n][e]);
        }
        __syncwarp();
        if (lane == 0 && ok) mbar_arrive(&empty[p.s]);
      }
      if (J.split > 1) {
        // Each column of a shared tile has a CTA that adds it up: the parts go to its memory, part by part.
        cluster_wait();                                  // (all have begun)
        const int owned = (8 * NB + J.split - 1) / J.split;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int c = n * 8 + 2 * t + (e & 1);
            st_cluster(smem_u32(red) + (uint32_t)((rank * owned + c / J.split) * MX4_ROWS + r + 8 * (e >> 1)) * 4u, c % J.split, acc[n][e]);
          }
        factor = f;
        continue;
      }
      // (two buffers in turn: a tile's sums are read before the barrier of the next one's)
      float* sums = red + (turn++ & 1) * (8 * NB * MX4_ROWS);
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[(n * 8 + 2 * t + (e & 1)) * MX4_ROWS + r + 8 * (e >> 1)] = acc[n][e];
      __syncwarp();
      asm volatile("bar.sync 1, 256;" ::: "memory");
      settle_factor<C::SHIFT>(f);
      const int row = tile.mt * MX4_ROWS + (threadIdx.x & 127);
      if (row < J.m)
        for (int c = threadIdx.x >> 7; c < tile.rows; c += 2)
          mx4_put(J, (long long)(tile.row0 + c) * J.y_stride + row, sums[c * MX4_ROWS + (threadIdx.x & 127)] * f.a * f.b);
    }
    if (!ok) atomicCAS(J.status, 0, (int)ST_GAVE_UP_PRODUCER);
  }
  __syncwarp();
  if (J.split > 1) {                                     // (one tile per cluster)
    if (first >= tiles || warp >= MV4_WARPS) cluster_wait();
    cluster_sync();
    if (first < tiles && warp < MV4_WARPS) {
      settle_factor<C::SHIFT>(factor);
      const Mx4Walk t(L, J.experts, first, step, tiles, J.m_tiles);
      const int r = threadIdx.x & 127, row = t.mt * MX4_ROWS + r, owned = (8 * NB + J.split - 1) / J.split;
      if (row < J.m)
        for (int c = threadIdx.x >> 7; c * J.split + rank < t.rows; c += 2) {
          float v = 0.0f;
#pragma unroll
          for (int s = 0; s < 8; ++s)
            if (s < J.split) v += red[(s * owned + c) * MX4_ROWS + r];
          mx4_put(J, (long long)(t.row0 + c * J.split + rank) * J.y_stride + row, v * factor.a * factor.b);
        }
    }
  }
  __syncthreads();
  if (*abort_flag && warp == MV4_WARPS && lane == 0)     // copies still under way
    for (uint32_t n = 0; n < min(loads, (uint32_t)STAGES); ++n) mbar_wait(&full[(loads - 1 - n) % STAGES], ((loads - 1 - n) / STAGES) & 1u);
}

}  // namespace

template <int F, typename T, int NB>
static size_t mv_smem(int experts) {
  using C = Mv4<F, T, NB>;
  return (size_t)C::STAGES * (C::STAGE + 16) + 2 * 8 * NB * MX4_ROWS * 4 + 8 + (size_t)(experts + 1) * 12;
}
int mx4_mv_clusters(int split) { return mx4_clusters(mx4_mv_kernel<GLQB_MX4_MXFP4, __half, 1>, Mv4<GLQB_MX4_MXFP4, __half, 1>::THREADS, mv_smem<GLQB_MX4_MXFP4, __half, 1>(1), split); }

cudaError_t mx4_mv_launch(int format, bool x_bf16, const Mx4Job& J, int sm_count, cudaStream_t stream) {
  const int nb = J.tn / 8;
  const long long tiles = (long long)J.max_tiles * J.m_tiles;
  const int grid = J.split > 1 ? (int)(tiles * J.split) : (int)std::min<long long>(tiles, 2ll * sm_count);
  auto run = [&](auto fmt, auto type, auto blocks) {
    using T = decltype(type);
    constexpr int F = decltype(fmt)::value, NB = decltype(blocks)::value;
    constexpr auto K = mx4_mv_kernel<F, T, NB>;
    return mx4_launch<K>(K, grid, Mv4<F, T, NB>::THREADS, mv_smem<F, T, NB>(J.experts), J.split, stream, J);
  };
  using M = std::integral_constant<int, GLQB_MX4_MXFP4>;
  using N = std::integral_constant<int, GLQB_MX4_NVFP4>;
  auto of = [&](auto blocks) {
    if (format == GLQB_MX4_MXFP4) return x_bf16 ? run(M(), __nv_bfloat16(), blocks) : run(M(), __half(), blocks);
    return x_bf16 ? run(N(), __nv_bfloat16(), blocks) : run(N(), __half(), blocks);
  };
  return nb == 1 ? of(std::integral_constant<int, 1>()) : of(std::integral_constant<int, 2>());
}

}  // namespace glqb
