// Rotary positions, appending to a paged cache, and attention of few rows over one: between a decoder's q/k/v and output projections.
#include "glqb_paged.cuh"
#include <algorithm>
#include <utility>
#include <atomic>
#include <chrono>
#include <climits>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <mutex>

namespace glqb {
namespace {

__device__ int g_paged_status;      // 0, or what gave up (ST_GAVE_UP_*): calls have no plan to keep it in
__device__ unsigned g_paged_gave_up; // how often

// ---- rotation and append --------------------------------------------------------------------------
// Heads of every token, in up to three parts (queries, keys, values).  One pass: a thread moves two pieces of eight values, those that
// are rotated with each other (half layout: i and i + pairs apart; interleaved: 16 consecutive values), or 16 that are not rotated.
// Bound by memory, or for few tokens by the launch.  Sines are of a token, not of a head: a block computes those of its tokens once.
constexpr int ROT_THREADS = 256, ROT_TOKENS = 4, ROT_UNITS = 8192;       // tokens and units of a block, at most
struct RotPart {
  const uint8_t* src;
  uint8_t* dst;
  long long src_token, src_head, dst_token, dst_head;    // (paged: dst_token a row's stride)
  long long dst_page;
  int heads, turn, paged;
};
struct RotJob {
  RotPart part[3];
  int heads;                        // of all parts
  const void *positions, *slots;
  const unsigned long long* turns;
  long long tokens, cache_rows;
  int positions_wide, slots_wide, page_log, head_dim, pairs, interleaved;
  int per_block, head_blocks, block_heads, units;        // tokens of a block, blocks that share a token's heads, their heads, units of a head
  uint32_t unit_mul, head_mul;                           // ceil(2^32 / units), ceil(2^32 / block_heads), 0 for 1
  float scale;
};

template <typename T> struct Eight;                      // eight values as they lie
template <> struct Eight<float> { float4 a, b; };
template <> struct Eight<__half> { uint4 a; };
template <> struct Eight<__nv_bfloat16> { uint4 a; };
// (read once: the first to leave L2, where what is written should stay.  4096 tokens appended: 27.7 us, 24.6 so)
template <typename T>
__device__ __forceinline__ Eight<T> load_eight(const T* p) {
  Eight<T> e;
  if constexpr (__is_same(T, float)) {
    e.a = __ldcs(reinterpret_cast<const float4*>(p));
    e.b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
  } else {
    e.a = __ldcs(reinterpret_cast<const uint4*>(p));
  }
  return e;
}
template <typename T>
__device__ __forceinline__ void to_floats(const Eight<T>& e, float (&v)[8]) {
  if constexpr (__is_same(T, float)) {
    v[0] = e.a.x; v[1] = e.a.y; v[2] = e.a.z; v[3] = e.a.w; v[4] = e.b.x; v[5] = e.b.y; v[6] = e.b.z; v[7] = e.b.w;
  } else {
    const uint32_t w[4] = {e.a.x, e.a.y, e.a.z, e.a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = pa_unpack<T>(w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ Eight<T> from_floats(const float (&v)[8]) {
  Eight<T> e;
  if constexpr (__is_same(T, float)) {
    e.a = make_float4(v[0], v[1], v[2], v[3]);
    e.b = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    e.a = make_uint4(pa_pack<T>(v[0], v[1]), pa_pack<T>(v[2], v[3]), pa_pack<T>(v[4], v[5]), pa_pack<T>(v[6], v[7]));
  }
  return e;
}
__device__ __forceinline__ void rotate_neighbours(float (&v)[8], const float2* cs, int step) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const float2 f = cs[j / 2 * step];
    const float a = v[j];
    v[j] = a * f.x - v[j + 1] * f.y;
    v[j + 1] = v[j + 1] * f.x + a * f.y;
  }
}

// TI: queries, keys and values as they come; TC: the cache's type (queries keep theirs).  WIDE: all pieces are whole and lie on 16 bytes.
template <typename TI, typename TC, bool WIDE>
__global__ void __launch_bounds__(ROT_THREADS) rotary_append_kernel(const __grid_constant__ RotJob J) {
  // Cosine and sine by token and pair; of WIDE units pairs p, p + 8, .. lie one behind the other, so that the units of neighbouring lanes are in
  // different banks (8191 tokens x 40 heads: 34 us in the order of the pairs, 30 so).
  extern __shared__ float2 turn_of[];
  __shared__ long long row_of[ROT_TOKENS];                      // row of the cache of each token, -1: none
  pdl_wait();
  pdl_trigger();
  const int block = blockIdx.x / J.head_blocks, head0 = (blockIdx.x % J.head_blocks) * J.block_heads;
  const long long token0 = (long long)block * J.per_block;
  const int n = (int)min((long long)J.per_block, J.tokens - token0), heads = min(J.block_heads, J.heads - head0);
  const int eighths = (J.pairs + 7) / 8, sines = WIDE ? eighths * 8 : J.pairs;
  for (int i = threadIdx.x; i < n * J.pairs; i += ROT_THREADS) {
    const int t = i / J.pairs, p = i - t * J.pairs;
    const long long pos = J.positions_wide ? reinterpret_cast<const long long*>(J.positions)[token0 + t] : reinterpret_cast<const int*>(J.positions)[token0 + t];
    // the fraction of a turn, as a signed 64-bit number: whole turns are what the product loses
    float s, c;
    sincospif((float)(long long)((unsigned long long)pos * J.turns[p]) * 0x1p-63f, &s, &c);
    turn_of[t * sines + (WIDE ? (p & 7) * eighths + (p >> 3) : p)] = make_float2(c * J.scale, s * J.scale);
  }
  if (J.slots && threadIdx.x < n) {
    const long long s = J.slots_wide ? reinterpret_cast<const long long*>(J.slots)[token0 + threadIdx.x] : reinterpret_cast<const int*>(J.slots)[token0 + threadIdx.x];
    row_of[threadIdx.x] = s >= 0 && s < J.cache_rows ? s : -1;
  }
  __syncthreads();
  const int total = n * J.block_heads * J.units;         // (below 2^16, so that a product divides exactly)
  for (int i = threadIdx.x; i < total; i += ROT_THREADS) {
    const int hu = J.unit_mul ? (int)__umulhi((uint32_t)i, J.unit_mul) : i, u = i - hu * J.units;
    const int t = J.head_mul ? (int)__umulhi((uint32_t)hu, J.head_mul) : hu, hr = hu - t * J.block_heads;
    if (hr >= heads) continue;
    int h = head0 + hr, k = 0;
    while (h >= J.part[k].heads) h -= J.part[k++].heads;
    const RotPart& P = J.part[k];
    const TI* src = reinterpret_cast<const TI*>(P.src) + (token0 + t) * P.src_token + h * P.src_head;
    long long at;
    if (P.paged) {
      const long long row = row_of[t];
      if (row < 0) continue;
      at = (row >> J.page_log) * P.dst_page + (row & ((1ll << J.page_log) - 1)) * P.dst_token + h * P.dst_head;
    } else {
      at = (token0 + t) * P.dst_token + h * P.dst_head;
    }
    const float2* cs = turn_of + t * sines;
    auto run = [&](auto type) {
      using TO = decltype(type);
      TO* dst = reinterpret_cast<TO*>(P.dst) + at;
      if constexpr (WIDE) {
        const bool apart = P.turn && !J.interleaved && u * 8 < J.pairs;
        const int first = apart ? u * 8 : u * 16, second = apart ? first + J.pairs : first + 8;
        const bool two = second < J.head_dim;
        float x[8], y[8];
        const Eight<TI> ex = load_eight(src + first), ey = two ? load_eight(src + second) : Eight<TI>{};
        to_floats<TI>(ex, x);
        to_floats<TI>(ey, y);
        if (apart) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float2 f = cs[j * eighths + u];
            const float v = x[j];
            x[j] = v * f.x - y[j] * f.y;
            y[j] = y[j] * f.x + v * f.y;
          }
        } else if (P.turn && J.interleaved) {
          if (first < 2 * J.pairs) rotate_neighbours(x, cs + u, eighths);
          if (second < 2 * J.pairs) rotate_neighbours(y, cs + 4 * eighths + u, eighths);
        }
        *reinterpret_cast<Eight<TO>*>(dst + first) = from_floats<TO>(x);
        if (two) *reinterpret_cast<Eight<TO>*>(dst + second) = from_floats<TO>(y);
      } else {
        // one pair, or one value that is not rotated; of a part without rotation one value, and the `pairs` last ones as second ones
        const int behind = J.head_dim - J.pairs + u;
        if (P.turn && u < J.pairs) {
          const int a = J.interleaved ? 2 * u : u, b = J.interleaved ? a + 1 : u + J.pairs;
          const float2 f = cs[u];
          const float v = (float)src[a], w = (float)src[b];
          dst[a] = pa_round<TO>(v * f.x - w * f.y);
          dst[b] = pa_round<TO>(w * f.x + v * f.y);
        } else if (P.turn) {
          dst[u + J.pairs] = pa_round<TO>((float)src[u + J.pairs]);
        } else {
          dst[u] = pa_round<TO>((float)src[u]);
          if (u < J.pairs) dst[behind] = pa_round<TO>((float)src[behind]);
        }
      }
    };
    if (P.paged) run(TC());
    else run(TI());
  }
}

// ---- attention of few rows ------------------------------------------------------------------------
// Sixteen rows (heads of a group that share a key head, times queries) against tiles of 64 keys: what bounds it is reading the cache.  One token of
// 131072 keys, fp16, 8 key heads of 128 values: 537 MB in 91.4 us, 5.87 TB/s; 64 sequences of up to 8192: 1.11 GB in 173 to 175 us, 6.4 TB/s.  Small calls are
// latency: one token of 4096 keys, 8.4 MB over 4 key heads, 11.5 us.
// Two warps bring tiles of keys and of values by TMA into a ring, a page's rows per copy, under the 128-byte swizzle (one warp that brings both was
// what a tile of four pages waited for); four warps multiply, each 16
// keys of every tile for itself (mma.sync: with so few rows the tensor cores are idle either way), with a running maximum and sum of its own, and add up when
// the item ends.  Scores are scale * log2(e) * q k, weights 2^(score - reference): the reference follows the largest score only when
// that has grown by more than 2^8, which scales all weights of a row alike and leaves their precision as it is.  Weights are rounded to the values'
// type for the product, as the tensor cores take them (fp16 ones are 2^7 larger: pa_up); sums stay in fp32.
constexpr int ST_WARPS = 4, ST_THREADS = (ST_WARPS + 2) * 32, ST_ITEMS = 4;
template <int DP>
struct StreamShape {
  static constexpr int HALF = PA_STREAM_KEYS * 128, K_BYTES = HALF * (DP / 64), STAGE = 2 * K_BYTES, STAGES = 96 * 1024 / STAGE;
};
struct __align__(16) StreamShared {
  PagedStart start;
  PagedItem item[ST_ITEMS];
  float2 ml[ST_WARPS][PA_STREAM_ROWS];
  uint64_t full[8], empty[8], item_full[ST_ITEMS], item_empty[ST_ITEMS], joined[2];
  int abort;
};
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (__is_same(T, __half))
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// parts of a row, added up: 4 Q of its values
template <int Q>
struct Joined {
  float4 v[Q];
  float most, sum;
  __device__ __forceinline__ Joined() : most(-INFINITY), sum(0.0f) {
#pragma unroll
    for (int q = 0; q < Q; ++q) v[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  template <int N>
  __device__ __forceinline__ void add(const float2 (&ml)[N], const float4 (&u)[N][Q]) {
    float now = most;
#pragma unroll
    for (int k = 0; k < N; ++k) now = fmaxf(now, ml[k].x);
    const float f = now == -INFINITY ? 1.0f : pa_exp2(most - now);
    sum *= f;
#pragma unroll
    for (int q = 0; q < Q; ++q) { v[q].x *= f; v[q].y *= f; v[q].z *= f; v[q].w *= f; }
    most = now;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (ml[k].x == -INFINITY && ml[k].y == 0.0f) continue;        // (no key of its own: nothing in its sums)
      const float w = pa_exp2(ml[k].x - now);
      sum += w * ml[k].y;
#pragma unroll
      for (int q = 0; q < Q; ++q) { v[q].x += w * u[k][q].x; v[q].y += w * u[k][q].y; v[q].z += w * u[k][q].z; v[q].w += w * u[k][q].w; }
    }
  }
};
template <typename T, int DP>
__global__ void __launch_bounds__(ST_THREADS, 2)
paged_stream_kernel(const __grid_constant__ PagedJob J, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  using C = StreamShape<DP>;
  constexpr int ROWS = PA_STREAM_ROWS, KEYS = PA_STREAM_KEYS, STEPS = DP / 16;      // (J.rows is ROWS)
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  StreamShared& B = *reinterpret_cast<StreamShared*>(ring + C::STAGES * C::STAGE);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) { mbar_init(&B.full[s], 2); mbar_init(&B.empty[s], ST_WARPS); }
    for (int s = 0; s < ST_ITEMS; ++s) { mbar_init(&B.item_full[s], 1); mbar_init(&B.item_empty[s], ST_WARPS + 1); }
    for (int s = 0; s < 2; ++s) mbar_init(&B.joined[s], ST_WARPS);
    B.abort = 0;
    fence_mbar_init();
  }
  if (warp == ST_WARPS && lane < 2) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(lane ? &map_v : &map_k)) : "memory");
  pdl_wait();
  pdl_trigger();
  pa_start<KEYS>(J, B.start);
  bool ok = true;

  if (warp >= ST_WARPS) {
    // the first of the two makes the list of items, the second one takes it from there, as the others do
    const bool values = warp > ST_WARPS;
    const CUtensorMap* map = values ? &map_v : &map_k;
    PagedWalk<KEYS, true> walk(J, B.start);
    const int piece = min(1 << J.page_log, PA_PIECE), pieces = KEYS / piece, page_mask = (1 << J.page_log) - 1;
    uint32_t stage = 0, phase = 1, ip = values ? 0 : 1, filled = 0;
    int is = 0;
    auto advance = [&] { ++filled; if (++stage == C::STAGES) { stage = 0; phase ^= 1u; } };
    for (;;) {
      PagedItem it;
      if (!values) it = walk.next(J);
      ok = ok && mbar_wait_warp(values ? &B.item_full[is] : &B.item_empty[is], ip, &B.abort);
      if (!ok) break;
      if (values) it = B.item[is];
      else if (lane == 0) B.item[is] = it;
      __syncwarp();
      if (lane == 0) mbar_arrive(values ? &B.item_empty[is] : &B.item_full[is]);
      if (!it.more) break;
      if (++is == ST_ITEMS) { is = 0; ip ^= 1u; }
      const int* table = J.pages + (long long)it.seq * J.page_stride;
      for (int tile = it.lo; tile < it.hi; ++tile) {
        const int left = it.keys - tile * KEYS, here = max(0, min(pieces, (left + piece - 1) / piece));       // pieces that hold keys
        int page = 0;
        if (lane < here) page = table[(tile * KEYS + lane * piece) >> J.page_log];
        if (!mbar_wait_warp(&B.empty[stage], phase, &B.abort)) { ok = false; break; }
        uint8_t* at = ring + stage * C::STAGE + (values ? C::K_BYTES : 0);
        if (lane == 0) mbar_expect_tx(&B.full[stage], (uint32_t)(here * piece) * (DP * 2));
        __syncwarp();
        if (lane < here) {
          const int row = (tile * KEYS + lane * piece) & page_mask;
#pragma unroll
          for (int h = 0; h < DP / 64; ++h) pa_load(at + h * C::HALF + lane * piece * 128, map, h * 64, it.kv_head, row, page, &B.full[stage]);
        }
        __syncwarp();
        advance();
      }
      if (!ok) break;
      // a stage without a tile: where the warps add up
      if (!mbar_wait_warp(&B.empty[stage], phase, &B.abort)) { ok = false; break; }
      if (lane == 0) mbar_arrive(&B.full[stage]);
      advance();
    }
    if (lane == 0) {
      if (!ok) { *(volatile int*)&B.abort = 1; atomicCAS(J.status, 0, (int)ST_GAVE_UP_LOADER); atomicAdd(J.gave_up, 1u); }
    }
    // copies in flight land before the block ends (a stage that the other of the two did not fill does not: the wait is bounded)
    if (!ok)
      for (uint32_t n = 1; n <= min(filled, (uint32_t)C::STAGES); ++n) mbar_wait(&B.full[(filled - n) % C::STAGES], (filled - n) / C::STAGES & 1u);
  } else {
    const int g = lane >> 2, t4 = lane & 3;
    const unsigned long long tag = (J.tag + *(volatile unsigned*)J.gave_up * 0x9E3779B97F4A7ull) & ((1ull << 52) - 1) | 1ull;
    if (J.clear) {
      const int first = pa_offset(J, 0), last = max(first, pa_offset(J, J.seqs)), rest = J.tokens - (last - first);
      for (int i = blockIdx.x; i < rest; i += gridDim.x) {
        T* p = reinterpret_cast<T*>(J.out) + (long long)(i < first ? i : i + last - first) * J.out_token;
        for (int k = threadIdx.x; k < J.heads * J.head_dim; k += ST_WARPS * 32) p[k / J.head_dim * J.out_head + k % J.head_dim] = pa_round<T>(0.0f);
      }
    }
    uint32_t stage = 0, phase = 0, ip = 0, turn = 0;
    int is = 0;
    auto advance = [&] { if (++stage == C::STAGES) { stage = 0; phase ^= 1u; } };
    // this warp's lanes in a tile: addresses of fragments but for the 16-byte column
    const uint32_t k_row = (uint32_t)(warp * 16 + ((lane >> 4) << 3) + (lane & 7)), v_row = (uint32_t)(warp * 16 + (lane & 15));
    const uint32_t k_col = (lane >> 3) & 1, v_col = lane >> 4;
    for (;;) {
      if (!mbar_wait_warp(&B.item_full[is], ip, &B.abort)) { ok = false; break; }
      const PagedItem it = B.item[is];
      __syncwarp();
      if (lane == 0) mbar_arrive(&B.item_empty[is]);
      if (!it.more) break;
      if (++is == ST_ITEMS) { is = 0; ip ^= 1u; }
      if (lane == 0 && it.slot >= 0 && warp * (128 / DP) < it.rows) pa_open(J.tickets + it.begun_by * ST_WARPS + warp, tag);
      // queries as fragments: rows g and g + 8
      uint32_t q[STEPS][4];
      int to[2], from[2];
      const PagedSeq seq{it.row0, it.queries, it.keys};
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const int row = it.first + min(g + 8 * a, it.rows - 1), i = pa_query(J, row);
        to[a] = pa_to(J, seq, i);
        from[a] = pa_from(J, seq, i);
        const bool there = g + 8 * a < it.rows;
        const uint16_t* src = J.q + (long long)(it.row0 + i) * J.q_token + (long long)(it.kv_head * J.group + row - i * J.group) * J.q_head;
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int col = s * 16 + b * 8 + t4 * 2;
            q[s][a + 2 * b] = there && col < J.head_dim ? *reinterpret_cast<const uint32_t*>(src + col) : 0u;
          }
      }
      const int all_from = it.all_from, all_to = it.all_to, any_from = it.any_from, any_to = it.any_to;
      float o[STEPS * 2][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
      for (int tile = it.lo; tile < it.hi; ++tile) {
        if (!mbar_wait_warp(&B.full[stage], phase, &B.abort)) { ok = false; break; }
        const int key0 = tile * KEYS + warp * 16;
        if (key0 < any_to && key0 + 16 > any_from) {
          const uint32_t base = smem_u32(ring) + stage * C::STAGE;
          float s[2][4] = {};
#pragma unroll
          for (int k = 0; k < STEPS; ++k) {
            uint32_t b[4];
            ldsm4(base + (k / 4) * C::HALF + k_row * 128 + ((((k % 4) * 2 + k_col) ^ (k_row & 7)) << 4), b);
            mma16816<T>(s[0], q[k], b[0], b[1]);
            mma16816<T>(s[1], q[k], b[2], b[3]);
          }
          const bool whole = key0 >= all_from && key0 + 16 <= all_to;
          // scores in powers of two; s[n][2 a + c]: row g + 8 a, key 8 n + 2 t4 + c
          uint32_t seen = 0xFFu;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s[n][e] *= J.scale_log2;
              if (!whole) {
                const int key = key0 + n * 8 + t4 * 2 + (e & 1);
                if (key < from[e >> 1] || key >= to[e >> 1]) { s[n][e] = -INFINITY; seen &= ~(1u << (n * 4 + e)); }
              }
            }
          float top[2], less[2];
          bool grown = false;
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            top[a] = fmaxf(fmaxf(s[0][2 * a], s[0][2 * a + 1]), fmaxf(s[1][2 * a], s[1][2 * a + 1]));
            top[a] = fmaxf(top[a], __shfl_xor_sync(0xFFFFFFFFu, top[a], 1));
            top[a] = fmaxf(top[a], __shfl_xor_sync(0xFFFFFFFFu, top[a], 2));
            grown = grown || top[a] > m[a] + PA_LAZY;
          }
          if (__any_sync(0xFFFFFFFFu, grown)) {
#pragma unroll
            for (int a = 0; a < 2; ++a) {
              const float now = fmaxf(m[a], top[a]), f = now == -INFINITY ? 1.0f : pa_exp2(m[a] - now);
              m[a] = now;
              l[a] *= f;
#pragma unroll
              for (int n = 0; n < STEPS * 2; ++n) { o[n][2 * a] *= f; o[n][2 * a + 1] *= f; }
            }
          }
#pragma unroll
          for (int a = 0; a < 2; ++a) less[a] = m[a] == -INFINITY ? 0.0f : m[a] - pa_up<T>();
          uint32_t p[4];
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int a = 0; a < 2; ++a) {
              const float u = pa_exp2(s[n][2 * a] - less[a]), v = pa_exp2(s[n][2 * a + 1] - less[a]);
              l[a] += u + v;
              p[n * 2 + a] = pa_pack<T>(u, v);
            }
          const uint32_t values = base + C::K_BYTES + v_row * 128;
          bool odd = false;
          if (!whole) {
            // Values in rows that a query does not see may be anything, NaN too: nothing times that is not nothing.  Rows that no query
            // sees (behind the sequence, in front of its window) are taken as zeros, and where others hold no finite value a slow path follows.
#pragma unroll
            for (int j = 0; j < STEPS; ++j) {
              uint32_t b[4];
              ldsm4_trans(values + (j / 4) * C::HALF + ((((j % 4) * 2 + v_col) ^ (v_row & 7)) << 4), b);
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const int key = key0 + (r & 1) * 8 + t4 * 2;
                if (key < any_from || key >= any_to) b[r] &= 0xFFFF0000u;
                if (key + 1 < any_from || key + 1 >= any_to) b[r] &= 0xFFFFu;
                odd = odd || pa_not_finite<T>(b[r]);
              }
            }
            odd = __any_sync(0xFFFFFFFFu, odd);
          }
          if (!odd) {
#pragma unroll
            for (int j = 0; j < STEPS; ++j) {
              uint32_t b[4];
              ldsm4_trans(values + (j / 4) * C::HALF + ((((j % 4) * 2 + v_col) ^ (v_row & 7)) << 4), b);
              if (!whole) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const int key = key0 + (r & 1) * 8 + t4 * 2;
                  if (key < any_from || key >= any_to) b[r] &= 0xFFFF0000u;
                  if (key + 1 < any_from || key + 1 >= any_to) b[r] &= 0xFFFFu;
                }
              }
              mma16816<T>(o[2 * j], p, b[0], b[1]);
              mma16816<T>(o[2 * j + 1], p, b[2], b[3]);
            }
          } else {
#pragma unroll 1
            for (int key = 0; key < 16; ++key) {
              // weights of rows g and g + 8: fragment register (key / 8) * 2 + a, half key % 2, of lane 4 g + key % 8 / 2
              const int src = (lane & 28) | ((key & 7) >> 1);
              float w[2];
              bool see[2];
#pragma unroll
              for (int a = 0; a < 2; ++a) {
                const uint32_t two = __shfl_sync(0xFFFFFFFFu, key < 8 ? p[a] : p[2 + a], src);
                const uint32_t flags = __shfl_sync(0xFFFFFFFFu, seen, src);
                const uint16_t half = (uint16_t)(key & 1 ? two >> 16 : two);
                w[a] = __is_same(T, __half) ? __half2float(__ushort_as_half(half)) : __uint_as_float((uint32_t)half << 16);
                see[a] = flags >> ((key >> 3) * 4 + 2 * a + (key & 1)) & 1u;
              }
              const uint32_t row = (uint32_t)(warp * 16 + key);
#pragma unroll
              for (int n = 0; n < STEPS * 2; ++n) {
                uint32_t two;
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(two) : "r"(base + C::K_BYTES + (n / 8) * C::HALF + row * 128 + (((n % 8) ^ (row & 7)) << 4) + t4 * 4) : "memory");
                const float2 v = pa_unpack<T>(two);
#pragma unroll
                for (int a = 0; a < 2; ++a)
                  if (see[a]) { o[n][2 * a] += w[a] * v.x; o[n][2 * a + 1] += w[a] * v.y; }
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.empty[stage]);
        advance();
      }
      if (!ok) break;
      // ---- the warps' sums together, in the order of the warps
      if (!mbar_wait_warp(&B.full[stage], phase, &B.abort)) { ok = false; break; }
      float* red = reinterpret_cast<float*>(ring + stage * C::STAGE);
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const int row = g + 8 * a;
        l[a] += __shfl_xor_sync(0xFFFFFFFFu, l[a], 1);
        l[a] += __shfl_xor_sync(0xFFFFFFFFu, l[a], 2);
        if (row < it.rows) {
          if (t4 == 0) B.ml[warp][row] = make_float2(m[a], l[a]);
#pragma unroll
          for (int n = 0; n < STEPS * 2; ++n) *reinterpret_cast<float2*>(red + (warp * ROWS + row) * DP + n * 8 + t4 * 2) = make_float2(o[n][2 * a], o[n][2 * a + 1]);
        }
      }
      // (not by a named barrier: a warp whose wait gave up does not come)
      __syncwarp();
      if (lane == 0) mbar_arrive(&B.joined[0]);
      if (!mbar_wait_warp(&B.joined[0], turn, &B.abort)) { ok = false; break; }
      const long long place = (2ll * blockIdx.x + max(it.slot, 0)) * ROWS;
      for (int i = threadIdx.x; i < it.rows * (DP / 4); i += ST_WARPS * 32) {
        const int row = i / (DP / 4), col = i % (DP / 4) * 4;
        float2 ml[ST_WARPS];
        float most = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < ST_WARPS; ++w) { ml[w] = B.ml[w][row]; most = fmaxf(most, ml[w].x); }
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < ST_WARPS; ++w) {
          if (ml[w].x == -INFINITY && ml[w].y == 0.0f) continue;      // (no key of its own: nothing in its sums)
          const float f = pa_exp2(ml[w].x - most);
          const float4 u = *reinterpret_cast<const float4*>(red + (w * ROWS + row) * DP + col);
          sum += f * ml[w].y;
          v.x += f * u.x; v.y += f * u.y; v.z += f * u.z; v.w += f * u.w;
        }
        if (it.slot < 0) {
          const float f = pa_row_factor(J, seq, it.first + row, sum);
          if (col < J.head_dim) pa_store4<T>(J, pa_out_row(J, it.row0, it.kv_head, it.first + row), col, make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
        } else {
          *reinterpret_cast<float4*>(J.part + (place + row) * DP + col) = v;
          if (col == 0) J.part_ml[place + row] = make_float2(most, sum);
        }
      }
      // (the sums lie where the next tile is copied to: ordinary stores are ordered before copies by this alone, not by the barrier)
      fence_async_smem();
      __syncwarp();
      if (lane == 0) { mbar_arrive(&B.joined[1]); mbar_arrive(&B.empty[stage]); }
      // An item that several CTAs have a part of: a warp has the same rows in each.  The last to arrive adds them up, all from the workspace, in the
      // order of the CTAs.  (In a launch of its own behind this one: 64 sequences of up to 8192 keys 178 us, 173 so.)
      if (it.slot >= 0 && warp * (128 / DP) < it.rows) {
        __threadfence();
        __syncwarp();
        int last = 0;
        if (lane == 0) last = pa_arrive(J.tickets + it.begun_by * ST_WARPS + warp, it.parts);
        if (__shfl_sync(0xFFFFFFFFu, last, 0)) {
          __threadfence();
          for (int i = threadIdx.x; i < it.rows * (DP / 4); i += ST_WARPS * 32) {
            const int row = i / (DP / 4), col = i % (DP / 4) * 4;
            Joined<1> j;
            for (int p0 = 0; p0 < it.parts; p0 += 8) {
              float2 ml[8];
              float4 u[8][1];
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                ml[k] = make_float2(-INFINITY, 0.0f);
                u[k][0] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (p0 + k < it.parts) {
                  const long long at = (2ll * (it.begun_by + p0 + k) + (p0 + k == 0)) * ROWS + row;
                  ml[k] = __ldcg(J.part_ml + at);
                  u[k][0] = __ldcg(reinterpret_cast<const float4*>(J.part + at * DP + col));
                }
              }
              j.add(ml, u);
            }
            const float f = pa_row_factor(J, seq, it.first + row, j.sum);
            if (col < J.head_dim) pa_store4<T>(J, pa_out_row(J, it.row0, it.kv_head, it.first + row), col, make_float4(j.v[0].x * f, j.v[0].y * f, j.v[0].z * f, j.v[0].w * f));
          }
          __syncwarp();
        }
      }
      if (!mbar_wait_warp(&B.joined[1], turn, &B.abort)) { ok = false; break; }       // (ml is read)
      turn ^= 1u;
      advance();
    }
    if (!ok && lane == 0) { *(volatile int*)&B.abort = 1; atomicCAS(J.status, 0, (int)ST_GAVE_UP_MMA); atomicAdd(J.gave_up, 1u); }
  }
}

// ---- what several CTAs have of an item of many rows, together -------------------------------------
// The parts of an item that CTA blockIdx.x began and did not end are that CTA's, then those of the CTAs behind it up to the one that ended
// the item.  A lane has 16 values of one row, a warp 32 rows, whose parts it reads a kilobyte at once.  The order is the same in every call.  Bound by latency and by
// blocks that wait for others to end: what a CTA has left, then the parts.  (Parts with a row's values one behind the other, a warp for two rows: prompt of 2048
// tokens 58.5 us, 52.1 so, 24 sequences of mixed lengths 55.0, 49.3; blocks of eight warps 52.8 and 49.4, three parts at once 53.9 and 50.1, one 53.5 and 51.0.
// One CTA could not do it in the first kernel, as it does with few rows: 256 rows of 18 CTAs are 2.4 MB.)
constexpr int CB_WARPS = 4, CB_BATCH = 2;
constexpr int cb_blocks(int dp) { return PA_TILE_ROWS / 32 * (dp / 16) / CB_WARPS; }        // of an item
template <typename T, int DP>
__global__ void __launch_bounds__(CB_WARPS * 32, 6) paged_combine_kernel(const __grid_constant__ PagedJob J, int ctas) {
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x;
  // (the first parts' ends are asked for before it is known whether this CTA has left a beginning)
  const PagedPart lead = J.part_of[2 * c + 1];
  auto ends = [&](int parts) {
    const int at = c + parts + lane;
    return __ballot_sync(0xFFFFFFFFu, at >= ctas || !J.part_of[2 * at].valid || J.part_of[2 * at].ends);
  };
  uint32_t end = ends(1);
  if (J.clear && blockIdx.y == 0) {
    const int first = pa_offset(J, 0), last = max(first, pa_offset(J, J.seqs)), rest = J.tokens - (last - first);
    for (int i = c; i < rest; i += gridDim.x) {
      T* p = reinterpret_cast<T*>(J.out) + (long long)(i < first ? i : i + last - first) * J.out_token;
      for (int k = threadIdx.x; k < J.heads * J.head_dim; k += CB_WARPS * 32) p[k / J.head_dim * J.out_head + k % J.head_dim] = pa_round<T>(0.0f);
    }
  }
  if (!lead.valid) return;
  int parts = 1;
  while (!end) end = ends(parts += 32);
  parts += __ffs(end);
  const int task = (int)blockIdx.y * CB_WARPS + warp, col = task % (DP / 16) * 16, r = task / (DP / 16) * 32 + lane;      // (r: 128 to a half)
  const int half = J.rows / 2, row = r < 128 ? r : half + r - 128;
  if ((r & 127) >= half || row >= lead.rows || col >= J.head_dim) return;
  Joined<4> j;
  for (int p0 = 0; p0 < parts; p0 += CB_BATCH) {
    float2 ml[CB_BATCH];
    float4 u[CB_BATCH][4];
#pragma unroll
    for (int k = 0; k < CB_BATCH; ++k) {
      ml[k] = make_float2(-INFINITY, 0.0f);
#pragma unroll
      for (int q = 0; q < 4; ++q) u[k][q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (p0 + k < parts) {
        const int slot = 2 * (c + p0 + k) + (p0 + k == 0);
        ml[k] = J.part_ml[(long long)slot * PA_TILE_ROWS + r];
#pragma unroll
        for (int q = 0; q < 2; ++q) load8(J.part + pa_part_at<DP>(slot, r, col / 8 + q), u[k][2 * q], u[k][2 * q + 1]);
      }
    }
    j.add(ml, u);
  }
  const float f = pa_row_factor(J, PagedSeq{lead.row0, lead.queries, lead.keys}, lead.first + row, j.sum);
  const long long at = pa_out_row(J, lead.row0, lead.kv_head, lead.first + row);
  if (J.out_sectors && col + 16 <= J.head_dim) {
    uint32_t y[8];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      y[2 * q] = pa_pack<T>(j.v[q].x * f, j.v[q].y * f);
      y[2 * q + 1] = pa_pack<T>(j.v[q].z * f, j.v[q].w * f);
    }
    store8(reinterpret_cast<uint16_t*>(J.out) + at + col, y);
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (col + 4 * q < J.head_dim) pa_store4<T>(J, at, col + 4 * q, make_float4(j.v[q].x * f, j.v[q].y * f, j.v[q].z * f, j.v[q].w * f));
  }
}

// ---- host -----------------------------------------------------------------------------------------
int pg_fail(int code, const char* fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  set_error_message(buf);
  return code;
}
int pg_launched(const char* what, cudaError_t e) { return e == cudaSuccess ? GLQB_OK : pg_fail(GLQB_E_CUDA, "%s: %s", what, cudaGetErrorString(e)); }
bool lies_on(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
bool dtype_ok(int d) { return d == GLQB_DT_F16 || d == GLQB_DT_BF16 || d == GLQB_DT_F32; }
size_t size_of(int d) { return d == GLQB_DT_F32 ? 4 : 2; }

struct PagedDevice {
  std::atomic<int> sms{0};
  int* status = nullptr;
  unsigned* gave_up = nullptr;
};
const PagedDevice* pg_device() {
  static PagedDevice known[64];
  static std::mutex building;
  PagedDevice& d = known[pg_device_index()];
  if (d.sms.load(std::memory_order_acquire) == 0) {
    std::lock_guard<std::mutex> lock(building);
    int n = 0;
    if (d.sms.load(std::memory_order_relaxed) == 0) {
      if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, pg_device_index()) != cudaSuccess || n < 1 ||
          cudaGetSymbolAddress(reinterpret_cast<void**>(&d.status), g_paged_status) != cudaSuccess ||
          cudaGetSymbolAddress(reinterpret_cast<void**>(&d.gave_up), g_paged_gave_up) != cudaSuccess)
        return nullptr;
      d.sms.store(n, std::memory_order_release);
    }
  }
  return &d;
}

int check_rotary(const GlqbRotary* r, int head_dim, const void* positions, int wide, const char* what) {
  if (!r->turns || !positions) return pg_fail(GLQB_E_INVALID, "%s: a rotation needs turns and positions", what);
  if (r->pairs < 1 || 2ll * r->pairs > head_dim) return pg_fail(GLQB_E_INVALID, "%s: %d pairs in heads of %d values", what, r->pairs, head_dim);
  if (!lies_on(r->turns, 8) || !lies_on(positions, wide ? 8 : 4)) return pg_fail(GLQB_E_INVALID, "%s: values that are not aligned", what);
  return GLQB_OK;
}
// tokens of a block, blocks per token, and the launch
template <typename TI, typename TC>
int rotary_launch(RotJob& J, int sms, cudaStream_t stream, const char* what) {
  bool wide = J.head_dim % 8 == 0 && J.pairs % (J.interleaved ? 4 : 8) == 0;
  J.heads = 0;
  for (const RotPart& p : J.part) {
    J.heads += p.heads;
    const size_t out = p.paged ? sizeof(TC) : sizeof(TI);
    const long long in = 16 / (long long)sizeof(TI), of = 16 / (long long)out;
    if (p.heads)
      wide = wide && lies_on(p.src, 16) && lies_on(p.dst, 16) && p.src_token % in == 0 && p.src_head % in == 0 && p.dst_token % of == 0 && p.dst_head % of == 0 && p.dst_page % of == 0;
  }
  J.units = wide ? (J.head_dim + 15) / 16 : J.head_dim - J.pairs;
  // a block has four tokens where that leaves eight blocks per SM, all heads of a token where they are fewer than ROT_UNITS units
  J.per_block = J.tokens >= 8ll * ROT_TOKENS * sms ? ROT_TOKENS : 1;
  J.block_heads = std::max(1, std::min(J.heads, ROT_UNITS / (J.units * J.per_block)));
  J.head_blocks = (J.heads + J.block_heads - 1) / J.block_heads;
  auto mul = [](int d) { return d == 1 ? 0u : (uint32_t)(((1ull << 32) + d - 1) / d); };
  J.unit_mul = mul(J.units);
  J.head_mul = mul(J.block_heads);
  const long long grid = (J.tokens + J.per_block - 1) / J.per_block * J.head_blocks;
  if (grid > INT_MAX) return pg_fail(GLQB_E_INVALID, "%s: %lld tokens of %d heads are too many for one call", what, J.tokens, J.heads);
  const size_t smem = (size_t)J.per_block * ((J.pairs + 7) / 8 * 8) * sizeof(float2);
  return pg_launched(what, wide ? launch_chained(true, rotary_append_kernel<TI, TC, true>, (int)grid, ROT_THREADS, smem, stream, J)
                                : launch_chained(true, rotary_append_kernel<TI, TC, false>, (int)grid, ROT_THREADS, smem, stream, J));
}
constexpr int ROT_MAX_DIM = 1024;        // of a head: its sines fit in a block's shared memory

int check_cache(const GlqbPagedCache* c, const char* what) {
  if (!c) return pg_fail(GLQB_E_INVALID, "%s: null argument", what);
  if (c->dtype != GLQB_DT_F16 && c->dtype != GLQB_DT_BF16) return pg_fail(GLQB_E_INVALID, "%s: a cache is fp16 or bf16", what);
  if (c->page_size < 8 || (c->page_size & (c->page_size - 1)) || c->page_size > 1 << 20)
    return pg_fail(GLQB_E_INVALID, "%s: pages of %d rows (a power of two, 8 at least)", what, c->page_size);
  if (c->head_dim < 8 || c->head_dim > 128 || c->head_dim % 8) return pg_fail(GLQB_E_INVALID, "%s: heads of %d values (a multiple of 8, 128 at most)", what, c->head_dim);
  if (c->kv_heads < 1 || c->kv_heads > 1 << 16 || c->pages < 1 || c->pages > INT_MAX) return pg_fail(GLQB_E_INVALID, "%s: %lld pages of %d heads", what, (long long)c->pages, c->kv_heads);
  if (!c->keys || !c->values) return pg_fail(GLQB_E_INVALID, "%s: null argument", what);
  const int64_t strides[6] = {c->key_page, c->key_row, c->key_head, c->value_page, c->value_row, c->value_head};
  for (const int64_t s : strides)
    if (s < 0 || s % 8 || s >= 1ll << 38) return pg_fail(GLQB_E_INVALID, "%s: a cache's strides are multiples of 8 values", what);
  if (!lies_on(c->keys, 16) || !lies_on(c->values, 16)) return pg_fail(GLQB_E_INVALID, "%s: a cache lies on 16 bytes", what);
  // no two rows in one place: each stride passes what the smaller ones reach over
  for (int i = 0; i < 6; i += 3) {
    std::pair<int64_t, int64_t> by[3] = {{strides[i], c->pages}, {strides[i + 1], c->page_size}, {strides[i + 2], c->kv_heads}};
    std::sort(by, by + 3);
    __int128 reach = c->head_dim;
    for (const auto& d : by)
      if (d.second > 1) {
        if (d.first < reach) return pg_fail(GLQB_E_INVALID, "%s: rows of a cache overlap", what);
        reach += (__int128)d.first * (d.second - 1);
      }
  }
  return GLQB_OK;
}

// Is |at + sum of e_i strides[i]| below `dim` for some |e_i| < counts[i]?  Strides pass what the ones behind them reach over, so that of each two e come into question.
bool rows_meet(__int128 at, const std::pair<int64_t, int64_t>* by, int n, int dim) {
  if (n == 0) return at < dim && at > -dim;
  const __int128 s = by->first, most = by->second - 1;
  const __int128 low = -(at >= 0 ? (at + s - 1) / s : at / s);       // floor(-at / s)
  for (__int128 e = low; e <= low + 1; ++e)
    if (e >= -most && e <= most && rows_meet(at + e * s, by + 1, n - 1, dim)) return true;
  return false;
}
// Have keys and values (check_cache) an address in common?  They may lie between one another, as those of one tensor do.
bool caches_meet(const GlqbPagedCache* c) {
  const __int128 at = ((__int128) reinterpret_cast<intptr_t>(c->values) - reinterpret_cast<intptr_t>(c->keys)) / 2;
  const int64_t k[3] = {c->key_page, c->key_row, c->key_head}, v[3] = {c->value_page, c->value_row, c->value_head}, n[3] = {c->pages, c->page_size, c->kv_heads};
  std::pair<int64_t, int64_t> by[3];
  int used = 0;
  bool alike = true;
  __int128 k_page = c->head_dim, v_page = c->head_dim;               // what a page reaches over
  for (int i = 0; i < 3; ++i) {
    if (n[i] < 2) continue;
    alike = alike && k[i] == v[i];
    by[used++] = {k[i], n[i]};
    if (i) k_page += (__int128)k[i] * (n[i] - 1), v_page += (__int128)v[i] * (n[i] - 1);
  }
  if (alike) {
    std::sort(by, by + used, [](const auto& a, const auto& b) { return a.first > b.first; });
    return rows_meet(at, by, used, c->head_dim);
  }
  const __int128 all = (__int128)(c->pages - 1);
  if (at >= k_page + all * k[0] || at + v_page + all * v[0] <= 0) return false;
  // rows or heads in another order: apart if whole pages are
  if (c->pages < 2 || k[0] != v[0] || k_page > k[0] || v_page > k[0]) return true;
  const __int128 r = (at % k[0] + k[0]) % k[0];
  return r < k_page || r + v_page > k[0];
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
// (a stride that a dimension of one place does not use has to be a multiple of 16 all the same, and so does one of 0 have to be more)
bool encode_cache(CUtensorMap* map, const GlqbPagedCache* c, const void* base, int64_t page, int64_t row, int64_t head) {
  const cuuint64_t dims[4] = {(cuuint64_t)c->head_dim, (cuuint64_t)c->kv_heads, (cuuint64_t)c->page_size, (cuuint64_t)c->pages};
  auto bytes = [](int64_t s, bool used) { return (cuuint64_t)(used ? s * 2 : 16); };
  const cuuint64_t strides[3] = {bytes(head, c->kv_heads > 1), bytes(row, true), bytes(page, c->pages > 1)};
  const cuuint32_t box[4] = {64, 1, (cuuint32_t)std::min(c->page_size, PA_PIECE), 1}, ones[4] = {1, 1, 1, 1};
  const EncodeTiled encode = encode_tiled();
  return encode && encode(map, c->dtype == GLQB_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, box, ones,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// heads that share a key head, of as many queries as make 128 rows
bool encode_queries(CUtensorMap* map, const GlqbPagedCache* c, const GlqbPagedAttention* a) {
  const int group = a->heads / c->kv_heads;
  const cuuint64_t dims[3] = {(cuuint64_t)c->head_dim, (cuuint64_t)a->heads, (cuuint64_t)a->tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)(a->heads > 1 ? a->query_head * 2 : 16), (cuuint64_t)(a->tokens > 1 ? a->query_token * 2 : 16)};
  const cuuint32_t box[3] = {64, (cuuint32_t)group, (cuuint32_t)(128 / group)}, ones[3] = {1, 1, 1};
  const EncodeTiled encode = encode_tiled();
  return encode && encode(map, c->dtype == GLQB_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(a->query), dims, strides, box, ones,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A call's tag: 52 bits of the splitmix64 sequence (Steele, Lea and Flood 2014), which starts anywhere.
unsigned long long next_tag() {
  static std::atomic<unsigned long long> state{(unsigned long long)std::chrono::steady_clock::now().time_since_epoch().count() ^ (unsigned long long)reinterpret_cast<uintptr_t>(&state) << 20};
  unsigned long long z = state.fetch_add(0x9E3779B97F4A7C15ull) + 0x9E3779B97F4A7C15ull;
  z = (z ^ z >> 30) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ z >> 27) * 0x94D049BB133111EBull;
  return (z ^ z >> 31) >> 12;
}

// What a call launches and keeps in its workspace, by its sizes alone.
struct PagedForm {
  bool tile;                        // on the tensor cores
  int rows, dp, ctas;
  size_t ml, part_of, bytes;        // where the workspace's second and third part begin, and its size
};
// Rows of a sequence and key head up to which the streaming kernel runs: those of one of its items.  More rows are several items, that read the cache once
// each.  64 sequences of 2048 keys, 8 key heads of 128 values, streaming / on the tensor cores: 8 rows 93 / 109 us, 16 98 / 112, 24 175 / 112, 32 176 / 113,
// 64 337 / 114; one sequence of 16384: 8 rows 21 / 27, 16 29 / 27, 24 29 / 27, 64 41 / 28.
constexpr int PA_STREAM_MOST = 16;
// What beginning an item costs a CTA of either kernel, in its key tiles.  (Of 1, 2, 4 and 6: one token of 4096 keys 11.8, 11.5, 12.1, 13.4 us, of 512 8.7, 9.2, 10.4,
// 11.9; 64 sequences of up to 1024 39.1, 34.1, 33.4, 34.1, of up to 8192 174.6, 173.0, 173.3, 174.8; prompt of 2048 tokens 53.5, 51.5, 52.9, 55.1; of 8192 493, 468, 474, 486.  Heads of 64 values, two
// processes each, which differ by more: 24 sequences of mixed lengths 49, 49, 49, 48; prompt of 2048 tokens 42 and 48, 44 and 51, 45 and 48, 49 and 51.)
constexpr int PA_STREAM_BEGIN = 2, PA_TILE_BEGIN = 2;
PagedForm paged_form(const GlqbPagedCache* c, const GlqbPagedAttention* a, int sms) {
  PagedForm f;
  const int group = a->heads / c->kv_heads;
  f.tile = (long long)std::max(1, a->max_query_len) * group > PA_STREAM_MOST && group <= 128;
  f.rows = f.tile ? PA_TILE_ROWS : PA_STREAM_ROWS;
  f.dp = c->head_dim <= 64 ? 64 : 128;
  f.ctas = f.tile ? sms : 2 * sms;
  f.ml = (size_t)f.ctas * 2 * f.rows * f.dp * sizeof(float);
  f.part_of = f.ml + (size_t)f.ctas * 2 * f.rows * sizeof(float2);
  // (many rows: what the CTAs leave; few: tickets)
  f.bytes = f.part_of + (size_t)f.ctas * (f.tile ? 2 * sizeof(PagedPart) : ST_WARPS * sizeof(unsigned long long));
  return f;
}
int check_attention(const GlqbPagedCache* c, const GlqbPagedAttention* a) {
  const char* what = "paged_attention";
  if (const int rc = check_cache(c, what)) return rc;
  if (!a) return pg_fail(GLQB_E_INVALID, "%s: null argument", what);
  if (a->tokens < 0 || a->sequences < 0 || a->sequences > 1 << 20) return pg_fail(GLQB_E_INVALID, "%s: %lld tokens of %d sequences", what, (long long)a->tokens, a->sequences);
  if (a->heads < 1 || a->heads % c->kv_heads) return pg_fail(GLQB_E_INVALID, "%s: %d query heads over %d key heads", what, a->heads, c->kv_heads);
  if (a->tokens >= 1ll << 30 || a->tokens * a->heads >= 1ll << 30) return pg_fail(GLQB_E_INVALID, "%s: %lld tokens of %d heads are too many for one call", what, (long long)a->tokens, a->heads);
  if (a->page_columns < 0 || (long long)a->page_columns * c->page_size > 1ll << 30) return pg_fail(GLQB_E_INVALID, "%s: %d pages of %d rows per sequence", what, a->page_columns, c->page_size);
  if (!(a->scale > 0.0f) || !std::isfinite(a->scale)) return pg_fail(GLQB_E_INVALID, "%s: the scale is positive", what);
  if (a->window < 0) return pg_fail(GLQB_E_INVALID, "%s: a window of %d keys", what, a->window);
  return GLQB_OK;
}

template <typename T, int DP>
cudaError_t attention_launch(const PagedJob& J, const PagedForm& f, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t stream) {
  using C = StreamShape<DP>;
  constexpr auto K = paged_stream_kernel<T, DP>;
  if (!f.tile) return paged_launch<K>(K, dim3((unsigned)f.ctas), ST_THREADS, C::STAGES * C::STAGE + sizeof(StreamShared) + 1024, stream, J, mk, mv);
  const cudaError_t e = paged_tile_launch(J, __is_same(T, __nv_bfloat16), mq, mk, mv, f.ctas, stream);
  if (e != cudaSuccess) return e;
  constexpr auto CB = paged_combine_kernel<T, DP>;
  return paged_launch<CB>(CB, dim3((unsigned)f.ctas, cb_blocks(DP)), CB_WARPS * 32, 0, stream, J, f.ctas);
}
}  // namespace
}  // namespace glqb

using namespace glqb;
extern "C" {

int glqb_rotary(const GlqbRotary* r, const void* x, int32_t dtype, int64_t x_token, int64_t x_head, void* out, int64_t out_token, int64_t out_head,
                int64_t tokens, int32_t heads, int32_t head_dim, const void* positions, int32_t positions_are_int64, void* stream_) {
  const char* what = "rotary";
  if (!r || !dtype_ok(dtype)) return pg_fail(GLQB_E_INVALID, "%s: dtype", what);
  if (tokens < 0 || heads < 0 || head_dim < 2 || head_dim > ROT_MAX_DIM || heads > 1 << 20) return pg_fail(GLQB_E_INVALID, "%s: %lld tokens of %d heads of %d values (at most %d)", what, (long long)tokens, heads, head_dim, ROT_MAX_DIM);
  if (tokens == 0 || heads == 0) return GLQB_OK;
  if (!x || !out) return pg_fail(GLQB_E_INVALID, "%s: null argument", what);
  if (!lies_on(x, size_of(dtype)) || !lies_on(out, size_of(dtype))) return pg_fail(GLQB_E_INVALID, "%s: values that are not aligned", what);
  if (const int rc = check_rotary(r, head_dim, positions, positions_are_int64, what)) return rc;
  const PagedDevice* d = pg_device();
  if (!d) return pg_fail(GLQB_E_CUDA, "%s: no device", what);
  RotJob J = {};
  J.part[0] = RotPart{(const uint8_t*)x, (uint8_t*)out, x_token, x_head, out_token, out_head, 0, heads, 1, 0};
  J.positions = positions;
  J.positions_wide = positions_are_int64;
  J.turns = (const unsigned long long*)r->turns;
  J.tokens = tokens;
  J.head_dim = head_dim;
  J.pairs = r->pairs;
  J.interleaved = r->interleaved;
  J.scale = r->scale;
  const int sms = d->sms.load(std::memory_order_relaxed);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  if (dtype == GLQB_DT_F16) return rotary_launch<__half, __half>(J, sms, stream, what);
  if (dtype == GLQB_DT_BF16) return rotary_launch<__nv_bfloat16, __nv_bfloat16>(J, sms, stream, what);
  return rotary_launch<float, float>(J, sms, stream, what);
}

int glqb_paged_append(const GlqbPagedCache* c, const GlqbPagedAppend* a, const GlqbRotary* r, void* stream_) {
  const char* what = "paged_append";
  if (const int rc = check_cache(c, what)) return rc;
  if (!a) return pg_fail(GLQB_E_INVALID, "%s: null argument", what);
  if (a->dtype != c->dtype && a->dtype != GLQB_DT_F32) return pg_fail(GLQB_E_INVALID, "%s: keys and values are fp32 or of the cache's type", what);
  if (a->tokens < 0 || a->heads < 0 || a->heads > 1 << 20) return pg_fail(GLQB_E_INVALID, "%s: %lld tokens, %d query heads", what, (long long)a->tokens, a->heads);
  if (a->tokens == 0) return GLQB_OK;
  if (!a->key || !a->value || !a->slots || (a->query && !a->query_out)) return pg_fail(GLQB_E_INVALID, "%s: null argument", what);
  if (a->query && !r) return pg_fail(GLQB_E_INVALID, "%s: queries are here to be rotated", what);
  const size_t size = size_of(a->dtype);
  if (!lies_on(a->key, size) || !lies_on(a->value, size) || !lies_on(a->query, size) || !lies_on(a->query_out, size) || !lies_on(a->slots, a->slots_are_int64 ? 8 : 4))
    return pg_fail(GLQB_E_INVALID, "%s: values that are not aligned", what);
  if (r)
    if (const int rc = check_rotary(r, c->head_dim, a->positions, a->positions_are_int64, what)) return rc;
  if (caches_meet(c)) return pg_fail(GLQB_E_INVALID, "%s: keys and values of the cache share addresses", what);
  const PagedDevice* d = pg_device();
  if (!d) return pg_fail(GLQB_E_CUDA, "%s: no device", what);
  RotJob J = {};
  J.part[0] = RotPart{(const uint8_t*)a->key, (uint8_t*)c->keys, a->key_token, a->key_head, c->key_row, c->key_head, c->key_page, c->kv_heads, r != nullptr, 1};
  J.part[1] = RotPart{(const uint8_t*)a->value, (uint8_t*)c->values, a->value_token, a->value_head, c->value_row, c->value_head, c->value_page, c->kv_heads, 0, 1};
  if (a->query) J.part[2] = RotPart{(const uint8_t*)a->query, (uint8_t*)a->query_out, a->query_token, a->query_head, a->query_out_token, a->query_out_head, 0, a->heads, 1, 0};
  J.slots = a->slots;
  J.slots_wide = a->slots_are_int64;
  J.cache_rows = c->pages * c->page_size;
  while (1 << J.page_log < c->page_size) ++J.page_log;
  J.tokens = a->tokens;
  J.head_dim = c->head_dim;
  if (r) {
    J.positions = a->positions;
    J.positions_wide = a->positions_are_int64;
    J.turns = (const unsigned long long*)r->turns;
    J.pairs = r->pairs;
    J.interleaved = r->interleaved;
    J.scale = r->scale;
  }
  const int sms = d->sms.load(std::memory_order_relaxed);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  if (c->dtype == GLQB_DT_F16) return a->dtype == GLQB_DT_F32 ? rotary_launch<float, __half>(J, sms, stream, what) : rotary_launch<__half, __half>(J, sms, stream, what);
  return a->dtype == GLQB_DT_F32 ? rotary_launch<float, __nv_bfloat16>(J, sms, stream, what) : rotary_launch<__nv_bfloat16, __nv_bfloat16>(J, sms, stream, what);
}

size_t glqb_paged_attention_workspace_bytes(const GlqbPagedCache* c, const GlqbPagedAttention* a) {
  if (check_attention(c, a) || a->tokens == 0) return 0;
  const PagedDevice* d = pg_device();
  return paged_form(c, a, d ? d->sms.load(std::memory_order_relaxed) : 148).bytes;
}

int glqb_paged_attention(const GlqbPagedCache* c, const GlqbPagedAttention* a, void* workspace, size_t workspace_bytes, void* stream_) {
  const char* what = "paged_attention";
  if (const int rc = check_attention(c, a)) return rc;
  if (a->tokens == 0) return GLQB_OK;
  if (!a->query || !a->out || (a->sequences && (!a->lengths || (a->page_columns && !a->page_table)))) return pg_fail(GLQB_E_INVALID, "%s: null argument", what);
  if (!lies_on(a->query, 16) || a->query_token % 8 || a->query_head % 8 || a->query_token < 0 || a->query_head < 0 || a->query_token >= 1ll << 38 || a->query_head >= 1ll << 38)
    return pg_fail(GLQB_E_INVALID, "%s: queries lie on 16 bytes, their strides are multiples of 8 values", what);
  if (!lies_on(a->out, 2) || !lies_on(a->page_table, 4) || !lies_on(a->lengths, a->lengths_are_int64 ? 8 : 4) || !lies_on(a->offsets, a->offsets_are_int64 ? 8 : 4))
    return pg_fail(GLQB_E_INVALID, "%s: values that are not aligned", what);
  if (!lies_on(workspace, 32)) return pg_fail(GLQB_E_INVALID, "%s: the workspace must be 32-byte aligned", what);
  const PagedDevice* d = pg_device();
  if (!d) return pg_fail(GLQB_E_CUDA, "%s: no device", what);
  const PagedForm f = paged_form(c, a, d->sms.load(std::memory_order_relaxed));
  if (workspace_bytes < f.bytes || !workspace) return pg_fail(GLQB_E_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, f.bytes);
  CUtensorMap mk, mv, mq = {};
  if (!encode_cache(&mk, c, c->keys, c->key_page, c->key_row, c->key_head) || !encode_cache(&mv, c, c->values, c->value_page, c->value_row, c->value_head))
    return pg_fail(GLQB_E_CUDA, "%s: cuTensorMapEncodeTiled refused the cache", what);
  if (f.tile && !encode_queries(&mq, c, a)) return pg_fail(GLQB_E_CUDA, "%s: cuTensorMapEncodeTiled refused the queries", what);
  PagedJob J = {};
  J.q = (const uint16_t*)a->query;
  J.out = a->out;
  J.q_token = a->query_token;
  J.q_head = a->query_head;
  J.out_token = a->out_token;
  J.out_head = a->out_head;
  J.lengths = a->lengths;
  J.offsets = a->offsets;
  J.lengths_wide = a->lengths_are_int64;
  J.offsets_wide = a->offsets_are_int64;
  J.pages = a->page_table;
  J.page_stride = a->page_stride;
  J.seqs = a->sequences;
  while (1 << J.page_log < c->page_size) ++J.page_log;
  J.tokens = (int)a->tokens;
  J.heads = a->heads;
  J.kv_heads = c->kv_heads;
  J.group = a->heads / c->kv_heads;
  J.head_dim = c->head_dim;
  J.causal = a->causal;
  J.window = a->window < 1 << 30 ? a->window : 0;        // (no sequence has more keys; so position - window stays within 32 bits)
  J.clear = a->clear_rest;
  J.scale_log2 = a->scale * 1.4426950408889634f;
  J.most_keys = a->page_columns * c->page_size;
  J.begin = f.tile ? PA_TILE_BEGIN : PA_STREAM_BEGIN;
  J.min_units = J.begin + (f.tile ? 2 : 1);
  J.rows = f.tile ? 128 / J.group * J.group * 2 : PA_STREAM_ROWS;
  J.by_group = pa_divisor(J.group);
  J.by_rows = pa_divisor(J.rows);
  J.out_wide = lies_on(a->out, 8) && a->out_token % 4 == 0 && a->out_head % 4 == 0;
  J.out_sectors = lies_on(a->out, 32) && a->out_token % 16 == 0 && a->out_head % 16 == 0;
  J.part = (float*)workspace;
  J.part_ml = (float2*)((uint8_t*)workspace + f.ml);
  J.part_of = (PagedPart*)((uint8_t*)workspace + f.part_of);
  J.tickets = (unsigned long long*)((uint8_t*)workspace + f.part_of);
  J.tag = next_tag();
  J.status = d->status;
  J.gave_up = d->gave_up;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  cudaError_t e;
  if (c->dtype == GLQB_DT_F16) e = f.dp == 64 ? attention_launch<__half, 64>(J, f, mq, mk, mv, stream) : attention_launch<__half, 128>(J, f, mq, mk, mv, stream);
  else e = f.dp == 64 ? attention_launch<__nv_bfloat16, 64>(J, f, mq, mk, mv, stream) : attention_launch<__nv_bfloat16, 128>(J, f, mq, mk, mv, stream);
  return pg_launched(what, e);
}

int glqb_paged_status(int32_t* status_out) {
  int code = 0;
  const int zero = 0;
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&code, g_paged_status, sizeof code);
  if (e == cudaSuccess && code) e = cudaMemcpyToSymbol(g_paged_status, &zero, sizeof zero);
  if (e != cudaSuccess) return pg_fail(GLQB_E_CUDA, "paged_status: %s", cudaGetErrorString(e));
  if (status_out) *status_out = code;
  return code ? pg_fail(GLQB_E_DEVICE, "a bounded wait in attention over a paged cache gave up (status %d): results are invalid", code) : GLQB_OK;
}

}  // extern "C"
