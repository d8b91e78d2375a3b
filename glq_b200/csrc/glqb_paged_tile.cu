// Attention of many rows over a paged cache, on the tensor cores.
//
// An item is up to 256 rows (heads of a group that share a key head, times queries) of one sequence, as two tiles of the whole queries that 128
// rows hold, against tiles of 128 keys.  Scores S = Q K^T go to tensor memory; a thread has a row of them: four warps per tile take their largest, turn them into weights
// P = 2^(scale (S - reference)) in the values' type and put those back over the scores, as the operand from tensor memory of O += P V.  While
// one tile's weights are formed, the tensor cores work for the other.  Tensor memory: 128 columns of scores and 128 of sums per tile, all of it.
//
// Warps 0-3 and 4-7: the tiles' weights, and their results; 8: one thread issues all MMAs; 9: TMA of keys and values (a stage is one tile
// of either), and the list of items; 10: values of tiles that not every row sees; 11: TMA of queries.  Rows of values behind the sequence, or in front
// of its window, may hold anything, and a weight of nothing times NaN is NaN: those rows are set to zero in shared memory.  Rows that only some queries
// see have to stay; where such a tile holds a value that is not finite, its product is left out of the MMAs and formed one row at a time.
//
// What bounds it: the exponentials of 256 rows x 128 keys take 2048 clocks of the special-function units, 16 a clock, and the two products 2048 of the tensor pipe (head_dim
// 128).  Either would be enough for 2048 from tile to tile; it takes 3300, as each half of the rows goes its way scores, weights, product, scores, and
// what its warps do beside the exponentials has to hide behind the other half.  32 heads over 8, bf16: a prompt of 8192 tokens 467 us
// (1178 TFLOP/s), 512 tokens behind 16384 keys 125 us (1120), with the parts joined.  Two halves rather than one tile of 128 rows: then neither unit has work while the other does.
// Five stages of 32 KB for keys and values (head_dim 128) are what 64 KB of queries leave of shared memory.
#include "glqb_paged.cuh"

namespace glqb {
namespace {

constexpr int TL_THREADS = 384, TL_ITEMS = 4, TL_CHECKED = 6;
constexpr int TL_MMA = 8, TL_LOAD = 9, TL_QUERY = 11;      // (10 checks values)
template <int DP>
struct TileShape {
  static constexpr int HALF = PA_TILE_KEYS * 128, STAGE = HALF * (DP / 64), Q_TILE = 128 * DP * 2, STAGES = DP == 64 ? 10 : 5;
  static constexpr uint32_t SUMS = 256;                    // first column of the sums; scores from 0 on
  // Values are checked as soon as they are there, ahead of those whose products are not done by as many tiles as the ring still holds.  A wait
  // by parity takes a barrier that is two phases on for one that is not there yet: so no barrier may come round within that distance.
  static_assert(TL_CHECKED > (STAGES - 1) / 2, "");
};
struct __align__(16) TileShared {
  PagedStart start;
  PagedItem item[TL_ITEMS];
  uint64_t full[10], empty[10], item_full[TL_ITEMS], item_empty[TL_ITEMS], q_full[2], q_empty[2], s_full[2], p_full[2], o_full[2], checked[TL_CHECKED], drain;
  int odd[TL_CHECKED];
  uint32_t tmem;
  int abort;
};

__device__ __forceinline__ void umma_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
               "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld4(uint32_t taddr, uint32_t (&r)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(taddr) : "memory");
}
// B from rows of keys with the values (N) one behind the other: atoms of 64 values x 8 keys under the 128-byte swizzle, eights of keys 1024 bytes
// apart, 64 values HALF bytes apart
__device__ __forceinline__ uint64_t values_desc(uint32_t smem_addr) {
  return (uint64_t)((smem_addr >> 4) & 0x3FFF) | (uint64_t)(PA_TILE_KEYS * 128 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// fp32 sums, A K-major, 128 rows; `turned`: B is N-major
__device__ __forceinline__ uint32_t tile_idesc(int bf16, int cols, int turned) {
  return (1u << 4) | (uint32_t)bf16 << 7 | (uint32_t)bf16 << 10 | (uint32_t)turned << 16 | (uint32_t)(cols >> 3) << 17 | (128u >> 4) << 24;
}
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Is there a key in the tile from key0 on that is not one of all_from .. all_to - 1, those that all rows see?
__device__ __forceinline__ bool ragged(int key0, int all_from, int all_to) { return key0 < all_from || key0 + PA_TILE_KEYS > all_to; }

// `rows` rows x 64 values of queries: coordinates (value, head, token)
__device__ __forceinline__ void load_queries(void* dst, const CUtensorMap* map, int x, int head, int token, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)), "l"(map),
               "r"(x), "r"(head), "r"(token), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
// the n lowest bits
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }
// the largest of three; not a number if one of them is not
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
struct f2 { uint64_t v; };
__device__ __forceinline__ f2 f2_of(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_to(f2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ f2 f2_fma(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ f2 f2_add(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

// Weights of 32 scores: to tensor memory in the values' type, their sum to `sum`.
template <typename T>
__device__ __forceinline__ void weights(const uint32_t (&s)[32], f2 c, f2 less, f2 (&sum)[2], uint32_t taddr) {
  uint32_t p[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const f2 x = f2_fma(f2_of(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1])), c, less);
    float u, v;
    f2_to(x, u, v);
    u = pa_exp2(u);
    v = pa_exp2(v);
    sum[k & 1] = f2_add(sum[k & 1], f2_of(u, v));
    p[k] = pa_pack<T>(u, v);
  }
  tmem_st16(taddr, p);
}

template <typename T, int DP>
__global__ void __launch_bounds__(TL_THREADS, 1)
paged_tile_kernel(const __grid_constant__ PagedJob J, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  using C = TileShape<DP>;
  constexpr int KEYS = PA_TILE_KEYS;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* queries = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* ring = queries + 2 * C::Q_TILE;
  TileShared& B = *reinterpret_cast<TileShared*>(ring + C::STAGES * C::STAGE);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) { mbar_init(&B.full[s], 1); mbar_init(&B.empty[s], 2); }
    for (int s = 0; s < TL_ITEMS; ++s) { mbar_init(&B.item_full[s], 1); mbar_init(&B.item_empty[s], 11); }
    for (int s = 0; s < 2; ++s) { mbar_init(&B.q_full[s], 1); mbar_init(&B.q_empty[s], 1); mbar_init(&B.s_full[s], 1); mbar_init(&B.p_full[s], 4); mbar_init(&B.o_full[s], 1); }
    for (int s = 0; s < TL_CHECKED; ++s) mbar_init(&B.checked[s], 1);
    mbar_init(&B.drain, 1);
    B.abort = 0;
    fence_mbar_init();
  }
  __syncwarp();
  if (warp == TL_MMA) {
    tmem_alloc(&B.tmem, 512);
    tmem_relinquish();
  }
  if (warp == TL_LOAD && lane < 3)
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(lane == 2 ? &map_q : lane ? &map_v : &map_k)) : "memory");
  tc_fence_before();
  pdl_wait();
  pdl_trigger();
  pa_start<KEYS>(J, B.start);                        // (ends with a block barrier)
  tc_fence_after();
  const uint32_t tmem = B.tmem;
  volatile int* abort = &B.abort;
  bool ok = true;
  uint32_t filled = 0;
  // the next item, for the warps that do not make the list
  int is = 0;
  uint32_t ip = 0;
  auto take = [&](PagedItem& it) {
    if (!mbar_wait_warp(&B.item_full[is], ip, abort)) return false;
    it = B.item[is];
    __syncwarp();
    if (lane == 0) mbar_arrive(&B.item_empty[is]);
    if (++is == TL_ITEMS) { is = 0; ip ^= 1u; }
    return true;
  };
  uint32_t stage = 0, phase = 0;
  auto advance = [&] { if (++stage == C::STAGES) { stage = 0; phase ^= 1u; } };

  if (warp < TL_MMA) {
    more_registers<200>();
    const int t = warp >> 2, quarter = warp & 3;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16, scores = tmem + lanes + (uint32_t)t * 128u, sums = tmem + lanes + C::SUMS + (uint32_t)t * 128u;
    uint32_t s_phase = 0, o_phase = 0, n_checked = 0;
    const float c = J.scale_log2;
    const int tile_rows = J.rows / 2;
    PagedItem it;
    ok = take(it);
    while (ok && it.more) {
      const PagedSeq seq{it.row0, it.queries, it.keys};
      const int item_from = it.all_from, item_to = it.all_to;
      // this thread's row (one behind the tile's last is computed as if it were that one, and not stored)
      const bool mine = t * tile_rows < it.rows;
      const int r = quarter * 32 + lane, row0 = it.first + (mine ? t * tile_rows : 0), rows = mine ? min(tile_rows, it.rows - t * tile_rows) : 1;
      const int row = row0 + min(r, rows - 1), i = pa_query(J, row);
      const int from = pa_from(J, seq, i), to = pa_to(J, seq, i);
      const int all_from = pa_from(J, seq, pa_query(J, row0 + rows - 1)), all_to = pa_to(J, seq, pa_query(J, row0));
      float m = -INFINITY, l = 0.0f;                       // (m: of scores without their scale)
      for (int tile = it.lo; tile < it.hi; ++tile) {
        const int key0 = tile * KEYS;
        const bool check = ragged(key0, item_from, item_to);
        if (mine) {
          if (!mbar_wait_warp(&B.s_full[t], s_phase, abort)) { ok = false; break; }
          s_phase ^= 1u;
          tc_fence_after();
          uint32_t s[4][32];
#pragma unroll
          for (int n = 0; n < 4; ++n) tmem_ld32(scores + n * 32u, s[n]);
          tmem_ld_wait();
          const bool cut = ragged(key0, all_from, all_to);
          if (cut) {
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              // (a bit per key)
              const uint32_t seen = below(to - key0 - n * 32) & ~below(from - key0 - n * 32);
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (!(seen >> k & 1u)) s[n][k] = 0xFF800000u;
            }
          }
          float top[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            top[n] = __uint_as_float(s[n][0]);
#pragma unroll
            for (int k = 1; k < 31; k += 2) top[n] = max3(top[n], __uint_as_float(s[n][k]), __uint_as_float(s[n][k + 1]));
          }
          // (not a number if a score is none: then the reference stays, and that score's weight says so)
          const float most = max3(max3(top[0], top[1], __uint_as_float(s[0][31])), max3(top[2], top[3], __uint_as_float(s[1][31])), max3(__uint_as_float(s[2][31]), __uint_as_float(s[3][31]), top[0]));
          // (from nothing: infinity; nothing from nothing: not a number, no.  What a row without a query holds decides nothing for its warp's others.)
          const bool grown = r < rows && (most - m) * c > PA_LAZY;
          if (__any_sync(0xFFFFFFFFu, grown)) {
            const float now = fmaxf(m, most), f = now == -INFINITY ? 1.0f : pa_exp2((m - now) * c);
            m = now;
            l *= f;
            if (tile > it.lo) {
              // the product before this one is complete: the scores came behind it
#pragma unroll 1
              for (int n = 0; n < DP / 32; ++n) {
                uint32_t o[32];
                tmem_ld32(sums + n * 32u, o);
                tmem_ld_wait();
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                tmem_st32(sums + n * 32u, o);
              }
            }
          }
          const float less = m == -INFINITY ? 0.0f : m * c - pa_up<T>();
          const f2 c2 = f2_of(c, c), less2 = f2_of(-less, -less);
          f2 sum[2] = {f2_of(l, 0.0f), f2_of(0.0f, 0.0f)};
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            weights<T>(s[n], c2, less2, sum, scores + n * 16u);
          }
          float part[4];
          f2_to(sum[0], part[0], part[1]);
          f2_to(sum[1], part[2], part[3]);
          l = (part[0] + part[1]) + (part[2] + part[3]);
          tmem_st_wait();
          if (check) {
            const uint32_t n = n_checked % TL_CHECKED;
            if (!mbar_wait_warp(&B.checked[n], n_checked / TL_CHECKED & 1u, abort)) { ok = false; break; }
            if (*(volatile int*)&B.odd[n]) {
              // a value that is not finite among those that only some rows see: this row's keys one at a time.  (The stage of the values: that
              // behind the keys', two stages per tile.)
              const uint32_t vs = (stage + 1u) % C::STAGES, base = smem_u32(ring) + vs * C::STAGE;
#pragma unroll 1
              for (int n32 = 0; n32 < DP / 32; ++n32) {
                uint32_t o[32];
                if (tile > it.lo) {
                  tmem_ld32(sums + n32 * 32u, o);
                  tmem_ld_wait();
                } else {
#pragma unroll
                  for (int k = 0; k < 32; ++k) o[k] = 0u;
                }
#pragma unroll 1
                for (int kb = 0; kb < KEYS; kb += 8) {
                  uint32_t w[4];
                  tmem_ld4(scores + kb / 2, w);
                  tmem_ld_wait();
#pragma unroll
                  for (int k = 0; k < 8; ++k) {
                    const int key = kb + k;
                    const float2 two = pa_unpack<T>(w[k / 2]);
                    const float weight = k & 1 ? two.y : two.x;
                    if (key0 + key >= from && key0 + key < to) {
#pragma unroll
                      for (int e = 0; e < 4; ++e) {
                        uint32_t x[4];
                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) :
                                     "r"(base + (n32 >> 1) * C::HALF + key * 128 + ((((n32 & 1) * 4 + e) ^ (key & 7)) << 4)) : "memory");
#pragma unroll
                        for (int f = 0; f < 4; ++f) {
                          const float2 v = pa_unpack<T>(x[f]);
                          o[e * 8 + 2 * f] = __float_as_uint(fmaf(weight, v.x, __uint_as_float(o[e * 8 + 2 * f])));
                          o[e * 8 + 2 * f + 1] = __float_as_uint(fmaf(weight, v.y, __uint_as_float(o[e * 8 + 2 * f + 1])));
                        }
                      }
                    }
                  }
                  __syncwarp();
                }
                tmem_st32(sums + n32 * 32u, o);
              }
              tmem_st_wait();
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&B.p_full[t]);
        }
        if (check) ++n_checked;
        advance();
        advance();
      }
      if (!ok) break;
      if (mine) {
        if (!mbar_wait_warp(&B.o_full[t], o_phase, abort)) { ok = false; break; }
        o_phase ^= 1u;
        tc_fence_after();
        // A thread has a row: 32 bytes of it at once are whole sectors.  (8 bytes at once took 12,000 clocks per item.)
        const bool there = r < rows;
        const float f = it.slot < 0 ? pa_row_factor(J, seq, row, l) : 1.0f;
        const long long at = pa_out_row(J, it.row0, it.kv_head, row);
        if (it.slot >= 0 && there) J.part_ml[(2ll * blockIdx.x + it.slot) * PA_TILE_ROWS + t * 128 + r] = make_float2(m * c, l);
        uint32_t o[DP / 32][32];
#pragma unroll
        for (int n = 0; n < DP / 32; ++n) tmem_ld32(sums + n * 32u, o[n]);
        tmem_ld_wait();
        if (there && it.slot >= 0) {
#pragma unroll
          for (int n = 0; n < DP / 32; ++n)
#pragma unroll
            for (int k = 0; k < 32; k += 8) store8(J.part + pa_part_at<DP>(2 * blockIdx.x + it.slot, t * 128 + r, n * 4 + k / 8), o[n] + k);
        } else if (there) {
#pragma unroll
          for (int n = 0; n < DP / 32; ++n) {
            if (J.out_sectors && n * 32 + 32 <= J.head_dim) {
              uint32_t y[16];
#pragma unroll
              for (int k = 0; k < 16; ++k) y[k] = pa_pack<T>(__uint_as_float(o[n][2 * k]) * f, __uint_as_float(o[n][2 * k + 1]) * f);
              store8(reinterpret_cast<uint16_t*>(J.out) + at + n * 32, y);
              store8(reinterpret_cast<uint16_t*>(J.out) + at + n * 32 + 16, y + 8);
            } else {
#pragma unroll
              for (int k = 0; k < 32; k += 4)
                if (n * 32 + k < J.head_dim)
                  pa_store4<T>(J, at, n * 32 + k, make_float4(__uint_as_float(o[n][k]) * f, __uint_as_float(o[n][k + 1]) * f, __uint_as_float(o[n][k + 2]) * f, __uint_as_float(o[n][k + 3]) * f));
            }
          }
        }
        __syncwarp();
        tc_fence_before();
      }
      ok = take(it);
    }
    if (!ok && lane == 0) { *abort = 1; atomicCAS(J.status, 0, (int)ST_GAVE_UP_EPILOGUE); }
  } else {
    fewer_registers<104>();
    if (warp == TL_MMA) {
      const uint32_t id_s = tile_idesc(__is_same(T, __nv_bfloat16), KEYS, 0), id_o = tile_idesc(__is_same(T, __nv_bfloat16), DP, 1);
      uint32_t q_phase[2] = {0, 0}, p_phase[2] = {0, 0}, n_checked = 0;
      const bool one = elect_one();
      // waits are the whole warp's, instructions one lane's
      auto scores_of = [&](int t, uint32_t s) {
        if (one) {
          const uint64_t a = umma_desc_sw128(smem_u32(queries) + t * C::Q_TILE), b = umma_desc_sw128(smem_u32(ring) + s * C::STAGE);
#pragma unroll
          for (int k = 0; k < DP / 16; ++k)
            umma_f16(tmem + (uint32_t)t * 128u, a + (uint64_t)(k / 4 * (128 * 128 >> 4) + k % 4 * 2), b + (uint64_t)(k / 4 * (C::HALF >> 4) + k % 4 * 2), id_s, k > 0);
        }
      };
      PagedItem it;
      for (;;) {
        ok = take(it);
        if (!ok || !it.more) break;
        const int item_from = it.all_from, item_to = it.all_to;
        const int tiles = it.rows > J.rows / 2 ? 2 : 1;
        ok = mbar_wait_warp(&B.full[stage], phase, abort);
        for (int t = 0; t < tiles && ok; ++t) {
          ok = mbar_wait_warp(&B.q_full[t], q_phase[t], abort);
          if (!ok) break;
          q_phase[t] ^= 1u;
          tc_fence_after();
          scores_of(t, stage);
          if (one) {
            umma_commit(&B.s_full[t]);
            if (it.lo + 1 == it.hi) umma_commit(&B.q_empty[t]);
          }
        }
        if (!ok) break;
        if (one) umma_commit(&B.empty[stage]);
        advance();
        for (int tile = it.lo; tile < it.hi && ok; ++tile) {
          const uint32_t vs = stage;
          const bool more = tile + 1 < it.hi;
          ok = mbar_wait_warp(&B.full[vs], phase, abort);
          if (!ok) break;
          advance();
          const uint32_t ks = stage;
          if (more) {
            ok = mbar_wait_warp(&B.full[ks], phase, abort);
            if (!ok) break;
            advance();
          }
          int odd = 0;
          if (ragged(tile * KEYS, item_from, item_to)) {
            const uint32_t n = n_checked % TL_CHECKED;
            ok = mbar_wait_warp(&B.checked[n], n_checked / TL_CHECKED & 1u, abort);
            if (!ok) break;
            ++n_checked;
            odd = *(volatile int*)&B.odd[n];
          }
          for (int t = 0; t < tiles; ++t) {
            ok = mbar_wait_warp(&B.p_full[t], p_phase[t], abort);
            if (!ok) break;
            p_phase[t] ^= 1u;
            tc_fence_after();
            if (one && !odd) {
              const uint64_t b = values_desc(smem_u32(ring) + vs * C::STAGE);
#pragma unroll
              for (int k = 0; k < KEYS / 16; ++k)
                umma_ta(tmem + C::SUMS + (uint32_t)t * 128u, tmem + (uint32_t)(t * 128 + k * 8), b + (uint64_t)(k * (2048 >> 4)), id_o, tile > it.lo || k > 0);
            }
            // (one thread's products run in the order they are issued in: the weights are read before new scores take their place)
            if (more) scores_of(t, ks);
            if (one) {
              umma_commit(more ? &B.s_full[t] : &B.o_full[t]);
              if (more && tile + 2 == it.hi) umma_commit(&B.q_empty[t]);
            }
          }
          if (!ok) break;
          if (one) {
            umma_commit(&B.empty[vs]);
            if (more) umma_commit(&B.empty[ks]);
          }
        }
        if (!ok) break;
      }
      if (!ok && lane == 0) { *abort = 1; atomicCAS(J.status, 0, (int)ST_GAVE_UP_MMA); }
      __syncwarp();
      if (!ok) {
        // what was issued is done before tensor memory is given back
        if (one) umma_commit(&B.drain);
        mbar_wait_warp(&B.drain, 0);
      }
    } else if (warp == TL_LOAD) {
      PagedWalk<KEYS, false> walk(J, B.start);
      const int piece = min(1 << J.page_log, PA_PIECE), pieces = KEYS / piece, page_mask = (1 << J.page_log) - 1;
      phase = 1;
      ip = 1;
      for (;;) {
        const PagedItem it = walk.next(J);
        ok = mbar_wait_warp(&B.item_empty[is], ip, abort);
        if (!ok) break;
        if (lane == 0) { B.item[is] = it; mbar_arrive(&B.item_full[is]); }
        if (!it.more) break;
        if (++is == TL_ITEMS) { is = 0; ip ^= 1u; }
        const int* table = J.pages + (long long)it.seq * J.page_stride;
        for (int tile = it.lo; tile < it.hi && ok; ++tile) {
          const int left = it.keys - tile * KEYS, here = max(0, min(pieces, (left + piece - 1) / piece));       // pieces that hold keys
          const int row = (tile * KEYS + lane * piece) & page_mask;
          int page = 0;
          if (lane < here) page = table[(tile * KEYS + lane * piece) >> J.page_log];
#pragma unroll
          for (int kind = 0; kind < 2; ++kind) {
            if (!mbar_wait_warp(&B.empty[stage], phase, abort)) { ok = false; break; }
            if (lane == 0) mbar_expect_tx(&B.full[stage], (uint32_t)(here * piece) * (DP * 2));
            __syncwarp();
            if (lane < here) {
#pragma unroll
              for (int h = 0; h < DP / 64; ++h)
                pa_load(ring + stage * C::STAGE + h * C::HALF + lane * piece * 128, kind ? &map_v : &map_k, h * 64, it.kv_head, row, page, &B.full[stage]);
            }
            __syncwarp();
            ++filled;
            advance();
          }
        }
        if (!ok) break;
      }
      if (lane == 0) {
        if (!ok) { *abort = 1; atomicCAS(J.status, 0, (int)ST_GAVE_UP_LOADER); }
        pa_publish(J, walk.part);
      }
      // copies in flight land before the block ends
      if (!ok)
        for (uint32_t n = 1; n <= min(filled, (uint32_t)C::STAGES); ++n) mbar_wait(&B.full[(filled - n) % C::STAGES], (filled - n) / C::STAGES & 1u);
    } else if (warp == TL_QUERY) {
      uint32_t e_phase[2] = {1, 1}, issued[2] = {0, 0};
      const int tile_rows = J.rows / 2;
      PagedItem it;
      for (;;) {
        ok = take(it);
        if (!ok || !it.more) break;
        for (int t = 0; t < 2 && t * tile_rows < it.rows; ++t) {
          if (!mbar_wait_warp(&B.q_empty[t], e_phase[t], abort)) { ok = false; break; }
          e_phase[t] ^= 1u;
          if (lane == 0) {
            // (rows behind the sequence's last query are another's, or zeros behind the last token: they are computed and not stored)
            mbar_expect_tx(&B.q_full[t], (uint32_t)tile_rows * DP * 2);
#pragma unroll
            for (int h = 0; h < DP / 64; ++h)
              load_queries(queries + t * C::Q_TILE + h * (128 * 128), &map_q, h * 64, it.kv_head * J.group, it.row0 + pa_query(J, it.first + t * tile_rows), &B.q_full[t]);
          }
          __syncwarp();
          ++issued[t];
        }
        if (!ok) break;
      }
      if (!ok) {
        if (lane == 0) { *abort = 1; atomicCAS(J.status, 0, (int)ST_GAVE_UP_LOADER); }
        for (int t = 0; t < 2; ++t)
          if (issued[t]) mbar_wait(&B.q_full[t], (issued[t] - 1) & 1u);
      }
    } else {
      // values of tiles that not every row sees
      uint32_t n_checked = 0;
      PagedItem it;
      for (;;) {
        ok = take(it);
        if (!ok || !it.more) break;
        const int item_from = it.all_from, item_to = it.all_to, any_from = it.any_from, any_to = it.any_to;
        for (int tile = it.lo; tile < it.hi; ++tile) {
          // Every stage is waited for and given back, also those with nothing to look at: a wait by parity takes a barrier that is two phases
          // behind for ready, so a warp may not be ahead of the ring, nor the ring ahead of it.
          if (!mbar_wait_warp(&B.full[stage], phase, abort)) { ok = false; break; }
          if (lane == 0) mbar_arrive(&B.empty[stage]);
          advance();
          if (!mbar_wait_warp(&B.full[stage], phase, abort)) { ok = false; break; }
          if (ragged(tile * KEYS, item_from, item_to)) {
            const uint32_t n = n_checked % TL_CHECKED;
            // (rows of 128 bytes, per 64 values; their 16-byte pieces lie somewhere within them.  Eight loads at once, and no branch.)
            uint32_t largest = 0u;
            const int first = min(KEYS, max(0, any_from - tile * KEYS)), last = max(first, min(KEYS, any_to - tile * KEYS));
#pragma unroll 1
            for (int h = 0; h < DP / 64; ++h) {
              uint4* values = reinterpret_cast<uint4*>(ring + stage * C::STAGE + h * C::HALF);
              for (int k = lane; k < first * 8; k += 32) values[k] = make_uint4(0, 0, 0, 0);
              for (int k = last * 8 + lane; k < KEYS * 8; k += 32) values[k] = make_uint4(0, 0, 0, 0);
#pragma unroll 1
              for (int k0 = first * 8; k0 < last * 8; k0 += 8 * 32) {
                uint4 v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = values[min(k0 + k * 32 + lane, last * 8 - 1)];
#pragma unroll
                for (int k = 0; k < 8; ++k)
                  largest = __vmaxu2(largest, __vmaxu2(__vmaxu2(v[k].x & 0x7FFF7FFFu, v[k].y & 0x7FFF7FFFu), __vmaxu2(v[k].z & 0x7FFF7FFFu, v[k].w & 0x7FFF7FFFu)));
              }
            }
            const bool odd = __any_sync(0xFFFFFFFFu, pa_not_finite<T>(largest));
            fence_async_smem();
            if (lane == 0) *(volatile int*)&B.odd[n] = odd;
            __syncwarp();
            if (lane == 0) mbar_arrive(&B.checked[n]);
            ++n_checked;
          }
          if (lane == 0) mbar_arrive(&B.empty[stage]);
          advance();
        }
        if (!ok) break;
      }
      if (!ok && lane == 0) { *abort = 1; atomicCAS(J.status, 0, (int)ST_GAVE_UP_PRODUCER); }
    }
  }
  // ---- every thread arrives here, also after a wait gave up
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == TL_MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int DP>
cudaError_t run(const PagedJob& J, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, int ctas, cudaStream_t stream) {
  using C = TileShape<DP>;
  constexpr size_t SMEM = 1024 + 2 * C::Q_TILE + C::STAGES * C::STAGE + sizeof(TileShared);
  static_assert(SMEM <= 227 * 1024, "");
  static_assert(SMEM > 114 * 1024, "two CTAs on an SM would wait for each other's tensor memory");
  constexpr auto K = paged_tile_kernel<T, DP>;
  return paged_launch<K>(K, dim3((unsigned)ctas), TL_THREADS, SMEM, stream, J, mq, mk, mv);
}
}  // namespace

cudaError_t paged_tile_launch(const PagedJob& J, bool bf16, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, int ctas, cudaStream_t stream) {
  if (J.head_dim <= 64) return bf16 ? run<__nv_bfloat16, 64>(J, mq, mk, mv, ctas, stream) : run<__half, 64>(J, mq, mk, mv, ctas, stream);
  return bf16 ? run<__nv_bfloat16, 128>(J, mq, mk, mv, ctas, stream) : run<__half, 128>(J, mq, mk, mv, ctas, stream);
}
}  // namespace glqb
