// Attention of many rows over a paged cache, on the tensor cores.
//
// An item is 256 rows (heads of a group that share a key head, times queries) of one sequence, as two tiles of 128, against tiles of 128
// keys.  Scores S = Q K^T go to tensor memory; a thread has a row of them: four warps per tile take their largest, turn them into weights
// P = 2^(scale (S - reference)) in the values' type and put those back over the scores, as the operand from tensor memory of O += P V.  While
// one tile's weights are formed, the tensor cores work for the other.  Tensor memory: 128 columns of scores and 128 of sums per tile, all of it.
//
// Warps 0-3 and 4-7: the tiles' weights, and their results; 8: one thread issues all MMAs; 9: TMA of keys and values (a stage is one tile
// of either), and the list of items; 10 and 11: values of tiles that not every row sees.  Rows of values behind the sequence, or in front
// of its window, may hold anything, and a weight of nothing times NaN is NaN: those rows are set to zero in shared memory.  Rows that only some queries
// see have to stay; where such a tile holds a value that is not finite, its product is left out of the MMAs and formed one row at a time.
//
// What bounds it: of a tile of 128 x 128, the exponentials take 1024 clocks of the special-function units and the two products 1024 of the tensor
// pipe (head_dim 128).
#include "glqb_paged.cuh"

namespace glqb {
namespace {

constexpr int TL_THREADS = 384, TL_ITEMS = 4, TL_CHECKED = 6;
constexpr int TL_MMA = 8, TL_LOAD = 9, TL_CHECK = 10, TL_CHECKERS = 2;
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
  uint64_t full[10], empty[10], item_full[TL_ITEMS], item_empty[TL_ITEMS], q_full[2], s_full[2], p_full[2], o_full[2], checked[TL_CHECKED], drain;
  int odd[TL_CHECKED][TL_CHECKERS];
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

// Is there a key in a tile that one of the rows first .. last (of the sequence's queries * group) does not see?
__device__ __forceinline__ bool ragged(int key0, int all_from, int all_to) { return key0 < all_from || key0 + PA_TILE_KEYS > all_to; }

// An item's rows of queries, as the operand of a tile: 128 rows, columns behind head_dim and rows behind the last zero.  16 lanes take a row.
template <int DP>
__device__ __forceinline__ void load_queries(const PagedJob& J, const PagedItem& it, int tile, int thread, uint4 (&v)[DP / 8]) {
  constexpr int LANES = DP / 8;
  const int col = thread % LANES * 8;
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) {
    const int r = tile * 128 + thread / LANES + n * (128 / LANES), row = it.first + r, i = pa_query(J, row);
    v[n] = make_uint4(0, 0, 0, 0);
    if (r < it.rows && col < J.head_dim)
      v[n] = *reinterpret_cast<const uint4*>(J.q + (long long)(it.row0 + i) * J.q_token + (long long)(it.kv_head * J.group + row - i * J.group) * J.q_head + col);
  }
}
template <int DP>
__device__ __forceinline__ void store_queries(uint8_t* q, int thread, const uint4 (&v)[DP / 8]) {
  constexpr int LANES = DP / 8;
  const int chunk = thread % LANES;
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) {
    const int r = thread / LANES + n * (128 / LANES);
    *reinterpret_cast<uint4*>(q + (chunk >> 3) * (128 * 128) + r * 128 + (((chunk & 7) ^ (r & 7)) << 4)) = v[n];
  }
}

template <typename T, int DP>
__global__ void __launch_bounds__(TL_THREADS, 1)
paged_tile_kernel(const __grid_constant__ PagedJob J, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  using C = TileShape<DP>;
  constexpr int ROWS = PA_TILE_ROWS, KEYS = PA_TILE_KEYS;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* queries = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* ring = queries + 2 * C::Q_TILE;
  TileShared& B = *reinterpret_cast<TileShared*>(ring + C::STAGES * C::STAGE);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) { mbar_init(&B.full[s], 1); mbar_init(&B.empty[s], 1); }
    for (int s = 0; s < TL_ITEMS; ++s) { mbar_init(&B.item_full[s], 1); mbar_init(&B.item_empty[s], 9 + TL_CHECKERS); }
    for (int s = 0; s < 2; ++s) { mbar_init(&B.q_full[s], 4); mbar_init(&B.s_full[s], 1); mbar_init(&B.p_full[s], 4); mbar_init(&B.o_full[s], 1); }
    for (int s = 0; s < TL_CHECKED; ++s) mbar_init(&B.checked[s], TL_CHECKERS);
    mbar_init(&B.drain, 1);
    B.abort = 0;
    fence_mbar_init();
  }
  __syncwarp();
  if (warp == TL_MMA) {
    tmem_alloc(&B.tmem, 512);
    tmem_relinquish();
  }
  if (warp == TL_LOAD && lane < 2) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(lane ? &map_v : &map_k)) : "memory");
  tc_fence_before();
  pdl_wait();
  pdl_trigger();
  pa_start<ROWS, KEYS>(J, B.start);                        // (ends with a block barrier)
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
    const int t = warp >> 2, thread = threadIdx.x & 127, quarter = warp & 3;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16, scores = tmem + lanes + (uint32_t)t * 128u, sums = tmem + lanes + C::SUMS + (uint32_t)t * 128u;
    uint8_t* q = queries + t * C::Q_TILE;
    uint32_t s_phase = 0, o_phase = 0, n_checked = 0;
    const float c = J.scale_log2;
    PagedItem it;
    ok = take(it);
    uint4 qv[DP / 8];
    bool mine = ok && it.more && t * 128 < it.rows;
    if (mine) {
      load_queries<DP>(J, it, t, thread, qv);
      store_queries<DP>(q, thread, qv);
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&B.q_full[t]);
    }
    while (ok && it.more) {
      const PagedSeq seq{it.row0, it.queries, it.keys};
      const int i0 = pa_query(J, it.first), i1 = pa_query(J, it.first + it.rows - 1);
      const int item_from = pa_from(J, seq, i1), item_to = pa_to(J, seq, i0);
      const int r = t * 128 + quarter * 32 + lane, row = it.first + min(r, it.rows - 1), i = pa_query(J, row);
      const int from = pa_from(J, seq, i), to = pa_to(J, seq, i);
      const int last = min(it.rows, t * 128 + 128) - 1;
      const int all_from = pa_from(J, seq, pa_query(J, it.first + last)), all_to = pa_to(J, seq, pa_query(J, it.first + t * 128));
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
          if (ragged(key0, all_from, all_to)) {
            const int lo = from - key0, hi = to - key0;
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (n * 32 + k < lo || n * 32 + k >= hi) s[n][k] = 0xFF800000u;
          }
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int k = 0; k < 32; ++k)
#pragma unroll
            for (int n = 0; n < 4; ++n) top[n] = fmaxf(top[n], __uint_as_float(s[n][k]));
          const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
          const bool grown = (most - m) * c > PA_LAZY;     // (from nothing: infinity; nothing from nothing: not a number, no)
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
          const float less = m == -INFINITY ? 0.0f : m * c;
          float sum[4] = {};
          uint32_t p[64];
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
              const float u = pa_exp2(fmaf(__uint_as_float(s[n][k]), c, -less)), v = pa_exp2(fmaf(__uint_as_float(s[n][k + 1]), c, -less));
              sum[n] += u + v;
              p[n * 16 + k / 2] = pa_pack<T>(u, v);
            }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          tmem_st32(scores, p);
          tmem_st32(scores + 32u, p + 32);
          tmem_st_wait();
          if (check) {
            const uint32_t n = n_checked % TL_CHECKED;
            if (!mbar_wait_warp(&B.checked[n], n_checked / TL_CHECKED & 1u, abort)) { ok = false; break; }
            int odd = 0;
#pragma unroll
            for (int k = 0; k < TL_CHECKERS; ++k) odd |= *(volatile int*)&B.odd[n][k];
            if (odd) {
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
      // the next item's queries, as soon as this one's products are done; then this one's results
      PagedItem then;
      if (!take(then)) { ok = false; break; }
      const bool mine_then = then.more && t * 128 < then.rows;
      if (mine_then) load_queries<DP>(J, then, t, thread, qv);
      if (mine) {
        if (!mbar_wait_warp(&B.o_full[t], o_phase, abort)) { ok = false; break; }
        o_phase ^= 1u;
        tc_fence_after();
      }
      if (mine_then) {
        store_queries<DP>(q, thread, qv);
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.q_full[t]);
      }
      if (mine) {
        const bool there = r < it.rows;
        const float f = it.slot < 0 ? pa_row_factor(J, seq, row, l) : 1.0f;
        const long long at = pa_out_row(J, it.row0, it.kv_head, row), place = (2ll * blockIdx.x + max(it.slot, 0)) * ROWS + r;
        if (it.slot >= 0 && there) J.part_ml[place] = make_float2(m * c, l);
#pragma unroll 1
        for (int n = 0; n < DP / 32; ++n) {
          uint32_t o[32];
          tmem_ld32(sums + n * 32u, o);
          tmem_ld_wait();
          if (there) {
#pragma unroll
            for (int k = 0; k < 32; k += 4) {
              const float4 v = make_float4(__uint_as_float(o[k]) * f, __uint_as_float(o[k + 1]) * f, __uint_as_float(o[k + 2]) * f, __uint_as_float(o[k + 3]) * f);
              const int col = n * 32 + k;
              if (it.slot >= 0) *reinterpret_cast<float4*>(J.part + place * DP + col) = v;
              else if (col < J.head_dim) pa_store4<T>(J, at, col, v);
            }
          }
          __syncwarp();
        }
        tc_fence_before();
      }
      it = then;
      mine = mine_then;
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
        const PagedSeq seq{it.row0, it.queries, it.keys};
        const int item_from = pa_from(J, seq, pa_query(J, it.first + it.rows - 1)), item_to = pa_to(J, seq, pa_query(J, it.first));
        const int tiles = it.rows > 128 ? 2 : 1;
        ok = mbar_wait_warp(&B.full[stage], phase, abort);
        for (int t = 0; t < tiles && ok; ++t) {
          ok = mbar_wait_warp(&B.q_full[t], q_phase[t], abort);
          if (!ok) break;
          q_phase[t] ^= 1u;
          tc_fence_after();
          scores_of(t, stage);
          if (one) umma_commit(&B.s_full[t]);
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
#pragma unroll
            for (int k = 0; k < TL_CHECKERS; ++k) odd |= *(volatile int*)&B.odd[n][k];
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
            if (one) umma_commit(more ? &B.s_full[t] : &B.o_full[t]);
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
      PagedWalk<ROWS, KEYS> walk(J, B.start);
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
    } else {
      // values of tiles that not every row sees
      const int thread = (warp - TL_CHECK) * 32 + lane;
      uint32_t n_checked = 0;
      PagedItem it;
      for (;;) {
        ok = take(it);
        if (!ok || !it.more) break;
        const PagedSeq seq{it.row0, it.queries, it.keys};
        const int i0 = pa_query(J, it.first), i1 = pa_query(J, it.first + it.rows - 1);
        const int item_from = pa_from(J, seq, i1), item_to = pa_to(J, seq, i0), any_from = pa_from(J, seq, i0), any_to = pa_to(J, seq, i1);
        for (int tile = it.lo; tile < it.hi; ++tile) {
          advance();                                       // (the keys')
          if (ragged(tile * KEYS, item_from, item_to)) {
            const uint32_t n = n_checked % TL_CHECKED;
            if (!mbar_wait_warp(&B.full[stage], phase, abort)) { ok = false; break; }
            bool odd = false;
#pragma unroll 4
            for (int k = thread; k < KEYS * (DP / 8); k += TL_CHECKERS * 32) {
              const int key = tile * KEYS + k / (DP / 8), chunk = k % (DP / 8);
              uint4* p = reinterpret_cast<uint4*>(ring + stage * C::STAGE + (chunk >> 3) * C::HALF + (k / (DP / 8)) * 128 + ((chunk & 7) << 4));
              if (key < any_from || key >= any_to) {
                *p = make_uint4(0, 0, 0, 0);
              } else {
                const uint4 v = *p;
                odd = odd || pa_not_finite<T>(v.x) || pa_not_finite<T>(v.y) || pa_not_finite<T>(v.z) || pa_not_finite<T>(v.w);
              }
            }
            odd = __any_sync(0xFFFFFFFFu, odd);
            fence_async_smem();
            if (lane == 0) *(volatile int*)&B.odd[n][warp - TL_CHECK] = odd;
            __syncwarp();
            if (lane == 0) mbar_arrive(&B.checked[n]);
            ++n_checked;
          }
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
cudaError_t run(const PagedJob& J, const CUtensorMap& mk, const CUtensorMap& mv, int ctas, cudaStream_t stream) {
  using C = TileShape<DP>;
  constexpr size_t SMEM = 1024 + 2 * C::Q_TILE + C::STAGES * C::STAGE + sizeof(TileShared);
  static_assert(SMEM <= 227 * 1024, "");
  static_assert(SMEM > 114 * 1024, "two CTAs on an SM would wait for each other's tensor memory");
  constexpr auto K = paged_tile_kernel<T, DP>;
  return paged_launch<K>(K, dim3((unsigned)ctas), TL_THREADS, SMEM, stream, J, mk, mv);
}
}  // namespace

cudaError_t paged_tile_launch(const PagedJob& J, bool bf16, const CUtensorMap& mk, const CUtensorMap& mv, int ctas, cudaStream_t stream) {
  if (J.head_dim <= 64) return bf16 ? run<__nv_bfloat16, 64>(J, mk, mv, ctas, stream) : run<__half, 64>(J, mk, mv, ctas, stream);
  return bf16 ? run<__nv_bfloat16, 128>(J, mk, mv, ctas, stream) : run<__half, 128>(J, mk, mv, ctas, stream);
}
}  // namespace glqb
