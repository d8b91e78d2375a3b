// Attention over a paged cache: the job, how its work is shared out, and what its kernels have in common.
#pragma once
#include "glqb_internal.h"
#include "glqb_ptx.cuh"
#include "glqb_launch.h"
#include <atomic>
#include <cuda.h>

namespace glqb {

constexpr int PA_PIECE = 64;         // most rows of a page that one copy brings
constexpr int PA_STREAM_ROWS = 16, PA_STREAM_KEYS = 64;      // rows of an item, and keys of a tile: few rows,
constexpr int PA_TILE_ROWS = 256, PA_TILE_KEYS = 128;        // and many (at most: whole queries)
constexpr float PA_LAZY = 8.0f;                              // a row's weights are relative to a score that its largest exceeds by no more

// Division of 0 .. 2^31 - 1 by one number: q = n * mul >> shift, mul = ceil(2^(31 + l) / d), l = ceil(log2 d) (Granlund and Montgomery 1994).
struct PagedDivisor {
  uint32_t mul;
  int shift;
};
inline PagedDivisor pa_divisor(int d) {
  int l = 0;
  while ((1ll << l) < d) ++l;
  return PagedDivisor{(uint32_t)(((1ull << (31 + l)) + d - 1) / d), 31 + l};
}

struct PagedJob {
  const uint16_t* q;
  void* out;
  long long q_token, q_head, out_token, out_head;
  const void *lengths, *offsets;
  const int* pages;
  long long page_stride;
  int lengths_wide, offsets_wide, seqs, page_log, tokens, heads, kv_heads, group, head_dim, causal, window, clear;
  float scale_log2;                  // scale * log2(e): weights are powers of two
  int most_keys;                     // columns * page size
  int min_units;                     // units of a share where the grid has more CTAs than there is work for (about: shares are equal)
  int rows;                          // of an item
  PagedDivisor by_group, by_rows;
  int begin;                         // what beginning an item costs, in key tiles
  bool out_wide, out_sectors;        // rows of out lie on 8, 32 bytes
  float* part;                       // workspace: sums of items that several CTAs share, [CTA][2][rows][padded head_dim]
  float2* part_ml;                   // their largest exponent and sum, [CTA][2][rows]
  struct PagedPart* part_of;         // many rows: [CTA][2]
  unsigned long long* tickets;       // few rows: [CTA that begins an item][warp], see pa_open
  unsigned long long tag;            // this call's
  unsigned* gave_up;                 // device: waits that gave up so far
  int* status;
};
// What a CTA left in the workspace: 0 the end, or the middle, of an item that another CTA began; 1 one that it began and did not end.
struct PagedPart { int valid, ends, row0, rows, first, kv_head, queries, keys; };

#ifdef __CUDACC__
// How work is shared out is arithmetic that the host can do as well, to look at it.
#define GLQB_LIST __host__ __device__ __forceinline__
struct PagedSeq { int row0, queries, keys; };
// Lengths and offsets are held to what there is, so that whatever they hold, nothing outside is read or written.
GLQB_LIST int pa_offset(const PagedJob& J, int i) {
  if (!J.offsets) return min(i, J.tokens);
  const long long o = J.offsets_wide ? reinterpret_cast<const long long*>(J.offsets)[i] : reinterpret_cast<const int*>(J.offsets)[i];
  return (int)max(0ll, min((long long)J.tokens, o));
}
GLQB_LIST PagedSeq pa_seq(const PagedJob& J, int i) {
  PagedSeq s;
  s.row0 = pa_offset(J, i);
  s.queries = max(0, pa_offset(J, i + 1) - s.row0);
  const long long n = J.lengths_wide ? reinterpret_cast<const long long*>(J.lengths)[i] : reinterpret_cast<const int*>(J.lengths)[i];
  s.keys = (int)max(0ll, min((long long)J.most_keys, n));
  return s;
}
// rows of an item are (query, head of the group) pairs, heads first
GLQB_LIST int pa_over(int n, const PagedDivisor& d) { return (int)((unsigned long long)(uint32_t)n * d.mul >> d.shift); }
GLQB_LIST int pa_query(const PagedJob& J, int row) { return pa_over(row, J.by_group); }
// keys that query i sees: from .. to - 1
GLQB_LIST int pa_to(const PagedJob& J, const PagedSeq& s, int i) { return J.causal ? max(0, s.keys - s.queries + i + 1) : s.keys; }
GLQB_LIST int pa_from(const PagedJob& J, const PagedSeq& s, int i) {
  return J.window ? max(0, s.keys - s.queries + i + 1 - J.window) : 0;
}
// An item: J.rows rows of one sequence and key head.  Its key tiles are [lo, hi): those that any of its rows sees, one at least, so that
// every row is written.
template <int KEYS>
GLQB_LIST int2 pa_tiles(const PagedJob& J, const PagedSeq& s, int qt) {
  const int last = min(s.queries - 1, pa_query(J, min(s.queries * J.group, (qt + 1) * J.rows) - 1));
  const int to = pa_to(J, s, last), from = min(pa_from(J, s, pa_query(J, qt * J.rows)), to);
  const int lo = from / KEYS;
  return make_int2(lo, max(lo + 1, (to + KEYS - 1) / KEYS));
}
GLQB_LIST int pa_q_tiles(const PagedJob& J, const PagedSeq& s) { return pa_over(s.queries * J.group + J.rows - 1, J.by_rows); }
template <int KEYS>
GLQB_LIST long long pa_units(const PagedJob& J, const PagedSeq& s) {
  const int n = pa_q_tiles(J, s);
  long long sum = 0;
  for (int qt = 0; qt < n; ++qt) {
    const int2 t = pa_tiles<KEYS>(J, s, qt);
    sum += t.y - t.x + J.begin;
  }
  return sum;
}

// Where a CTA's share of the work begins: item (seq, kv_head, q_tile), `skip` units into it, `units` units in all.
struct PagedStart {
  PagedSeq s;
  int seq, kv_head, q_tile, skip, q_tiles;
  int2 tiles;                        // the item's
  int ctas;                          // that have a share
  long long units, at, total;        // units: of this share, which begins at unit `at`
  long long warp_sum[32];
};
// quotient of numbers >= 0 (a division of 64 bits takes some hundred clocks)
GLQB_LIST long long pa_div(long long a, long long b) { return (a | b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b); }
// CTAs that have a share of `total` units, and where that of CTA c begins: the one behind it begins where it ends.
GLQB_LIST long long pa_ctas(const PagedJob& J, long long total, int grid) {
  const long long n = pa_div(total + J.min_units - 1, J.min_units);
  return n < grid ? n : grid;
}
GLQB_LIST long long pa_begin(long long total, long long ctas, long long c) { return pa_div(total * c, ctas); }
// The item that unit r of a sequence's belongs to.
template <int KEYS>
GLQB_LIST void pa_place_start(const PagedJob& J, PagedStart& S, int seq, const PagedSeq& s, long long per_head, long long r, long long units) {
  S.s = s;
  S.seq = seq;
  S.kv_head = (int)pa_div(r, per_head);
  r -= S.kv_head * per_head;
  int qt = 0;
  int2 t;
  for (;; ++qt) {
    t = pa_tiles<KEYS>(J, s, qt);
    if (r < t.y - t.x + J.begin) break;
    r -= t.y - t.x + J.begin;
  }
  S.q_tile = qt;
  S.q_tiles = pa_q_tiles(J, s);
  S.tiles = t;
  S.skip = (int)r;
  S.units = units;
}
// The work is one list of units: sequence after sequence, of each one key head after another, of each one row tile after another, of each such item
// J.begin units for its beginning and one per key tile; every CTA takes an equal run of it.  So batches of any lengths keep all SMs busy, and an item is cut only where a run ends.  Every
// CTA counts the list itself: a thread some sequences, then a scan; up to 32 sequences are one warp's.  Called by all threads; ends with a block barrier.
template <int KEYS>
__device__ __forceinline__ void pa_start(const PagedJob& J, PagedStart& S) {
  const int threads = blockDim.x, warps = threads >> 5, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool small = J.seqs <= 32;
  if (threadIdx.x == 0) S.units = 0;
  __syncwarp();                                          // (another lane of this warp may have a share to write there)
  if (small && warp > 0) {
    __syncthreads();
    return;
  }
  const int per = small ? 1 : (J.seqs + threads - 1) / threads, first = min(J.seqs, (int)threadIdx.x * per), last = min(J.seqs, first + per);
  PagedSeq s{0, 0, 0};
  long long own = 0, per_head = 0;
  for (int i = first; i < last; ++i) {
    s = pa_seq(J, i);
    per_head = pa_units<KEYS>(J, s);
    own += per_head * J.kv_heads;
  }
  long long sum = own;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long u = __shfl_up_sync(0xFFFFFFFFu, sum, d);
    if (lane >= d) sum += u;
  }
  long long before = sum - own, total = 0;
  if (small) {
    total = __shfl_sync(0xFFFFFFFFu, sum, 31);
  } else {
    if (lane == 31) S.warp_sum[warp] = sum;
    __syncthreads();
    for (int w = 0; w < warps; ++w) {
      if (w < warp) before += S.warp_sum[w];
      total += S.warp_sum[w];
    }
  }
  const long long ctas = pa_ctas(J, total, (int)gridDim.x);
  if ((long long)blockIdx.x < ctas) {
    const long long begin = pa_begin(total, ctas, blockIdx.x), end = pa_begin(total, ctas, blockIdx.x + 1);
    if (begin >= before && begin < before + own) {
      long long r = begin - before;
      S.at = begin;
      S.total = total;
      S.ctas = (int)ctas;
      if (per == 1) {
        pa_place_start<KEYS>(J, S, first, s, per_head, r, end - begin);
      } else {
        for (int i = first; i < last; ++i) {
          s = pa_seq(J, i);
          per_head = pa_units<KEYS>(J, s);
          if (r >= per_head * J.kv_heads) { r -= per_head * J.kv_heads; continue; }
          pa_place_start<KEYS>(J, S, i, s, per_head, r, end - begin);
          break;
        }
      }
    }
  }
  __syncthreads();
}

// A CTA's items one after the other, as its loading warp hands them to the others.
struct PagedItem {
  int more;                          // 0: no item, the CTA is done
  int row0, queries, keys;           // the sequence
  int seq, kv_head, first;           // first row of the item within the sequence's queries * group
  int rows;                          // of it
  int lo, hi;                        // key tiles of this CTA
  int all_from, all_to;              // keys that all rows see: all_from .. all_to - 1
  int any_from, any_to;              // and that any row does
  int slot;                          // -1: the whole item; else its place in the workspace
  int begun_by, parts;               // CTA that has its beginning, CTAs that have a part (JOIN)
};
template <int KEYS, bool JOIN>
struct PagedWalk {
  PagedSeq s;
  int seq, kv_head, qt, skip, q_tiles;
  int2 t;                            // the item's key tiles
  int ctas;
  long long left, at, total;
  PagedPart part[2];                 // what the CTA leaves in the workspace
  GLQB_LIST PagedWalk(const PagedJob& J, const PagedStart& S)
      : s(S.s), seq(S.seq), kv_head(S.kv_head), qt(S.q_tile), skip(S.skip), q_tiles(S.q_tiles), t(S.tiles), ctas(S.ctas), left(S.units), at(S.at), total(S.total) {
    part[0] = part[1] = PagedPart{0, 1, 0, 0, 0, 0, 0, 0};
  }
  // the CTA that has unit u: the last c with total * c / ctas <= u
  GLQB_LIST int cta_of(long long u) const { return (int)pa_div((u + 1) * ctas - 1, total); }
  GLQB_LIST PagedItem next(const PagedJob& J) {
    PagedItem it{};
    while (left > 0 && !it.more) {
      const int n = t.y - t.x, take = (int)min((long long)(n + J.begin - skip), left);
      const int from = max(0, skip - J.begin), to = max(0, skip + take - J.begin);
      if (from < to) {                   // (a run that ends before the first tile leaves the item to the next CTA)
        it.more = 1;
        it.row0 = s.row0;
        it.queries = s.queries;
        it.keys = s.keys;
        it.seq = seq;
        it.kv_head = kv_head;
        it.first = qt * J.rows;
        it.rows = min(J.rows, s.queries * J.group - it.first);
        it.lo = t.x + from;
        it.hi = t.x + to;
        const int i0 = pa_query(J, it.first), i1 = pa_query(J, it.first + it.rows - 1);
        it.all_from = pa_from(J, s, i1);
        it.all_to = pa_to(J, s, i0);
        it.any_from = pa_from(J, s, i0);
        it.any_to = pa_to(J, s, i1);
        it.slot = to - from == n ? -1 : from ? 0 : 1;
        if (JOIN && it.slot >= 0) {
          const long long first = at - skip + J.begin;
          it.begun_by = cta_of(first);
          it.parts = cta_of(first + n - 1) - it.begun_by + 1;
        }
        if (it.slot >= 0) part[it.slot] = PagedPart{1, to == n, s.row0, it.rows, it.first, kv_head, s.queries, s.keys};
      }
      left -= take;
      at += take;
      skip = 0;
      if (++qt == q_tiles) {
        qt = 0;
        if (++kv_head == J.kv_heads) {
          kv_head = 0;
          if (left > 0) {
            do { s = pa_seq(J, ++seq); } while (s.queries == 0 && seq + 1 < J.seqs);
            q_tiles = pa_q_tiles(J, s);
          }
        }
      }
      if (left > 0) t = pa_tiles<KEYS>(J, s, qt);
    }
    return it;
  }
};
// A ticket counts the parts of an item that are there.  It is the call's tag (52 bits) and a number (12), so that nothing has to be cleared in
// front of a call: whoever is to arrive at it opens it first, which sets it to (tag, 0) if it has another tag, whatever the memory held
// before.  The last to arrive leaves it cleared, as a captured call that is replayed has the same tag again.  Tags are numbers of a 52-bit sequence that
// starts anywhere; a launch whose waits gave up, which may leave tickets behind, moves the tags of those after it (J.gave_up).  (Counting by
// compare and swap alone: 37 CTAs that arrive together took 15 us.)
__device__ __forceinline__ void pa_open(unsigned long long* ticket, unsigned long long tag) {
  const unsigned long long old = *(volatile unsigned long long*)ticket;
  if (old >> 12 != tag) atomicCAS(ticket, old, tag << 12);         // (where that fails, another has opened it)
}
// true for the last of `parts`
__device__ __forceinline__ bool pa_arrive(unsigned long long* ticket, int parts) {
  const bool last = (int)(atomicAdd(ticket, 1ull) & 4095u) + 1 == parts;
  if (last) *(volatile unsigned long long*)ticket = 0ull;
  return last;
}
// 32 bytes at once
__device__ __forceinline__ void store8(void* p, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void load8(const float* p, float4& a, float4& b) {
  asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : "=f"(a.x), "=f"(a.y), "=f"(a.z), "=f"(a.w), "=f"(b.x), "=f"(b.y), "=f"(b.z), "=f"(b.w) : "l"(p) : "memory");
}
// Where eight values of a row are in a part of many rows: row r (128 to a half), values 8 g and up.  A warp that has 32 rows writes, and reads, a
// kilobyte of them at once.
template <int DP>
__device__ __forceinline__ long long pa_part_at(int slot, int r, int g) {
  return (long long)slot * PA_TILE_ROWS * DP + (((r >> 7) * (DP / 8) + g) * 128 + (r & 127)) * 8;
}
__device__ __forceinline__ void pa_publish(const PagedJob& J, const PagedPart (&part)[2]) {
  J.part_of[2 * blockIdx.x] = part[0];
  J.part_of[2 * blockIdx.x + 1] = part[1];
}

// `rows` rows (PA_PIECE at most) x 64 values of one head of a page: coordinates (value, head, row, page)
__device__ __forceinline__ void pa_load(void* dst, const CUtensorMap* map, int x, int head, int row, int page, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
                   smem_u32(dst)),
               "l"(map), "r"(x), "r"(head), "r"(row), "r"(page), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ float pa_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pa_pack(float a, float b) {
  if constexpr (__is_same(T, __half)) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename T> __device__ __forceinline__ T pa_round(float v) {
  if constexpr (__is_same(T, float)) return v;
  else if constexpr (__is_same(T, __half)) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}
template <typename T>
__device__ __forceinline__ float2 pa_unpack(uint32_t two) {
  if constexpr (__is_same(T, __half)) return __half22float2(*reinterpret_cast<const __half2*>(&two));
  else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&two));
}
// Weights are 2^(score - reference + this), of which a row's sums, its parts and their sums all have the factor, so that the quotient loses it.  fp16's
// smallest number is 2^-24: without it what weighs 2^-25 of a row's strongest key is nothing in the sum over the values and something in the sum that divides it
// (131,071 such keys beside a strong one: 0.4 % of the result).  PA_LAZY more is 2^15, of at most 65,504.  bf16 has fp32's exponents.
template <typename T> __device__ __forceinline__ constexpr float pa_up() { return __is_same(T, __half) ? 7.0f : 0.0f; }
// four columns of a row of the result
template <typename T>
__device__ __forceinline__ void pa_store4(const PagedJob& J, long long at, int col, float4 v) {
  T* p = reinterpret_cast<T*>(J.out) + at + col;
  if (J.out_wide) {                                        // (head_dim is a multiple of 8: four columns are all there, or none)
    *reinterpret_cast<uint2*>(p) = make_uint2(pa_pack<T>(v.x, v.y), pa_pack<T>(v.z, v.w));
  } else {
    p[0] = pa_round<T>(v.x); p[1] = pa_round<T>(v.y); p[2] = pa_round<T>(v.z); p[3] = pa_round<T>(v.w);
  }
}
__device__ __forceinline__ long long pa_out_row(const PagedJob& J, int row0, int kv_head, int row) {
  const int i = pa_query(J, row);
  return (long long)(row0 + i) * J.out_token + (long long)(kv_head * J.group + row - i * J.group) * J.out_head;
}
// What a row's sums are multiplied by.  Weights of nothing: a row that sees no key is zero; one that does has only scores of minus
// infinity, which have no softmax.
__device__ __forceinline__ float pa_row_factor(const PagedJob& J, const PagedSeq& s, int row, float sum) {
  if (sum != 0.0f) return 1.0f / sum;
  const int i = pa_query(J, row);
  return pa_to(J, s, i) > pa_from(J, s, i) ? NAN : 0.0f;
}
// has one of two 16-bit values no finite value?
template <typename T>
__device__ __forceinline__ bool pa_not_finite(uint32_t two) {
  constexpr uint32_t E = __is_same(T, __half) ? 0x7C00u : 0x7F80u;
  return (two & E) == E || (two >> 16 & E) == E;
}
#endif  // __CUDACC__

inline int pg_device_index() {       // the current one, 0..63
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64 ? dev : 0;
}
// Chained to the kernel in front (launch_chained).
template <auto K, typename... P, typename... A>
inline cudaError_t paged_launch(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream, A... args) {
  static std::atomic<bool> raised[64];   // per device: may the kernel have the shared memory it needs?
  std::atomic<bool>& r = raised[pg_device_index()];
  if (smem > 48 * 1024 && !r.load(std::memory_order_relaxed)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    r.store(true, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled();
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// ---- glqb_paged_tile.cu
// Many rows, on the tensor cores: one CTA per SM, items of two tiles of J.rows / 2 rows.  `queries`: boxes of 64 values x a group of heads x 128 / group tokens.
cudaError_t paged_tile_launch(const PagedJob& J, bool bf16, const CUtensorMap& queries, const CUtensorMap& keys, const CUtensorMap& values, int ctas, cudaStream_t stream);

}  // namespace glqb
