// The list of attention's work on the host: what each CTA takes, from the functions that the kernels call.  Built by test_paged.py.
#include "glqb_paged.cuh"

using namespace glqb;

template <int KEYS>
static int walk(const PagedJob& J, int grid, int* out, int most) {
  long long total = 0;
  for (int i = 0; i < J.seqs; ++i) total += pa_units<KEYS>(J, pa_seq(J, i)) * J.kv_heads;
  const long long ctas = pa_ctas(J, total, grid);
  int n = 0;
  for (long long c = 0; c < ctas; ++c) {
    const long long begin = pa_begin(total, ctas, c), end = pa_begin(total, ctas, c + 1);
    PagedStart S = {};
    S.at = begin;
    S.total = total;
    S.ctas = (int)ctas;
    long long r = begin;
    for (int i = 0; i < J.seqs; ++i) {
      const PagedSeq s = pa_seq(J, i);
      const long long per_head = pa_units<KEYS>(J, s);
      if (r >= per_head * J.kv_heads) { r -= per_head * J.kv_heads; continue; }
      pa_place_start<KEYS>(J, S, i, s, per_head, r, end - begin);
      break;
    }
    PagedWalk<KEYS, true> w(J, S);
    for (PagedItem it = w.next(J); it.more; it = w.next(J)) {
      const int row[] = {(int)c, it.seq, it.kv_head, it.first, it.rows, it.lo, it.hi, it.slot, it.begun_by, it.parts, it.all_from, it.all_to, it.any_from, it.any_to};
      if (n == most) return -1;
      for (int k = 0; k < 14; ++k) out[n * 14 + k] = row[k];
      ++n;
    }
  }
  return n;
}

// rows of 14 numbers: CTA, sequence, key head, first row, rows, key tiles from and to, slot, CTA that began the item and number of its parts (of items
// that are cut), keys that all rows see from and to, and that any row does
extern "C" int paged_list(const long long* lengths, const long long* offsets, int seqs, int tokens, int most_keys, int group, int kv_heads, int rows, int keys, int grid, int begin,
                          int least, int causal, int window, int* out, int most) {
  PagedJob J = {};
  J.lengths = lengths;
  J.offsets = offsets;
  J.lengths_wide = J.offsets_wide = 1;
  J.seqs = seqs;
  J.tokens = tokens;
  J.most_keys = most_keys;
  J.group = group;
  J.kv_heads = kv_heads;
  J.heads = group * kv_heads;
  J.rows = rows;
  J.by_group = pa_divisor(group);
  J.by_rows = pa_divisor(rows);
  J.begin = begin;
  J.min_units = least;
  J.causal = causal;
  J.window = window;
  return keys == PA_STREAM_KEYS ? walk<PA_STREAM_KEYS>(J, grid, out, most) : walk<PA_TILE_KEYS>(J, grid, out, most);
}
