// Host build of the packed attention's schedule (packed_schedule.cuh).
#include "packed_schedule.cuh"

using namespace hokv;

extern "C" {

// Every piece of every CTA, 16 ints each: cta, begins, ends, then PaItem's
// fields.  Returns the number of pieces, or -1 when `cap` is too small.
int64_t host_schedule(const int* cu_q, const int* cu_k, const int* kv_len, int n_seqs, int T, int Hkv, int TT,
                      int64_t kv_rows, int prefix, int causal, int n_ctas, int* out, int64_t cap, int64_t* units) {
  PaSched p = {cu_q, cu_k, kv_len, n_seqs, T, Hkv, TT, kv_rows, prefix, causal, n_ctas};
  const int n_s = pa_n_seqs(p);
  int64_t total = 0;
  for (int s = 0; s < n_s; ++s) total += pa_seq_units(p, pa_seq(p, s));
  *units = total;
  const int64_t share = pa_share(p, total);
  int64_t n = 0;
  for (int c = 0; c < n_ctas; ++c) {
    const int64_t begin = pa_min(c * share, total), end = pa_min(begin + share, total);
    if (begin >= end) continue;
    int s = 0;
    int64_t at = 0;
    for (; at + pa_seq_units(p, pa_seq(p, s)) <= begin; ++s) at += pa_seq_units(p, pa_seq(p, s));
    const bool ok = pa_walk(p, c, begin, end, s, at, pa_find_pair(p, pa_seq(p, s), at, begin), [&](const PaItem& w, bool begins, bool ends, int64_t item_at, int sh, int tiles) {
      if (n == cap) return false;
      int* o = out + 16 * n++;
      const int f[16] = {c, begins, ends, w.tok0, w.n_tok, w.src, w.row0, w.slot, w.hk, w.j0, w.j1, w.kv_len, w.pos0,
                         w.out_mode, w.out_at, 0};
      for (int i = 0; i < 16; ++i) o[i] = f[i];
      if (tiles > 0) o[15] = pa_first_cta(share, item_at) * 1000 + pa_last_cta(share, item_at, sh, tiles);
      return true;
    });
    if (!ok) return -1;
  }
  return n;
}
}
