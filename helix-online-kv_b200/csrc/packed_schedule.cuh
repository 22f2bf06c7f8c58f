// packed_schedule.cuh -- how the packed attention cuts its work over the CTAs.
//
// An item is up to 2 TT query tokens of one sequence and one KV head (a pair of
// 128-row tiles, TT = 128 / G tokens each) against the keys it sees.  It costs
// PA_ITEM units plus 2 per visible key, 1 when its tokens fit one tile.  The
// units of all items, ordered by (sequence, pair, KV head), form one line; CTA
// c takes units [c, c + 1) * share.  A border inside an item cuts it between
// two key tiles into pieces; a short item goes whole to the CTA its keys start
// in.  The units before a pair are an arithmetic
// series, so a CTA finds its first item without walking the others, and with
// few instructions: a short call waits for this code from cold caches.
//
// Plain C++ apart from the HD marks, so the host can check the same code.
#pragma once
#include "hokv_math.cuh"

namespace hokv {

// Loops are kept rolled on the device: the roles of the kernel share one
// instruction cache.
#if defined(__CUDACC__)
#define ROLLED _Pragma("unroll 1")
#else
#define ROLLED
#endif

constexpr int PA_BN = 128;          // keys of a tile
constexpr int PA_ITEM = 512;        // units of an item besides its keys (start, epilogue, half an unseen
                                    // key tile; in turns on one box, 448: 16K prompt 1 % slower, 576: the same and single
                                    // tokens 1 % slower)
// An item up to this (8 one-tile key tiles) is not cut: one token at 300 keys takes 11 us whole, 18 in pieces, 8 at
// 700 keys 17 and 20; at 1,000 keys both take 18.
constexpr int PA_WHOLE = 1536;
constexpr int PA_MIN_SHARE = 768;   // smallest share of a CTA: an item's start and two key tiles of a one-tile item

enum { PA_DIRECT = 0, PA_PIECE = 1, PA_ROWWISE = 2, PA_STOP = 3 };

struct PaItem {
  int tok0, n_tok;     // query tokens [tok0, tok0 + n_tok)
  int src;             // 0: own keys, 1: shared prefix
  int row0, slot;      // first key row and slot of the sequence in its tensor
  int hk;
  int j0, j1;          // key tiles of this piece
  int kv_len, pos0;    // token i sees keys < min(kv_len, pos0 + i + 1)
  int out_mode;        // PA_DIRECT: final rows; PA_PIECE: workspace slot out_at; PA_ROWWISE: a result per row
  int out_at;
};

struct PaSched {
  const int* cu_q;               // [n_seqs + 1] or null: one token each
  const int* cu_k;               // packed keys: [n_seqs + 1]
  const int* kv_len;             // keys in slots: [n_seqs]
  int n_seqs, T, Hkv, TT;
  int64_t kv_rows;               // rows of the packed keys, or of a slot
  int prefix;                    // shared prefix length, 0 without one
  int causal, n_ctas;
};

struct PaSeq {
  int q0, nq, row0, slot, kv, src, causal, bad;
};

HD int64_t pa_min(int64_t a, int64_t b) { return a < b ? a : b; }
HD int64_t pa_max(int64_t a, int64_t b) { return a > b ? a : b; }

HD int pa_n_seqs(const PaSched& p) { return p.n_seqs + (p.prefix > 0 ? 1 : 0); }
// The query tokens [first, used) belong to the sequences.
HD int pa_first(const PaSched& p) { return p.cu_q && p.n_seqs > 0 ? (int)pa_min(pa_max(p.cu_q[0], 0), p.T) : 0; }
HD int pa_used(const PaSched& p) {
  if (!p.cu_q || p.n_seqs == 0) return p.n_seqs;
  return (int)pa_min(pa_max(p.cu_q[p.n_seqs], 0), p.T);
}

// Sequence s of the schedule (with a prefix, 0 is the prefix against all
// tokens).  One whose lengths do not fit the tensors is `bad` and empty, so
// that nothing outside the buffers is read or written.
HD PaSeq pa_seq(const PaSched& p, int s) {
  PaSeq r;
  r.bad = 0;
  if (p.prefix > 0) {
    if (s == 0) {
      r.row0 = r.slot = 0;
      r.q0 = pa_first(p);
      r.nq = (int)pa_max(pa_used(p) - r.q0, 0);
      r.kv = p.prefix;
      r.src = 1;
      r.causal = 0;
      return r;
    }
    s -= 1;
  }
  const int a = p.cu_q ? p.cu_q[s] : s, e = p.cu_q ? p.cu_q[s + 1] : s + 1;
  bool bad = a < 0 || e < a || e > p.T;
  r.src = 0;
  r.causal = p.causal;
  if (p.cu_k) {
    const int ka = p.cu_k[s], ke = p.cu_k[s + 1];
    bad = bad || ka < 0 || ke < ka || ke > p.kv_rows;
    r.row0 = ka;
    r.slot = 0;
    r.kv = bad ? 0 : ke - ka;
  } else {
    r.row0 = 0;
    r.slot = s;
    r.kv = p.kv_len[s];
    bad = bad || r.kv < 0 || r.kv > p.kv_rows;
  }
  r.q0 = bad ? 0 : a;
  r.nq = bad ? 0 : e - a;
  r.bad = bad;
  return r;
}

// Keys that token pair `pr` (W = 2 TT tokens) of a sequence sees.
HD int pa_keys(const PaSeq& s, int W, int pr) {
  if (!s.causal) return s.kv;
  const int last = s.nq - pr * W < W ? s.nq : (pr + 1) * W;
  return (int)pa_max(s.kv - s.nq + last, 0);
}

// Units, of one KV head, of the first n pairs (none of them the last) of nq
// tokens against kv keys.
HD int64_t pa_units_before(int kv, int nq, int causal, int W, int n) {
  int64_t keys = (int64_t)n * kv;
  if (causal) {
    const int64_t off = (int64_t)kv - nq;
    const int skip = off < 0 ? (int)pa_min(n, (int)-off / W) : 0;   // pairs that see nothing
    const int64_t m = n - skip;
    keys = m * off + W * (m * (m + 1) / 2 + m * skip);
  }
  return (int64_t)n * PA_ITEM + 2 * keys;
}

// Units of one KV head's item of pair `pr`.
HD int64_t pa_item_units(const PaSeq& s, int W, int pr) {
  return PA_ITEM + ((int64_t)pa_keys(s, W, pr) << (s.nq - pr * W > W / 2 ? 1 : 0));
}

HD int64_t pa_seq_units(const PaSched& p, const PaSeq& s) {
  const int W = 2 * p.TT;
  if (s.nq <= 0) return 0;
  const int last = (s.nq + W - 1) / W - 1;
  return (int64_t)p.Hkv * (pa_units_before(s.kv, s.nq, s.causal, W, last) + pa_item_units(s, W, last));
}

// A share of at least total / n_ctas (the same value in every CTA; the product
// is off by less than 1).
HD int64_t pa_share(const PaSched& p, int64_t total) {
  return pa_max((int64_t)((double)total * (1.0 / p.n_ctas)) + 1, PA_MIN_SHARE);
}

// The key tile at which x units behind an item's fixed part cut it (tiles of
// 2^sh units): a tile belongs to the piece in which its units start.
HD int pa_cut(int64_t x, int sh, int tiles) {
  return x <= 0 ? 0 : (int)pa_min((x + ((int64_t)1 << sh) - 1) >> sh, tiles);
}

// The CTAs that hold the first and the last piece of a cut item at unit
// item_at: its pieces are slot 1 of the first and slot 0 of every CTA behind it
// up to the last (a share is longer than a key tile, so none is empty).
HD int pa_first_cta(int64_t share, int64_t item_at) {
  const int c = (int)(item_at / share);   // unless only the units ahead of its keys lie there
  return (int64_t)(c + 1) * share - item_at - PA_ITEM > 0 ? c : c + 1;
}
HD int pa_last_cta(int64_t share, int64_t item_at, int sh, int tiles) {
  return (int)((item_at + PA_ITEM + ((int64_t)(tiles - 1) << sh)) / share);
}

// Where a CTA's share begins is found by a warp.  The host runs the same code
// over 32 lanes in turn: f(lane) is each lane's value.
template <typename F>
HD unsigned pa_ballot(F f) {
#if defined(__CUDA_ARCH__)
  return __ballot_sync(0xffffffffu, f((int)(threadIdx.x & 31)));
#else
  unsigned votes = 0;
  for (int lane = 0; lane < 32; ++lane) votes |= (f(lane) ? 1u : 0u) << lane;
  return votes;
#endif
}
template <typename F>
HD int64_t pa_from(int lane, F f) {
#if defined(__CUDA_ARCH__)
  return __shfl_sync(0xffffffffu, f((int)(threadIdx.x & 31)), lane);
#else
  return f(lane);
#endif
}
HD int pa_lowest(unsigned votes) {   // of at least one
#if defined(__CUDA_ARCH__)
  return __ffs(votes) - 1;
#else
  return __builtin_ctz(votes);
#endif
}
HD int pa_highest(unsigned votes) {
#if defined(__CUDA_ARCH__)
  return 31 - __clz(votes);
#else
  return 31 - __builtin_clz(votes);
#endif
}

// Units of the sequences that are one lane's to count, and whether one of them is bad.
HD int pa_lane_first(const PaSched& p, int lane) {
  const int n_s = pa_n_seqs(p);
  return (int)pa_min((int64_t)lane * ((n_s + 31) / 32), n_s);
}
HD int64_t pa_lane_units(const PaSched& p, int lane, bool& bad) {
  const int last = pa_lane_first(p, lane + 1);
  int64_t units = 0;
  ROLLED for (int s = pa_lane_first(p, lane); s < last; ++s) {
    const PaSeq q = pa_seq(p, s);
    bad = bad || q.bad;
    units += pa_seq_units(p, q);
  }
  return units;
}

// The last pair of sequence q (`at` units before it) that starts at or before
// unit pos, 32 probes at a time.
HD int pa_find_pair(const PaSched& p, const PaSeq& q, int64_t at, int64_t pos) {
  const int W = 2 * p.TT;
  int pr = 0;
  ROLLED for (int n = (q.nq + W - 1) / W; n > 1;) {
    const int step = (n + 31) / 32;
    const unsigned before = pa_ballot([&](int lane) {   // lane 0's always is
      const int probe = (int)pa_min(pr + lane * step, pr + n - 1);
      return at + (int64_t)p.Hkv * pa_units_before(q.kv, q.nq, q.causal, W, probe) <= pos && lane * step < n;
    });
    const int k = pa_highest(before);
    n = (int)pa_min(step, n - k * step);
    pr += k * step;
  }
  return pr;
}

// The sequence and pair that hold unit `begin` (below the total), and the units
// before the sequence.  mine(lane), upto(lane): a lane's units, and those of
// all lanes up to it.
struct PaStart {
  int s, pr;
  int64_t at;
};
template <typename Mine, typename Upto>
HD PaStart pa_find_start(const PaSched& p, int64_t begin, Mine mine, Upto upto) {
  PaStart r;
  const int owner = pa_lowest(pa_ballot([&](int lane) { return upto(lane) > begin; }));
  r.s = pa_lane_first(p, owner);
  r.at = pa_from(owner, [&](int lane) { return upto(lane) - mine(lane); });
  PaSeq q = pa_seq(p, r.s);
  const bool several = pa_n_seqs(p) > 32;   // sequences of a lane
  ROLLED for (int64_t units; several && r.at + (units = pa_seq_units(p, q)) <= begin; q = pa_seq(p, ++r.s)) r.at += units;
  r.pr = pa_find_pair(p, q, r.at, begin);
  return r;
}

// CTA `cta`'s items: units [begin, end), which start in pair `pr` of sequence s
// (`at` units before it).  emit(item, begins, ends, ...): whether the piece
// holds the item's first and its last key tile, and the item's place and tiles
// (pa_first_cta, pa_last_cta); false stops the walk.
template <typename Emit>
HD bool pa_walk(const PaSched& p, int cta, int64_t begin, int64_t end, int s, int64_t at, int pr, Emit emit) {
  const int W = 2 * p.TT, n_s = pa_n_seqs(p);
  int64_t pos = begin;
  ROLLED for (; s < n_s && pos < end; ++s) {
    const PaSeq q = pa_seq(p, s);
    if (q.nq <= 0) continue;
    const int np = (q.nq + W - 1) / W;
    int64_t item_at = at + (int64_t)p.Hkv * pa_units_before(q.kv, q.nq, q.causal, W, pr);
    ROLLED for (; pr < np && pos < end; ++pr) {
      const int left = q.nq - pr * W;
      const int n_tok = left < W ? left : W;
      const int keys = pa_keys(q, W, pr);
      const int tiles = (keys + PA_BN - 1) / PA_BN;
      const int sh = n_tok > p.TT ? 8 : 7;          // units of a key tile: 2^sh
      const int64_t iu = pa_item_units(q, W, pr);
      ROLLED for (int hk = 0; hk < p.Hkv; ++hk, item_at += iu) {
        if (item_at + iu <= pos) continue;
        if (pos >= end) break;
        const bool start = pos == item_at, short_item = iu <= PA_WHOLE;
        const int t0 = short_item ? 0 : pa_cut(pos - item_at - PA_ITEM, sh, tiles);
        const int t1 = short_item ? (pos <= item_at + PA_ITEM && item_at + PA_ITEM < end ? tiles : 0) : pa_cut(end - item_at - PA_ITEM, sh, tiles);
        pos = pa_min(item_at + iu, end);
        if (tiles > 0 ? t0 == t1 : !start) continue;
        PaItem w;
        w.tok0 = q.q0 + pr * W;
        w.n_tok = n_tok;
        w.src = q.src;
        w.row0 = q.row0;
        w.slot = q.slot;
        w.hk = hk;
        w.j0 = t0;
        w.j1 = t1;
        w.kv_len = q.kv;
        w.pos0 = q.causal ? q.kv - q.nq + pr * W : 0x3fffffff;
        const bool begins = t0 == 0, ends = t1 == tiles;
        w.out_mode = !(begins && ends) ? PA_PIECE : p.prefix > 0 ? PA_ROWWISE : PA_DIRECT;
        // a CTA's share begins with at most one unfinished item and ends with at most one
        w.out_at = cta * 2 + (begins ? 1 : 0);
        if (!emit(w, begins, ends, item_at, sh, tiles)) return false;
      }
    }
    at = item_at;
    pr = 0;
  }
  return true;
}

}  // namespace hokv
