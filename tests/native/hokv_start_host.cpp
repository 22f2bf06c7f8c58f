// Host build of the search for where a CTA's share begins (packed_schedule.cuh),
// over 32 emulated lanes.
#include "packed_schedule.cuh"

using namespace hokv;

extern "C" {

// Sequence, pair and units before the sequence for each of the n units `begin`;
// returns the total.
int64_t host_starts(const int* cu_q, const int* kv_len, int n_seqs, int T, int Hkv, int TT, int64_t kv_rows, int prefix,
                    int causal, const int64_t* begin, int n, int64_t* out) {
  PaSched p = {cu_q, nullptr, kv_len, n_seqs, T, Hkv, TT, kv_rows, prefix, causal, 148};
  int64_t mine[32], upto[32], total = 0;
  bool bad = false;
  for (int lane = 0; lane < 32; ++lane) {
    mine[lane] = pa_lane_units(p, lane, bad);
    upto[lane] = total += mine[lane];
  }
  for (int i = 0; i < n; ++i) {
    const PaStart r = pa_find_start(p, begin[i], [&](int lane) { return mine[lane]; }, [&](int lane) { return upto[lane]; });
    out[3 * i] = r.s;
    out[3 * i + 1] = r.pr;
    out[3 * i + 2] = r.at;
  }
  return bad ? -1 : total;
}
}
