// norm_rotate.cuh -- the new tokens of a packed batch on their way into the
// slots: RMS norm of each query and key head, rotary position, append.
//
// For token i of sequence b (position P = kv_len[b] + i, or positions[t]):
//   y = x w / sqrt(mean(x^2) + eps)              per head of q and k (w optional)
//   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin),  angle = P inv_freq[f]
// for the first 2 n_freq dims, pairs (f, f + n_freq) or, interleaved,
// (2f, 2f + 1); q goes to `out`, k and v to row kv_len[b] + i of b's slot.
//
// Bound by memory: q, k and v are read once and written once.  A group of
// LPR = D / 16 lanes (rounded up to a power of two) owns a row; a lane holds
// both elements of its pairs, as two 16-byte chunks of 8 (16-bit types), so
// the rotation needs no exchange and the norm only the sum of squares over
// the group.  A group keeps the cosines of its token in registers over several
// heads.  The angle is formed in 64 bits as a fraction of a turn (a position
// of 10^6 times an fp32 frequency loses its phase in 32 bits); norms and
// products are fp32, rounded once at the store.
#pragma once
#include "hokv_common.cuh"

namespace hokv {

struct NraP {
  const void *q, *k, *v, *qw, *kw;
  void *out, *ks, *vs;
  int64_t q_t, q_h, k_t, k_h, v_t, v_h, out_t, out_h, ks_b, ks_h, ks_t, vs_b, vs_h, vs_t;   // element strides
  const int *cu, *kv_len, *pos;
  const float* inv_freq;
  int64_t cap;
  int n_seqs, T, Hq, Hkv, D, n_freq, interleaved, zero_tail;
  int chunks, hpg;   // head rows of a token over `chunks` groups, `hpg` each
  float eps;
};

constexpr int NRA_THREADS = 256;

// The sequence that holds token t, by the whole warp (t warp-uniform): 32-way
// search of the ascending starts.  n_seqs when t lies behind the last one.
__device__ __forceinline__ int nra_sequence(const int* cu, int n_seqs, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = n_seqs;   // first s of [lo, hi) with cu[s + 1] > t, hi when there is none
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32;
    const int probe = min(lo + (lane + 1) * step, hi) - 1;   // the last s of this lane's part
    const unsigned past = __ballot_sync(0xffffffffu, cu[probe + 1] > t);
    if (!past) return hi == n_seqs ? n_seqs : hi;
    const int f = __ffs(past) - 1;
    hi = min(lo + (f + 1) * step, hi);
    lo = lo + f * step;
    if (step == 1) return lo;
  }
  return n_seqs;
}

struct NraTok {
  int b, row, pos;   // sequence (-1: none), row in its slot, rotary position
  bool keep;         // the row lies in the slot
};

// Sequence, slot row and position of token t (warp-uniform).
__device__ __forceinline__ NraTok nra_token(const NraP& p, int t) {
  NraTok r;
  int b, i = 0;
  if (p.cu) {
    b = nra_sequence(p.cu, p.n_seqs, t);
    if (b < p.n_seqs) i = t - p.cu[b];
  } else {
    b = t;
  }
  r.b = b < p.n_seqs ? b : -1;
  r.row = r.pos = 0;
  r.keep = false;
  if (r.b >= 0) {
    const int n = p.kv_len[b];
    r.row = n + i;
    r.keep = n >= 0 && i >= 0 && (int64_t)n + i < p.cap;
    if (!r.keep) dev_flag(HOKV_ERR_DEVICE_INPUT);
    r.pos = p.pos ? p.pos[t] : r.row;
  }
  return r;
}

// cos and sin of pos * f: the product and its fraction of a turn in 64 bits.
__device__ __forceinline__ void nra_angle(int pos, float f, float& c, float& s) {
  const double turns = (double)pos * (double)f * 0.15915494309189533577;   // 1 / (2 pi)
  const float frac = (float)(turns - rint(turns));
  sincospif(2.f * frac, &s, &c);
}

template <typename T>
struct Vec8 {
  T x[8];
};
template <typename T>
__device__ __forceinline__ void nra_load8(const T* p, float (&f)[8]) {
  if constexpr (sizeof(T) == 2) {
    const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p));
    const Vec8<T> w = *reinterpret_cast<const Vec8<T>*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)w.x[i];
  } else {
    const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
}
template <typename T>
__device__ __forceinline__ void nra_store8(T* p, const float (&f)[8]) {
  if constexpr (sizeof(T) == 2) {
    Vec8<T> w;
#pragma unroll
    for (int i = 0; i < 8; ++i) w.x[i] = T(f[i]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&w);
  } else {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
}

// Source and destination of head row h of token t (q heads, then k, then v);
// kind 0 q, 1 k, 2 v.
template <typename T>
__device__ __forceinline__ int nra_row(const NraP& p, int t, int h, const NraTok& k, const T*& src, T*& dst) {
  if (h < p.Hq) {
    src = reinterpret_cast<const T*>(p.q) + t * p.q_t + h * p.q_h;
    dst = reinterpret_cast<T*>(p.out) + t * p.out_t + h * p.out_h;
    return 0;
  }
  h -= p.Hq;
  if (h < p.Hkv) {
    src = reinterpret_cast<const T*>(p.k) + t * p.k_t + h * p.k_h;
    dst = reinterpret_cast<T*>(p.ks) + k.b * p.ks_b + h * p.ks_h + k.row * p.ks_t;
    return 1;
  }
  h -= p.Hkv;
  src = reinterpret_cast<const T*>(p.v) + t * p.v_t + h * p.v_h;
  dst = reinterpret_cast<T*>(p.vs) + k.b * p.vs_b + h * p.vs_h + k.row * p.vs_t;
  return 2;
}

// Vector form: D a multiple of 16, and of the rotated dims too unless
// interleaved.  grid (ceil(T chunks / groups of a block)).
template <typename T, int LPR>
__global__ void __launch_bounds__(NRA_THREADS) k_norm_rotate(const NraP p) {
  constexpr int GROUPS = NRA_THREADS / LPR, WG = 32 / LPR;
  const int lane = threadIdx.x & 31, l = threadIdx.x % LPR;
  const int64_t unit = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LPR;
  const int64_t units = (int64_t)p.T * p.chunks;
  const bool live = unit < units;
  const int t = live ? (int)(unit / p.chunks) : p.T - 1, chunk = (int)(unit % p.chunks);
  // this lane's chunks of 8: both halves of its pairs
  const int nl = p.D / 16, lr = p.interleaved ? 0 : p.n_freq / 8;   // lanes in use, lanes of the half-split rotation
  const bool on = live && l < nl;
  const int ca = l < lr ? l : 2 * lr + 2 * (l - lr), cb = l < lr ? l + lr : ca + 1;
  const int heads = p.Hq + 2 * p.Hkv;

  // the token of each of the warp's groups (usually one for all of them)
  NraTok tok;
  if (p.chunks >= WG && __all_sync(0xffffffffu, t == __shfl_sync(0xffffffffu, t, 0))) {
    tok = nra_token(p, __shfl_sync(0xffffffffu, t, 0));
  } else {
    for (int g = 0; g < WG; ++g) {
      const NraTok k = nra_token(p, __shfl_sync(0xffffffffu, t, g * LPR));
      if (lane / LPR == g) tok = k;
    }
  }
  float c[8], s[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    c[j] = 1.f;
    s[j] = 0.f;
    const int f = 8 * l + j;
    if (on && f < p.n_freq) nra_angle(tok.pos, p.inv_freq[f], c[j], s[j]);
  }
  for (int i = 0; i < p.hpg; ++i) {
    const int h = chunk + i * p.chunks;
    const bool row_on = on && h < heads;
    const T* src = nullptr;
    T* dst = nullptr;
    const int kind = nra_row<T>(p, t, min(h, heads - 1), tok, src, dst);
    float a[8] = {}, b[8] = {};
    if (row_on) {
      nra_load8(src + ca * 8, a);
      nra_load8(src + cb * 8, b);
    }
    if (kind < 2) {
      const T* w = reinterpret_cast<const T*>(kind == 0 ? p.qw : p.kw);
      if (w) {   // uniform over the group: its lanes share the row
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += a[j] * a[j] + b[j] * b[j];
        const unsigned mask = LPR == 32 ? 0xffffffffu : ((1u << LPR) - 1u) << (lane / LPR * LPR);
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
        const float r = rsqrtf(ss / (float)p.D + p.eps);
        if (row_on) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            a[j] *= r * (float)w[ca * 8 + j];
            b[j] *= r * (float)w[cb * 8 + j];
          }
        }
      }
      if (p.interleaved) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (8 * l + j < p.n_freq) {
            const float x = a[2 * j], y = a[2 * j + 1];
            a[2 * j] = x * c[j] - y * s[j];
            a[2 * j + 1] = y * c[j] + x * s[j];
          }
          if (8 * l + 4 + j < p.n_freq) {
            const float x = b[2 * j], y = b[2 * j + 1];
            b[2 * j] = x * c[j + 4] - y * s[j + 4];
            b[2 * j + 1] = y * c[j + 4] + x * s[j + 4];
          }
        }
      } else if (l < lr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x = a[j], y = b[j];
          a[j] = x * c[j] - y * s[j];
          b[j] = y * c[j] + x * s[j];
        }
      }
    }
    const bool store = kind == 0 ? tok.b >= 0 || p.zero_tail : tok.keep;
    if (kind == 0 && tok.b < 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] = b[j] = 0.f;
    }
    if (row_on && store) {
      nra_store8(dst + ca * 8, a);
      nra_store8(dst + cb * 8, b);
    }
  }
}

// Scalar form, any even D up to 256 and any number of rotated pairs: a warp
// per head row, a lane owns whole pairs.
template <typename T>
__global__ void __launch_bounds__(NRA_THREADS) k_norm_rotate_scalar(const NraP p) {
  const int lane = threadIdx.x & 31;
  const int heads = p.Hq + 2 * p.Hkv;
  const int64_t row = (int64_t)blockIdx.x * (NRA_THREADS / 32) + (threadIdx.x >> 5);
  if (row >= (int64_t)p.T * heads) return;
  const int t = (int)(row / heads), h = (int)(row % heads);
  const NraTok tok = nra_token(p, t);
  const T* src;
  T* dst;
  const int kind = nra_row<T>(p, t, h, tok, src, dst);
  // pair e: rotated for e < n_freq, then the dims left over, two by two
  float a[4], b[4];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = lane + 32 * i;
    if (e < p.D / 2) {
      const int ia = e < p.n_freq && !p.interleaved ? e : 2 * e;
      const int ib = e < p.n_freq && !p.interleaved ? e + p.n_freq : ia + 1;
      a[i] = (float)src[ia];
      b[i] = (float)src[ib];
      ss += a[i] * a[i] + b[i] * b[i];
    }
  }
  const T* w = reinterpret_cast<const T*>(kind == 0 ? p.qw : p.kw);
  float r = 1.f;
  if (kind < 2 && w) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    r = rsqrtf(ss / (float)p.D + p.eps);
  }
  if (kind == 0 ? tok.b < 0 && !p.zero_tail : !tok.keep) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = lane + 32 * i;
    if (e < p.D / 2) {
      const int ia = e < p.n_freq && !p.interleaved ? e : 2 * e;
      const int ib = e < p.n_freq && !p.interleaved ? e + p.n_freq : ia + 1;
      float x = a[i], y = b[i];
      if (kind < 2) {
        if (w) {
          x *= r * (float)w[ia];
          y *= r * (float)w[ib];
        }
        if (e < p.n_freq) {
          float c, s;
          nra_angle(tok.pos, p.inv_freq[e], c, s);
          const float u = x * c - y * s;
          y = y * c + x * s;
          x = u;
        }
      }
      if (kind == 0 && tok.b < 0) x = y = 0.f;
      dst[ia] = T(x);
      dst[ib] = T(y);
    }
  }
}

}  // namespace hokv
