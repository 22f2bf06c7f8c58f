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
// the group.  The cosines of a token are formed once for all its heads.  The
// angle is formed in 64 bits as a fraction of a turn (a position of 10^6 times
// an fp32 frequency loses its phase in 32 bits); norms and products are fp32,
// rounded once at the store.
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
  int tokens;   // tokens of a block
  float eps, inv_dim;   // inv_dim: 1 / D
};

constexpr int NRA_THREADS = 256;
// 4 blocks of an SM (64 registers).  A 16K-token prompt of 32 + 2 x 8 heads of 128 dims, bf16 (403 MB): 78 us, 5.2 TB/s;
// 82 with 5 blocks (48 registers, spills), 84 to 110 with 2 to 4 rows of a group on their way and 4 to 2 blocks, 103 with
// a token's angles formed by each group that works on it; the same reads and writes without the arithmetic take 69.
// With addresses multiplied out for each row 79, and 4,196 tokens of 3 sequences 27.6 instead of 25.3.
constexpr int NRA_BLOCKS = 4;
constexpr int NRA_TOKENS = 8;   // most tokens of a block

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
  bool bad = false;   // a negative start
  if (p.cu) {
    b = nra_sequence(p.cu, p.n_seqs, t);
    if (b < p.n_seqs) {
      const int start = p.cu[b];
      i = t - start;
      bad = start < 0;
      if (b == 0 && i < 0) b = p.n_seqs;   // ahead of the first sequence
    }
  } else {
    b = t;
  }
  r.b = b < p.n_seqs ? b : -1;
  r.row = r.pos = 0;
  r.keep = false;
  if (r.b >= 0) {
    const int n = p.kv_len[b];
    r.row = n + i;
    r.keep = !bad && n >= 0 && i >= 0 && (int64_t)n + i < p.cap;
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

// Two pairs (a, b) turned by their angles: packed fp32.
__device__ __forceinline__ void turn2(float& a0, float& a1, float& b0, float& b1, float2 c, float2 s) {
  const float2 a = make_float2(a0, a1), b = make_float2(b0, b1);
  const float2 x = __ffma2_rn(b, make_float2(-s.x, -s.y), __fmul2_rn(a, c)), y = __ffma2_rn(a, s, __fmul2_rn(b, c));
  a0 = x.x; a1 = x.y; b0 = y.x; b1 = y.y;
}

// Two elements times their weights and the row's factor.
template <typename T>
__device__ __forceinline__ void scale2(float& x, float& y, T wx, T wy, float q) {
  const float2 r = __fmul2_rn(make_float2(x, y), __fmul2_rn(make_float2((float)wx, (float)wy), make_float2(q, q)));
  x = r.x; y = r.y;
}

template <typename T>
struct alignas(16) Vec8 {
  T x[8];
};
// 8 elements as they lie in memory, and as fp32.
template <typename T>
struct Raw8 {
  uint4 u[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ void nra_load8(const T* p, Raw8<T>& r) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.u[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
}
template <typename T>
__device__ __forceinline__ void nra_weight8(const T* p, Vec8<T>& w) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i)
    reinterpret_cast<uint4*>(&w)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
}
template <typename T>
__device__ __forceinline__ void nra_widen(const Raw8<T>& r, float (&f)[8]) {
  const Vec8<T> w = *reinterpret_cast<const Vec8<T>*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (float)w.x[i];
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

// Source of head row h of token t (q heads, then k, then v).
template <typename T>
__device__ __forceinline__ const T* nra_source(const NraP& p, int t, int h) {
  if (h < p.Hq) return reinterpret_cast<const T*>(p.q) + t * p.q_t + h * p.q_h;
  h -= p.Hq;
  if (h < p.Hkv) return reinterpret_cast<const T*>(p.k) + t * p.k_t + h * p.k_h;
  return reinterpret_cast<const T*>(p.v) + t * p.v_t + (h - p.Hkv) * p.v_h;
}
// Its destination; returns 0 for q, 1 for k, 2 for v.
template <typename T>
__device__ __forceinline__ int nra_target(const NraP& p, int t, int h, const NraTok& k, T*& dst) {
  if (h < p.Hq) {
    dst = reinterpret_cast<T*>(p.out) + t * p.out_t + h * p.out_h;
    return 0;
  }
  h -= p.Hq;
  const bool is_v = h >= p.Hkv;
  dst = is_v ? reinterpret_cast<T*>(p.vs) + k.b * p.vs_b + (h - p.Hkv) * p.vs_h + k.row * p.vs_t
             : reinterpret_cast<T*>(p.ks) + k.b * p.ks_b + h * p.ks_h + k.row * p.ks_t;
  return is_v ? 2 : 1;
}

// Vector form: D a multiple of 16, and of the rotated dims too unless
// interleaved.  A block takes p.tokens tokens with all their head rows: their
// slots, row addresses and angles once, through shared memory, then rows by
// groups of LPR lanes, the next row on its way while one is worked on.
template <typename T, int LPR>
__global__ void __launch_bounds__(NRA_THREADS, NRA_BLOCKS) k_norm_rotate(const NraP p) {
  constexpr int GROUPS = NRA_THREADS / LPR;
  __shared__ NraTok s_tok[NRA_TOKENS];
  __shared__ T* s_dst[NRA_TOKENS][3];          // the token's rows: of q, k and v
  __shared__ const T* s_src[NRA_TOKENS][3];
  __shared__ int64_t s_step[2][3];             // head strides: source, destination
  __shared__ __align__(16) float s_cos[NRA_TOKENS][128 + 8], s_sin[NRA_TOKENS][128 + 8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = threadIdx.x % LPR;
  const int t0 = (int)blockIdx.x * p.tokens, n_tok = min(p.tokens, p.T - t0);
  const int heads = p.Hq + 2 * p.Hkv;
  // this lane's chunks of 8: both halves of its pairs
  const int lr = p.interleaved ? 0 : p.n_freq / 8;   // lanes of the half-split rotation
  const bool on = l < p.D / 16;
  const int ca = l < lr ? l : 2 * lr + 2 * (l - lr), cb = l < lr ? l + lr : ca + 1;
  Raw8<T> next[2];
  int fk = 0, fh = threadIdx.x / LPR, kind = 0, head = 0;   // the next row: token, head row; kind and head of its own
  auto locate = [&]() __attribute__((always_inline)) {
    while (fh >= heads) fh -= heads, ++fk;
    kind = (fh >= p.Hq) + (fh >= p.Hq + p.Hkv);
    head = fh - (kind > 0 ? p.Hq : 0) - (kind > 1 ? p.Hkv : 0);
  };
  locate();
  if (on && fk < n_tok) {
    const T* src = nra_source<T>(p, t0 + fk, fh);
    nra_load8(src + ca * 8, next[0]);
    nra_load8(src + cb * 8, next[1]);
  }
  if (warp < n_tok) {
    const NraTok k = nra_token(p, t0 + warp);
    const int64_t t = t0 + warp;
    if (lane == 0) {
      s_tok[warp] = k;
      s_src[warp][0] = reinterpret_cast<const T*>(p.q) + t * p.q_t;
      s_src[warp][1] = reinterpret_cast<const T*>(p.k) + t * p.k_t;
      s_src[warp][2] = reinterpret_cast<const T*>(p.v) + t * p.v_t;
      s_dst[warp][0] = reinterpret_cast<T*>(p.out) + t * p.out_t;
      s_dst[warp][1] = reinterpret_cast<T*>(p.ks) + (k.keep ? k.b * p.ks_b + k.row * p.ks_t : 0);
      s_dst[warp][2] = reinterpret_cast<T*>(p.vs) + (k.keep ? k.b * p.vs_b + k.row * p.vs_t : 0);
    }
  }
  if (threadIdx.x == 0) {
    s_step[0][0] = p.q_h; s_step[0][1] = p.k_h; s_step[0][2] = p.v_h;
    s_step[1][0] = p.out_h; s_step[1][1] = p.ks_h; s_step[1][2] = p.vs_h;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < n_tok * p.n_freq; e += NRA_THREADS) {
    const int k = e / p.n_freq, f = e - k * p.n_freq;
    nra_angle(s_tok[k].pos, p.inv_freq[f], s_cos[k][f], s_sin[k][f]);
  }
  __syncthreads();
  const unsigned mask = LPR == 32 ? 0xffffffffu : ((1u << LPR) - 1u) << (lane / LPR * LPR);
#pragma unroll 1
  while (fk < n_tok) {
    float a[8], b[8];
    nra_widen(next[0], a);
    nra_widen(next[1], b);
    const int k = fk, row_kind = kind;
    const NraTok tok = s_tok[k];
    T* dst = s_dst[k][kind] + head * s_step[1][kind];
    fh += GROUPS;
    locate();
    if (on && fk < n_tok) {
      const T* src = s_src[fk][kind] + head * s_step[0][kind];
      nra_load8(src + ca * 8, next[0]);
      nra_load8(src + cb * 8, next[1]);
    }
    if (row_kind < 2) {
      const T* w = reinterpret_cast<const T*>(row_kind == 0 ? p.qw : p.kw);
      if (w) {   // uniform over the group: its lanes share the row
        float ss = 0.f;
        if (on) {
          float2 s2 = make_float2(0.f, 0.f), r2 = s2;
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            s2 = __ffma2_rn(make_float2(a[j], a[j + 1]), make_float2(a[j], a[j + 1]), s2);
            r2 = __ffma2_rn(make_float2(b[j], b[j + 1]), make_float2(b[j], b[j + 1]), r2);
          }
          s2 = __fadd2_rn(s2, r2);
          ss = s2.x + s2.y;
        }
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
        const float q = rsqrtf(ss * p.inv_dim + p.eps);
        if (on) {
          Vec8<T> wa, wb;
          nra_weight8(w + ca * 8, wa);
          nra_weight8(w + cb * 8, wb);
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            scale2(a[j], a[j + 1], wa.x[j], wa.x[j + 1], q);
            scale2(b[j], b[j + 1], wb.x[j], wb.x[j + 1], q);
          }
        }
      }
      const float *cos = &s_cos[k][8 * l], *sin = &s_sin[k][8 * l];
      if (p.interleaved) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (8 * l + j < p.n_freq) {
            const float x = a[2 * j], y = a[2 * j + 1];
            a[2 * j] = x * cos[j] - y * sin[j];
            a[2 * j + 1] = y * cos[j] + x * sin[j];
          }
          if (8 * l + 4 + j < p.n_freq) {
            const float x = b[2 * j], y = b[2 * j + 1];
            b[2 * j] = x * cos[j + 4] - y * sin[j + 4];
            b[2 * j + 1] = y * cos[j + 4] + x * sin[j + 4];
          }
        }
      } else if (l < lr) {
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          const float4 c = *reinterpret_cast<const float4*>(cos + j), d = *reinterpret_cast<const float4*>(sin + j);
          turn2(a[j], a[j + 1], b[j], b[j + 1], make_float2(c.x, c.y), make_float2(d.x, d.y));
          turn2(a[j + 2], a[j + 3], b[j + 2], b[j + 3], make_float2(c.z, c.w), make_float2(d.z, d.w));
        }
      }
      if (row_kind == 0 && tok.b < 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = b[j] = 0.f;
      }
    }
    if (on && (row_kind == 0 ? tok.b >= 0 || p.zero_tail : tok.keep)) {
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
  const T* src = nra_source<T>(p, t, h);
  T* dst;
  const int kind = nra_target<T>(p, t, h, tok, dst);
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
    r = rsqrtf(ss * p.inv_dim + p.eps);
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
