// Rotary positions of queries and keys, and their RMS norm per head with the rotation in the same pass, with gradients:
//
//   y = rot(x * r * gamma),   r = (mean(x^2) + eps)^-1/2 over a head's dims (rotation alone: y = rot(x))
//   g = rot^T(dy),  dgamma = sum g x r,  h = g gamma,  dx = r (h - x r mean(h x r))
//
// rot turns pair i of the first 2n dims by position * freqs[i] and multiplies it by `scale`; the dims behind stay. It is
// linear, so its backward pass is the transposed rotation of the gradients alone; the norm's backward pass reads x again
// and takes r from it, as the row is in registers anyway.
//
// Bound: HBM (2 passes over the tensors per direction, 3 for the norm's backward pass). A team of lanes (the next power of
// two of hd / 8) keeps a token and walks over its heads, so that cosines and sines are computed once per token and not
// read from a table.
#include <cmath>

#include "train_common.cuh"

namespace {

using namespace ub::train;

constexpr int THREADS = 256;
constexpr int MAX_HD = 256;
constexpr int VEC = 8;

enum Mode { ROTATE = 0, NORM = 1, NORM_BACKWARD = 2 };

// CTAs per SM that the registers have to allow, and that are launched.
constexpr int resident(bool vectors, int elem, int mode) {
  return !vectors ? 2 : (mode == NORM_BACKWARD ? 3 : 4) - (elem == 4);
}

struct Side {  // q or k
  const void* x;   // input; backward: the output's gradient
  const void* x0;  // backward of the norm: the forward's input
  void* out;       // contiguous
  UnblendHeadStrides s, s0;
  const void* gamma;
  int heads;
};

struct Args {
  Side side[2];
  const void* freqs;
  const void* positions;
  const int* lens;
  float* part;  // backward of the norm: [gridDim.x][2 hd] sums for the weights' gradients, may be null
  long long pos_stride;  // of a sequence
  unsigned length, inner, items;
  int split;  // teams that share a token's heads
  int hd, pairs, half;
  float scale, eps, sign;
  bool f64, pos64, w_is_t;
};

// Cosine and sine of position p times a frequency, times scale. The frequency comes in turns, as the sum of two doubles,
// and the whole turns are taken off the product before anything is rounded to fp32: the error is that of the final
// functions for every integer below 2^53.
__device__ __forceinline__ void turn(double p, double2 f, float scale, float& c, float& s) {
  const double hi = p * f.x;
  const double lo = fma(p, f.y, fma(p, f.x, -hi));
  double t = (hi - rint(hi)) + lo;  // beyond 2^53 turns the low part has whole ones too
  t -= rint(t);
  sincospif(2.f * (float)t, &s, &c);
  c *= scale;
  s *= scale;
}

template <int G>
__device__ __forceinline__ float team_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Frequencies in turns, and the norm's weights in fp32 (1 without).
template <typename T, int MODE>
__device__ __forceinline__ void load_tables(const Args& a, double2* freqs, float (*gamma)[MAX_HD]) {
  for (int j = threadIdx.x; j < a.pairs; j += THREADS) {
    constexpr double HI = 0x1.45f306dc9c883p-3, LO = -0x1.6b01ec5417056p-57;  // 1 / (2 pi) as a sum
    const double f = a.f64 ? static_cast<const double*>(a.freqs)[j] : (double)static_cast<const float*>(a.freqs)[j];
    const double hi = f * HI;
    freqs[j] = make_double2(hi, fma(f, HI, -hi) + f * LO);
  }
  if constexpr (MODE != ROTATE) {
    for (int j = threadIdx.x; j < 2 * MAX_HD; j += THREADS) {
      const int k = j / MAX_HD, e = j % MAX_HD;
      const void* g = a.side[k].gamma;
      if (e < a.hd)
        gamma[k][e] = g == nullptr ? 1.f : a.w_is_t ? to_f(static_cast<const T*>(g)[e]) : static_cast<const float*>(g)[e];
    }
  }
  __syncthreads();
}

// Where a team's work item lies.
struct Token {
  unsigned token, o, i, l;
  int part;
  bool active, inside;
  double p;

  __device__ __forceinline__ Token(const Args& a, unsigned item) {
    active = item < a.items;
    token = active ? item / (unsigned)a.split : 0;
    part = active ? (int)(item - token * a.split) : 0;
    const unsigned seq = token / a.length;
    l = token - seq * a.length;
    o = seq / a.inner, i = seq - o * a.inner;
    inside = a.lens == nullptr || (int)l < a.lens[seq];
    p = (double)l;
    if (a.positions) {
      const long long at = seq * a.pos_stride + l;
      p = a.pos64 ? (double)static_cast<const long long*>(a.positions)[at]
                  : (double)static_cast<const int*>(a.positions)[at];
    }
  }
};

// ---------------------------------------------------------------------------------- rows of 8-element pieces

// A lane's four pairs (a, b) as packed fp32: A = (a0, a1), (a2, a3), B likewise.
struct Pairs {
  float2 A[2], B[2];
};

// Eight elements of a row in two groups of four at off0 and off1. Adjacent pairs: the groups follow one another for 16-bit
// types (one 16-byte access) and are half a row apart for fp32 (whole lines per access). Half layout: the groups are the
// pairs' first and second members, so that a pair is in one lane; behind the pairs they are consecutive.
template <typename T, bool HALF>
struct Piece {
  uint32_t w[2 * sizeof(T)];

  __device__ __forceinline__ void load(const T* row, int off0, int off1, bool on) {
    if constexpr (sizeof(T) == 4) {
      const uint4 u = on ? *reinterpret_cast<const uint4*>(row + off0) : make_uint4(0, 0, 0, 0);
      const uint4 v = on ? *reinterpret_cast<const uint4*>(row + off1) : make_uint4(0, 0, 0, 0);
      w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w, w[4] = v.x, w[5] = v.y, w[6] = v.z, w[7] = v.w;
    } else if constexpr (!HALF) {
      const uint4 u = on ? *reinterpret_cast<const uint4*>(row + off0) : make_uint4(0, 0, 0, 0);
      w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    } else {
      const uint2 u = on ? *reinterpret_cast<const uint2*>(row + off0) : make_uint2(0, 0);
      const uint2 v = on ? *reinterpret_cast<const uint2*>(row + off1) : make_uint2(0, 0);
      w[0] = u.x, w[1] = u.y, w[2] = v.x, w[3] = v.y;
    }
  }

  __device__ __forceinline__ void store(T* row, int off0, int off1) const {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<uint4*>(row + off0) = make_uint4(w[0], w[1], w[2], w[3]);
      *reinterpret_cast<uint4*>(row + off1) = make_uint4(w[4], w[5], w[6], w[7]);
    } else if constexpr (!HALF) {
      *reinterpret_cast<uint4*>(row + off0) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      *reinterpret_cast<uint2*>(row + off0) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(row + off1) = make_uint2(w[2], w[3]);
    }
  }

  __device__ __forceinline__ static float2 two(uint32_t u, __nv_bfloat16) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
  }
  __device__ __forceinline__ static float2 two(uint32_t u, __half) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
  __device__ __forceinline__ static uint32_t word(float x, float y, __nv_bfloat16) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&b);
  }
  __device__ __forceinline__ static uint32_t word(float x, float y, __half) {
    const __half2 b = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&b);
  }

  __device__ __forceinline__ Pairs get() const {
    Pairs r;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if constexpr (sizeof(T) == 4) {
        const float* f = reinterpret_cast<const float*>(w);
        if (HALF) {
          r.A[k] = make_float2(f[2 * k], f[2 * k + 1]);
          r.B[k] = make_float2(f[4 + 2 * k], f[5 + 2 * k]);
        } else {
          r.A[k] = make_float2(f[4 * k], f[4 * k + 2]);
          r.B[k] = make_float2(f[4 * k + 1], f[4 * k + 3]);
        }
      } else if (HALF) {
        r.A[k] = two(w[k], T());
        r.B[k] = two(w[2 + k], T());
      } else {
        const float2 u = two(w[2 * k], T()), v = two(w[2 * k + 1], T());
        r.A[k] = make_float2(u.x, v.x);
        r.B[k] = make_float2(u.y, v.y);
      }
    }
    return r;
  }

  __device__ __forceinline__ void set(const Pairs& r) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if constexpr (sizeof(T) == 4) {
        float* f = reinterpret_cast<float*>(w);
        if (HALF) {
          f[2 * k] = r.A[k].x, f[2 * k + 1] = r.A[k].y, f[4 + 2 * k] = r.B[k].x, f[5 + 2 * k] = r.B[k].y;
        } else {
          f[4 * k] = r.A[k].x, f[4 * k + 1] = r.B[k].x, f[4 * k + 2] = r.A[k].y, f[4 * k + 3] = r.B[k].y;
        }
      } else if (HALF) {
        w[k] = word(r.A[k].x, r.A[k].y, T());
        w[2 + k] = word(r.B[k].x, r.B[k].y, T());
      } else {
        w[2 * k] = word(r.A[k].x, r.B[k].x, T());
        w[2 * k + 1] = word(r.A[k].y, r.B[k].y, T());
      }
    }
  }
};

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 neg(float2 v) { return make_float2(-v.x, -v.y); }

// A lane's place in its row: its groups' offsets, and for pair j which one it is (-1: not turned).
template <typename T, bool HALF>
struct Place {
  int off0, off1, c;
  bool has;

  __device__ __forceinline__ Place(const Args& a, int lane) {
    c = lane;
    has = c * VEC < a.hd;
    if (HALF) {
      const int turned = a.pairs / 4;  // lanes with pairs
      off0 = c < turned ? 4 * c : 2 * a.pairs + VEC * (c - turned);
      off1 = c < turned ? a.pairs + 4 * c : off0 + 4;
    } else if (sizeof(T) == 4) {
      off0 = 4 * c, off1 = a.hd / 2 + 4 * c;
    } else {
      off0 = VEC * c, off1 = off0 + 4;
    }
  }
  // element that A (b = 0) or B (b = 1) holds of pair j
  __device__ __forceinline__ int element(int j, int b) const {
    if (HALF) return (b ? off1 : off0) + j;
    return (j < 2 ? off0 : off1 - 4) + 2 * j + b;
  }
  __device__ __forceinline__ int pair(const Args& a, int j) const {
    const int p = HALF ? 4 * c + j : element(j, 0) / 2;
    return has && p < a.pairs ? p : -1;
  }
};

__device__ __forceinline__ float& part_of(float2 (&v)[2], int j) { return j & 1 ? v[j >> 1].y : v[j >> 1].x; }

template <typename T, bool HALF, int G, int MODE>
struct Team {
  static constexpr int U = sizeof(T) == 4 || MODE == NORM_BACKWARD ? 2 : 4;  // heads in flight

  // One token's heads of one side. C, S: cosines and sines; NORM folds gamma into them for each side.
  static __device__ __forceinline__ void heads(const Args& a, const Side& sd, const Place<T, HALF>& at, const Token& t,
                                               const float2 (&C)[2], const float2 (&S)[2], unsigned turns,
                                               const float* gamma, Pairs& dgamma) {
    const T* x = static_cast<const T*>(sd.x) + (t.o * sd.s.outer + t.i * sd.s.inner + t.l * sd.s.row + t.part * sd.s.head);
    const long long x_step = sd.s.head * a.split;
    const T* x0 = nullptr;
    long long x0_step = 0;
    if constexpr (MODE == NORM_BACKWARD) {
      x0 = static_cast<const T*>(sd.x0) + (t.o * sd.s0.outer + t.i * sd.s0.inner + t.l * sd.s0.row + t.part * sd.s0.head);
      x0_step = sd.s0.head * a.split;
    }
    T* out = static_cast<T*>(sd.out) + ((long long)t.token * sd.heads + t.part) * a.hd;
    const int out_step = a.hd * a.split;
    Pairs gm;  // weights
    float2 CA[2], SA[2], CB[2], SB[2];
    if constexpr (MODE != ROTATE) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        part_of(gm.A, j) = at.has ? gamma[at.element(j, 0)] : 0.f;
        part_of(gm.B, j) = at.has ? gamma[at.element(j, 1)] : 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      CA[k] = MODE == NORM ? mul2(C[k], gm.A[k]) : C[k];
      CB[k] = MODE == NORM ? mul2(C[k], gm.B[k]) : C[k];
      SA[k] = MODE == NORM ? mul2(S[k], gm.A[k]) : S[k];
      SB[k] = neg(MODE == NORM ? mul2(S[k], gm.B[k]) : S[k]);
    }
    const float inv_hd = 1.f / (float)a.hd;
    const bool partial = 2 * a.pairs != a.hd;
    const bool reads = t.active && t.inside && at.has, writes = t.active && at.has;
    int left = sd.heads - t.part;
    for (int rounds = (sd.heads + U * a.split - 1) / (U * a.split); rounds > 0; --rounds) {  // the same for all parts
      Piece<T, HALF> r[U], r0[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool on = reads && u * a.split < left;
        r[u].load(x + u * x_step, at.off0, at.off1, on);
        if constexpr (MODE == NORM_BACKWARD) r0[u].load(x0 + u * x0_step, at.off0, at.off1, on);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const Pairs v = r[u].get();
        Pairs y;
        if constexpr (MODE == NORM) {
          float2 ss = mul2(v.A[0], v.A[0]);
          ss = ub::fma2(v.A[1], v.A[1], ss);
          ss = ub::fma2(v.B[0], v.B[0], ss);
          ss = ub::fma2(v.B[1], v.B[1], ss);
          const float2 rstd = both(rsqrtf(team_sum<G>(ss.x + ss.y) * inv_hd + a.eps));
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 A = mul2(v.A[k], rstd), B = mul2(v.B[k], rstd);
            y.A[k] = ub::fma2(SB[k], B, mul2(CA[k], A));
            y.B[k] = ub::fma2(SA[k], A, mul2(CB[k], B));
          }
        } else {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            y.A[k] = ub::fma2(SB[k], v.B[k], mul2(CA[k], v.A[k]));
            y.B[k] = ub::fma2(SA[k], v.A[k], mul2(CB[k], v.B[k]));
          }
          if (partial) {  // not 1 a - 0 b: b may be infinite
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (!(turns >> j & 1)) {
                Pairs w = v;
                part_of(y.A, j) = part_of(w.A, j);
                part_of(y.B, j) = part_of(w.B, j);
              }
          }
        }
        if constexpr (MODE == NORM_BACKWARD) {
          const Pairs w = r0[u].get(), g = y;
          float2 ss = both(0.f), dot = both(0.f);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            y.A[k] = mul2(g.A[k], gm.A[k]);
            y.B[k] = mul2(g.B[k], gm.B[k]);
            ss = ub::fma2(w.A[k], w.A[k], ss);
            dot = ub::fma2(y.A[k], w.A[k], dot);
            ss = ub::fma2(w.B[k], w.B[k], ss);
            dot = ub::fma2(y.B[k], w.B[k], dot);
          }
          const float rstd = rsqrtf(team_sum<G>(ss.x + ss.y) * inv_hd + a.eps);
          const float2 m = both(-team_sum<G>(dot.x + dot.y) * rstd * inv_hd);
          // Rows that do not count: not 0 * x r, as their r may be infinite.
          const float2 rs = both(rstd), live = both(t.active && t.inside && u * a.split < left ? rstd : 0.f);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            dgamma.A[k] = ub::fma2(g.A[k], mul2(w.A[k], live), dgamma.A[k]);
            dgamma.B[k] = ub::fma2(g.B[k], mul2(w.B[k], live), dgamma.B[k]);
            y.A[k] = mul2(rs, ub::fma2(mul2(w.A[k], rs), m, y.A[k]));
            y.B[k] = mul2(rs, ub::fma2(mul2(w.B[k], rs), m, y.B[k]));
          }
        }
        if (writes && u * a.split < left) {
          Piece<T, HALF> o;
          o.set(y);
          if (MODE != ROTATE && !t.inside) {
#pragma unroll
            for (int k = 0; k < (int)(2 * sizeof(T)); ++k) o.w[k] = 0;
          }
          o.store(out + u * out_step, at.off0, at.off1);
        }
      }
      x += U * x_step;
      if constexpr (MODE == NORM_BACKWARD) x0 += U * x0_step;
      out += U * out_step;
      left -= U * a.split;
    }
  }
};

template <typename T, bool HALF, int G, int MODE>
__global__ void __launch_bounds__(THREADS, resident(true, sizeof(T), MODE)) rotary_kernel(const __grid_constant__ Args a) {
  constexpr int TEAMS = THREADS / G;
  __shared__ double2 freqs[MAX_HD / 2];
  __shared__ float gamma[2][MODE != ROTATE ? MAX_HD : 1];
  __shared__ float red[MODE == NORM_BACKWARD ? THREADS * VEC : 1];
  load_tables<T, MODE>(a, freqs, reinterpret_cast<float (*)[MAX_HD]>(gamma));
  const Place<T, HALF> at(a, threadIdx.x % G);
  unsigned turns = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) turns |= at.pair(a, j) >= 0 ? 1u << j : 0u;
  Pairs d[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) d[0].A[k] = d[0].B[k] = d[1].A[k] = d[1].B[k] = both(0.f);

  for (long long base = (long long)blockIdx.x * TEAMS; base < a.items; base += (long long)gridDim.x * TEAMS) {
    const Token t(a, (unsigned)base + threadIdx.x / G);
    float2 C[2], S[2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float c = 1.f, s = 0.f;
      if (turns >> j & 1) turn(t.p, freqs[at.pair(a, j)], a.scale, c, s);
      part_of(C, j) = c;
      part_of(S, j) = s * a.sign;
    }
    Team<T, HALF, G, MODE>::heads(a, a.side[0], at, t, C, S, turns, gamma[0], d[0]);
    Team<T, HALF, G, MODE>::heads(a, a.side[1], at, t, C, S, turns, gamma[1], d[1]);
  }
  if constexpr (MODE == NORM_BACKWARD) {
    if (a.part == nullptr) return;
    const int team = threadIdx.x / G;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      __syncthreads();
      if (at.has) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          red[team * (G * VEC) + at.element(j, 0)] = part_of(d[k].A, j);
          red[team * (G * VEC) + at.element(j, 1)] = part_of(d[k].B, j);
        }
      }
      __syncthreads();
      for (int e = threadIdx.x; e < a.hd; e += THREADS) {
        float s = red[e];
#pragma unroll
        for (int y = 1; y < TEAMS; ++y) s += red[y * (G * VEC) + e];
        a.part[((long long)blockIdx.x * 2 + k) * a.hd + e] = s;
      }
    }
  }
}

// --------------------------------------------------------------------------------------------- any other row

// A warp per item; lane c holds elements c, c + 32, ... of a row and reads what stands across from them in their pairs.
template <typename T, int MODE>
__global__ void __launch_bounds__(THREADS) rotary_any_kernel(const __grid_constant__ Args a) {
  constexpr int WARPS = THREADS / 32;
  __shared__ double2 freqs[MAX_HD / 2];
  __shared__ float gamma[2][MODE != ROTATE ? MAX_HD : 1];
  __shared__ float red[MODE == NORM_BACKWARD ? THREADS * VEC : 1];
  load_tables<T, MODE>(a, freqs, reinterpret_cast<float (*)[MAX_HD]>(gamma));
  const int lane = threadIdx.x & 31;
  float d[2][VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) d[0][j] = d[1][j] = 0.f;
  const float inv_hd = 1.f / (float)a.hd;
  for (long long base = (long long)blockIdx.x * WARPS; base < a.items; base += (long long)gridDim.x * WARPS) {
    const Token t(a, (unsigned)base + threadIdx.x / 32);
    float c[VEC], s[VEC];
    int across[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int e = lane + 32 * j;
      c[j] = 1.f, s[j] = 0.f, across[j] = e;
      if (e < 2 * a.pairs) {
        const bool second = a.half ? e >= a.pairs : e & 1;
        across[j] = a.half ? (second ? e - a.pairs : e + a.pairs) : e ^ 1;
        turn(t.p, freqs[a.half ? (second ? e - a.pairs : e) : e >> 1], a.scale, c[j], s[j]);
        s[j] *= second ? a.sign : -a.sign;
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const Side& sd = a.side[k];
      const T* x = static_cast<const T*>(sd.x) + (t.o * sd.s.outer + t.i * sd.s.inner + t.l * sd.s.row);
      const T* x0 = static_cast<const T*>(sd.x0) + (t.o * sd.s0.outer + t.i * sd.s0.inner + t.l * sd.s0.row);
      T* out = static_cast<T*>(sd.out) + (long long)t.token * sd.heads * a.hd;
      for (int h = t.part; t.active && h < sd.heads; h += a.split) {  // the same for the whole warp
        float own[VEC], y[VEC], w[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int e = lane + 32 * j;
          const bool has = t.inside && e < a.hd;
          own[j] = has ? to_f(x[h * sd.s.head + e]) : 0.f;
          y[j] = has && across[j] != e ? to_f(x[h * sd.s.head + across[j]]) : 0.f;
          w[j] = MODE == NORM_BACKWARD && has ? to_f(x0[h * sd.s0.head + e]) : 0.f;
        }
        if constexpr (MODE == NORM) {
          float ss = 0.f;
#pragma unroll
          for (int j = 0; j < VEC; ++j) ss += own[j] * own[j];
          const float rstd = rsqrtf(team_sum<32>(ss) * inv_hd + a.eps);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const int e = lane + 32 * j;
            own[j] = e < a.hd ? own[j] * rstd * gamma[k][e] : 0.f;
            y[j] = across[j] != e ? y[j] * rstd * gamma[k][across[j]] : 0.f;
          }
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) y[j] = across[j] != lane + 32 * j ? c[j] * own[j] + s[j] * y[j] : own[j];
        if constexpr (MODE == NORM_BACKWARD) {
          float ss = 0.f, dot = 0.f, g[VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const int e = lane + 32 * j;
            g[j] = y[j];
            y[j] = e < a.hd ? g[j] * gamma[k][e] : 0.f;
            ss += w[j] * w[j];
            dot += y[j] * w[j];
          }
          const float rstd = rsqrtf(team_sum<32>(ss) * inv_hd + a.eps);
          const float m = team_sum<32>(dot) * rstd * inv_hd;
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float xhat = w[j] * rstd;
            d[k][j] += t.inside ? g[j] * xhat : 0.f;
            y[j] = rstd * (y[j] - xhat * m);
          }
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (lane + 32 * j < a.hd)
            out[(long long)h * a.hd + lane + 32 * j] = from_f<T>(MODE == ROTATE || t.inside ? y[j] : 0.f);
      }
    }
  }
  if constexpr (MODE == NORM_BACKWARD) {
    if (a.part == nullptr) return;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < VEC; ++j) red[(threadIdx.x >> 5) * (32 * VEC) + lane + 32 * j] = d[k][j];
      __syncthreads();
      for (int e = threadIdx.x; e < a.hd; e += THREADS) {
        float s = red[e];
#pragma unroll
        for (int y = 1; y < WARPS; ++y) s += red[y * (32 * VEC) + e];
        a.part[((long long)blockIdx.x * 2 + k) * a.hd + e] = s;
      }
    }
  }
}

// What a call launches: teams of G lanes, `split` of them to a token, `grid` CTAs.
struct Plan {
  bool vectors;
  int lanes, split;
  unsigned grid, items;
};

bool heads_ok(const UnblendHeadStrides& s, const void* x, const UnblendRotaryParams* p, int heads, int elem) {
  return aligned16(x) && (p->outer <= 1 || s.outer * elem % 16 == 0) && (p->inner <= 1 || s.inner * elem % 16 == 0) &&
         (p->length <= 1 || s.row * elem % 16 == 0) && (heads <= 1 || s.head * elem % 16 == 0);
}

// Enough teams for all SMs come first: a token's heads are divided among teams, which compute its cosines each for
// itself, until there are about 1024 threads per SM. Larger calls keep a token's heads together.
Plan make_plan(const UnblendRotaryParams* p, bool vectors, int mode) {
  Plan r;
  r.vectors = vectors;
  r.lanes = 32;
  if (vectors) {
    r.lanes = 4;
    while (r.lanes * VEC < p->hd) r.lanes *= 2;
  }
  const long long tokens = (long long)p->outer * p->inner * p->length;
  const int most = p->heads > p->k_heads ? p->heads : p->k_heads;
  long long split = (ub::kNumSMs * 1024LL + tokens * r.lanes - 1) / (tokens * r.lanes);
  if (split > most) split = most;
  r.split = (int)split;
  r.items = (unsigned)(tokens * split);
  const long long teams = THREADS / r.lanes, ctas = (r.items + teams - 1) / teams;
  const long long cap = ub::kNumSMs * resident(vectors, elem_size(p->dtype), mode);
  r.grid = (unsigned)(ctas < cap ? ctas : cap);
  return r;
}

bool params_ok(const UnblendRotaryParams* p) {
  if (!p || !known_type(p->dtype) || p->outer < 1 || p->inner < 1 || p->length < 1 || p->heads < 1 || p->k_heads < 0 ||
      p->hd < 1 || p->hd > MAX_HD || p->pairs < 0 || 2 * p->pairs > p->hd || (p->pairs > 0 && !p->freqs) ||
      !(std::fabs(p->scale) <= 3.402823466e38f))
    return false;
  const long long rows = (long long)p->outer * p->inner;
  const long long most = p->heads > p->k_heads ? p->heads : p->k_heads;
  return rows < (1LL << 31) && rows * p->length < (1LL << 31) && rows * p->length * most < (1LL << 31) &&
         (p->freqs == nullptr || reinterpret_cast<uintptr_t>(p->freqs) % (p->freqs_f64 ? 8 : 4) == 0) &&
         (p->positions == nullptr || reinterpret_cast<uintptr_t>(p->positions) % (p->positions_i64 ? 8 : 4) == 0);
}

template <typename T, bool HALF, int MODE>
int launch_lanes(const Args& a, const Plan& pl, cudaStream_t st) {
  switch (pl.lanes) {
    case 4: rotary_kernel<T, HALF, 4, MODE><<<pl.grid, THREADS, 0, st>>>(a); break;
    case 8: rotary_kernel<T, HALF, 8, MODE><<<pl.grid, THREADS, 0, st>>>(a); break;
    case 16: rotary_kernel<T, HALF, 16, MODE><<<pl.grid, THREADS, 0, st>>>(a); break;
    default: rotary_kernel<T, HALF, 32, MODE><<<pl.grid, THREADS, 0, st>>>(a); break;
  }
  UB_CHECK_LAUNCH();
  return 0;
}

template <typename T, int MODE>
int launch_layout(const Args& a, const Plan& pl, cudaStream_t st) {
  if (pl.vectors) return a.half ? launch_lanes<T, true, MODE>(a, pl, st) : launch_lanes<T, false, MODE>(a, pl, st);
  rotary_any_kernel<T, MODE><<<pl.grid, THREADS, 0, st>>>(a);
  UB_CHECK_LAUNCH();
  return 0;
}

template <int MODE>
int run(Args& a, const UnblendRotaryParams* p, const void* q, const void* k, const void* q0, const void* k0, void* qo,
        void* ko, bool inverse, Plan& pl, cudaStream_t st) {
  a.side[0] = Side{q, q0, qo, p->q, p->q0, MODE != ROTATE ? p->gamma_q : nullptr, p->heads};
  a.side[1] = Side{k, k0, ko, p->k, p->k0, MODE != ROTATE ? p->gamma_k : nullptr, p->k_heads};
  a.freqs = p->freqs;
  a.positions = p->positions;
  a.lens = MODE != ROTATE ? p->lens : nullptr;
  a.pos_stride = p->positions_stride;
  a.length = p->length;
  a.inner = p->inner;
  a.items = pl.items;
  a.split = pl.split;
  a.hd = p->hd;
  a.pairs = p->pairs;
  a.half = p->half;
  a.scale = p->scale;
  a.eps = p->eps;
  a.sign = inverse ? -1.f : 1.f;
  a.f64 = p->freqs_f64;
  a.pos64 = p->positions_i64;
  a.w_is_t = MODE != ROTATE && p->w_dtype == p->dtype && p->dtype != UNBLEND_F32;
  switch (p->dtype) {
    case UNBLEND_F32: return launch_layout<float, MODE>(a, pl, st);
    case UNBLEND_BF16: return launch_layout<__nv_bfloat16, MODE>(a, pl, st);
    default: return launch_layout<__half, MODE>(a, pl, st);
  }
}

// Whether every row is whole pieces of eight dims on 16-byte boundaries, half layouts four pairs at a time.
bool vectors_ok(const UnblendRotaryParams* p, const void* q, const void* k, const void* q0, const void* k0,
                const void* qo, const void* ko) {
  const int e = elem_size(p->dtype);
  if (p->hd % VEC || (p->half && p->pairs % 4)) return false;
  if (!heads_ok(p->q, q, p, p->heads, e) || !aligned16(qo) || (q0 && !heads_ok(p->q0, q0, p, p->heads, e)))
    return false;
  return p->k_heads == 0 ||
         (heads_ok(p->k, k, p, p->k_heads, e) && aligned16(ko) && (!k0 || heads_ok(p->k0, k0, p, p->k_heads, e)));
}

bool norm_ok(const UnblendRotaryParams* p) {
  return p->eps >= 0.f && (p->w_dtype == UNBLEND_F32 || p->w_dtype == p->dtype);
}

}  // namespace

extern "C" int unblend_rotary(const void* q, const void* k, void* q_out, void* k_out, const UnblendRotaryParams* p,
                              int inverse, void* stream) {
  UB_REQUIRE(params_ok(p) && q && q_out && (p->k_heads == 0 || (k && k_out)));
  Plan pl = make_plan(p, vectors_ok(p, q, k, nullptr, nullptr, q_out, k_out), ROTATE);
  Args a{};
  return run<ROTATE>(a, p, q, k, nullptr, nullptr, q_out, k_out, inverse, pl, ub::as_stream(stream));
}

extern "C" int unblend_qk_norm_rotary_forward(const void* q, const void* k, void* q_out, void* k_out,
                                              const UnblendRotaryParams* p, void* stream) {
  UB_REQUIRE(params_ok(p) && norm_ok(p) && q && q_out && (p->k_heads == 0 || (k && k_out)));
  Plan pl = make_plan(p, vectors_ok(p, q, k, nullptr, nullptr, q_out, k_out), NORM);
  Args a{};
  return run<NORM>(a, p, q, k, nullptr, nullptr, q_out, k_out, false, pl, ub::as_stream(stream));
}

extern "C" int unblend_qk_norm_rotary_grad_workspace(const UnblendRotaryParams* p, long long* bytes) {
  UB_REQUIRE(params_ok(p) && bytes);
  const unsigned a = make_plan(p, true, NORM_BACKWARD).grid, b = make_plan(p, false, NORM_BACKWARD).grid;  // alignment is not known here
  *bytes = (long long)(a > b ? a : b) * 2 * p->hd * (long long)sizeof(float);
  return 0;
}

extern "C" int unblend_qk_norm_rotary_backward(const void* dq, const void* dk, const void* q, const void* k,
                                               void* dq_out, void* dk_out, void* dgamma_q, void* dgamma_k, float* work,
                                               const UnblendRotaryParams* p, void* stream) {
  UB_REQUIRE(params_ok(p) && norm_ok(p) && dq && q && dq_out && (p->k_heads == 0 || (dk && k && dk_out)));
  UB_REQUIRE((dgamma_q == nullptr) == (dgamma_k == nullptr) && (dgamma_q == nullptr || work != nullptr));
  Plan pl = make_plan(p, vectors_ok(p, dq, dk, q, k, dq_out, dk_out), NORM_BACKWARD);
  Args a{};
  a.part = dgamma_q ? work : nullptr;
  cudaStream_t st = ub::as_stream(stream);
  const int rc = run<NORM_BACKWARD>(a, p, dq, dk, q, k, dq_out, dk_out, true, pl, st);
  if (rc || !dgamma_q) return rc;
  switch (p->w_dtype) {
    case UNBLEND_F32: return launch_column_sums<float>(work, pl.grid, p->hd, 2, dgamma_q, dgamma_k, st);
    case UNBLEND_BF16: return launch_column_sums<__nv_bfloat16>(work, pl.grid, p->hd, 2, dgamma_q, dgamma_k, st);
    default: return launch_column_sums<__half>(work, pl.grid, p->hd, 2, dgamma_q, dgamma_k, st);
  }
}
