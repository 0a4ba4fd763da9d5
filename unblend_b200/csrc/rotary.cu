// Rotary positions of queries and keys, and their RMS norm per head with the rotation in the same pass, with gradients:
//
//   y = rot(x * r * gamma),   r = (mean(x^2) + eps)^-1/2 over a head's dims (rotation alone: y = rot(x))
//   g = rot^T(dy),  dgamma = sum g x r,  h = g gamma,  dx = r (h - x r mean(h x r))
//
// rot turns pair i of the first 2n dims by position * freqs[i] and multiplies it by `scale`; the dims behind stay. It is
// linear, so its backward pass is the transposed rotation of the gradients alone; the norm's backward pass reads x again
// and takes r from it, as the row is in registers anyway.
//
// Bound: HBM (2 passes over the tensors per direction, 3 for the norm's backward pass). Eight dims per lane, a head's
// row on the next power of two of lanes (a team), sums over a row by shuffles within the team. A team keeps a token and
// walks over its heads, so that cosines and sines are computed once per token and chunk instead of read from a table.
#include <cmath>

#include "train_common.cuh"

namespace {

using namespace ub::train;

constexpr int THREADS = 256;
constexpr int MAX_HD = 256;
constexpr int VEC = 8;

enum Layout { PAIRS_ADJACENT = 0, PAIRS_HALF = 1, ANY = 2 };

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
  unsigned tokens, length, inner, items;
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

template <typename T>
struct Raw {
  uint4 w[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ void load_raw(Raw<T>& r, const T* p, bool on) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i)
    r.w[i] = on ? reinterpret_cast<const uint4*>(p)[i] : make_uint4(0, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ void unpack(const Raw<T>& r, float (&v)[VEC]) {
  constexpr int N = 16 / (int)sizeof(T);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
    float2 u[N / 2];
    unpack16(r.w[i], u, T());
#pragma unroll
    for (int j = 0; j < N / 2; ++j) v[i * N + 2 * j] = u[j].x, v[i * N + 2 * j + 1] = u[j].y;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[VEC]) {
  store_vec<T, VEC>(p, v);
}

template <typename T>
__device__ __forceinline__ Raw<T> shuffled(const Raw<T>& r, int lane) {
  Raw<T> o;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
    o.w[i].x = __shfl_sync(0xffffffffu, r.w[i].x, lane);
    o.w[i].y = __shfl_sync(0xffffffffu, r.w[i].y, lane);
    o.w[i].z = __shfl_sync(0xffffffffu, r.w[i].z, lane);
    o.w[i].w = __shfl_sync(0xffffffffu, r.w[i].w, lane);
  }
  return o;
}

// What a lane holds of a row: elements at(0) .. at(7), those below hd.
template <int LAYOUT>
struct Place {
  int lane, first, hd;  // lane of the warp; first element

  __device__ __forceinline__ int at(int j) const { return LAYOUT == ANY ? first + 32 * j : first + j; }
  __device__ __forceinline__ bool has(int j) const { return LAYOUT == ANY ? first + 32 * j < hd : first < hd; }
};

// The rotation of a lane's elements of one token: y = c own + s other, for elements with `turns`.
template <int LAYOUT>
struct Rotation {
  static constexpr int N = LAYOUT == PAIRS_ADJACENT ? VEC / 2 : VEC;
  float c[N], s[N];
  unsigned turns;  // bit j: element (adjacent pairs: pair) j is turned
  int other;       // lane that holds the other halves (PAIRS_HALF)

  __device__ __forceinline__ void make(const Args& a, const Place<LAYOUT>& at, const double2* freqs, double p) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      int pair;
      float sign = a.sign;
      if (LAYOUT == PAIRS_ADJACENT) {
        pair = at.first / 2 + j;
      } else {
        const int e = at.at(j);
        if (LAYOUT == ANY && !a.half) {
          pair = e >> 1;
          if (!(e & 1)) sign = -sign;
        } else {
          pair = e < a.pairs ? e : e - a.pairs;
          if (e < a.pairs) sign = -sign;
        }
      }
      if (turns >> j & 1) {
        turn(p, freqs[pair], a.scale, c[j], s[j]);
        s[j] *= sign;
      } else {
        c[j] = 1.f;
        s[j] = 0.f;
      }
    }
  }

  __device__ __forceinline__ void apply(const float (&own)[VEC], const float (&oth)[VEC], float (&y)[VEC]) const {
    if constexpr (LAYOUT == PAIRS_ADJACENT) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const bool on = turns >> j & 1;
        const float u = own[2 * j], v = own[2 * j + 1];
        y[2 * j] = on ? c[j] * u - s[j] * v : u;
        y[2 * j + 1] = on ? s[j] * u + c[j] * v : v;
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) y[j] = turns >> j & 1 ? c[j] * own[j] + s[j] * oth[j] : own[j];
    }
  }
};

template <int G>
__device__ __forceinline__ float team_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A lane's elements of one row and what stands across from them in their pairs.
template <typename T, int LAYOUT>
struct Row {
  Raw<T> raw;
  float own[LAYOUT == ANY ? VEC : 1], oth[LAYOUT == ANY ? VEC : 1];

  // base: the row's first element
  __device__ __forceinline__ void load(const Args& a, const Place<LAYOUT>& at, const T* base, bool on, bool others) {
    if constexpr (LAYOUT == ANY) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int e = at.at(j);
        const bool has = on && at.has(j);
        own[j] = has ? to_f(base[e]) : 0.f;
        if (others) {
          const int o = !a.half ? e ^ 1 : e < a.pairs ? e + a.pairs : e - a.pairs;
          oth[j] = has && e < 2 * a.pairs ? to_f(base[o]) : 0.f;
        }
      }
    } else {
      load_raw(raw, base + at.first, on && at.has(0));
    }
  }

  __device__ __forceinline__ void get(const Rotation<LAYOUT>& r, float (&x)[VEC], float (&y)[VEC], bool others) const {
    if constexpr (LAYOUT == ANY) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        x[j] = own[j];
        if (others) y[j] = oth[j];
      }
    } else {
      unpack(raw, x);
      if (LAYOUT == PAIRS_HALF && others) unpack(shuffled(raw, r.other), y);
    }
  }
};

template <typename T, int LAYOUT>
__device__ __forceinline__ void put(const Place<LAYOUT>& at, T* base, const float (&v)[VEC], bool on) {
  if constexpr (LAYOUT == ANY) {
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (on && at.has(j)) base[at.at(j)] = from_f<T>(v[j]);
  } else {
    if (on && at.has(0)) store8(base + at.first, v);
  }
}

// What stands across from element e in its pair (e itself behind the pairs).
__device__ __forceinline__ int across(const Args& a, int e) {
  if (e >= 2 * a.pairs) return e;
  return !a.half ? e ^ 1 : e < a.pairs ? e + a.pairs : e - a.pairs;
}

// One token's heads of one side. U heads are in flight.
template <typename T, int LAYOUT, int G, bool NORM, bool BWD, int U>
__device__ __forceinline__ void heads_of(const Args& a, const Side& sd, const Place<LAYOUT>& at,
                                         const Rotation<LAYOUT>& rot, const float* gamma, unsigned token, unsigned o,
                                         unsigned i, unsigned l, int part, bool active, bool inside,
                                         float (&dgamma)[VEC]) {
  const T* x = static_cast<const T*>(sd.x) + (o * sd.s.outer + i * sd.s.inner + l * sd.s.row);
  const T* x0 = nullptr;
  if constexpr (BWD && NORM) x0 = static_cast<const T*>(sd.x0) + (o * sd.s0.outer + i * sd.s0.inner + l * sd.s0.row);
  T* out = static_cast<T*>(sd.out) + (long long)token * sd.heads * a.hd;
  const bool others = !NORM || BWD || LAYOUT == PAIRS_HALF || LAYOUT == ANY;
  float go[VEC], gx[VEC];
  if constexpr (NORM) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int e = at.has(j) ? at.at(j) : 0;
      go[j] = at.has(j) ? gamma[e] : 0.f;
      if (!BWD && LAYOUT != PAIRS_ADJACENT) gx[j] = gamma[across(a, e)];
    }
  }
  const float inv_hd = 1.f / (float)a.hd;
  for (int h0 = part; h0 < sd.heads + part; h0 += U * a.split) {  // the same number of rounds for all parts
    Row<T, LAYOUT> r[U], r0[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * a.split;
      const bool on = active && inside && h < sd.heads;
      r[u].load(a, at, x + h * sd.s.head, on, others);
      if constexpr (BWD && NORM) r0[u].load(a, at, x0 + h * sd.s0.head, on, false);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * a.split;
      float own[VEC], oth[VEC], y[VEC];
      r[u].get(rot, own, oth, others);
      if constexpr (!NORM) {
        rot.apply(own, oth, y);
      } else if constexpr (!BWD) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) ss += own[j] * own[j];
        ss = team_sum<G>(ss);
        const float rstd = rsqrtf(ss * inv_hd + a.eps);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          own[j] = own[j] * rstd * go[j];
          if (LAYOUT != PAIRS_ADJACENT) oth[j] = oth[j] * rstd * gx[j];
        }
        rot.apply(own, oth, y);
      } else {
        float g[VEC], v[VEC];
        rot.apply(own, oth, g);
        r0[u].get(rot, v, oth, false);
        float ss = 0.f, dot = 0.f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          ss += v[j] * v[j];
          y[j] = g[j] * go[j];
          dot += y[j] * v[j];
        }
        ss = team_sum<G>(ss);
        dot = team_sum<G>(dot);
        const float rstd = rsqrtf(ss * inv_hd + a.eps);
        const float m = dot * rstd * inv_hd;
        const bool live = inside && active && h < sd.heads;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float xhat = v[j] * rstd;
          dgamma[j] += live ? g[j] * xhat : 0.f;  // not 0 * x: rows that do not count may have an r of infinity
          y[j] = rstd * (y[j] - xhat * m);
        }
      }
      if (!inside) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) y[j] = 0.f;
      }
      put<T, LAYOUT>(at, out + (long long)h * a.hd, y, active && h < sd.heads);
    }
  }
}

template <typename T, int LAYOUT, int G, bool NORM, bool BWD>
__global__ void __launch_bounds__(THREADS) rotary_kernel(const __grid_constant__ Args a) {
  constexpr int TEAMS = THREADS / G;
  constexpr int U = BWD && NORM ? 2 : 4;
  __shared__ double2 freqs[MAX_HD / 2];
  __shared__ float gamma[NORM ? 2 : 1][NORM ? MAX_HD : 1];
  __shared__ float red[NORM && BWD ? THREADS * VEC : 1];
  for (int j = threadIdx.x; j < a.pairs; j += THREADS) {
    constexpr double HI = 0x1.45f306dc9c883p-3, LO = -0x1.6b01ec5417056p-57;  // 1 / (2 pi) as a sum
    const double f = a.f64 ? static_cast<const double*>(a.freqs)[j] : (double)static_cast<const float*>(a.freqs)[j];
    const double hi = f * HI;
    freqs[j] = make_double2(hi, fma(f, HI, -hi) + f * LO);
  }
  if constexpr (NORM) {
    for (int j = threadIdx.x; j < a.hd; j += THREADS)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const void* g = a.side[k].gamma;
        gamma[k][j] = g == nullptr ? 1.f : a.w_is_t ? to_f(static_cast<const T*>(g)[j]) : static_cast<const float*>(g)[j];
      }
  }
  __syncthreads();
  Place<LAYOUT> at;
  at.lane = threadIdx.x & 31;
  at.hd = a.hd;
  const int c = threadIdx.x % G;
  at.first = LAYOUT == ANY ? c : c * VEC;
  Rotation<LAYOUT> rot;
  rot.turns = 0;
#pragma unroll
  for (int j = 0; j < Rotation<LAYOUT>::N; ++j) {
    const int e = LAYOUT == PAIRS_ADJACENT ? at.first + 2 * j : at.at(j);
    if (at.has(j) && e < 2 * a.pairs) rot.turns |= 1u << j;
  }
  rot.other = at.lane;
  if (LAYOUT == PAIRS_HALF && rot.turns) rot.other += at.first < a.pairs ? a.pairs / VEC : -(a.pairs / VEC);
  float dq[VEC], dk[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) dq[j] = dk[j] = 0.f;

  for (long long base = (long long)blockIdx.x * TEAMS; base < a.items; base += (long long)gridDim.x * TEAMS) {
    const unsigned item = (unsigned)base + threadIdx.x / G;
    const bool active = item < a.items;
    const unsigned token = active ? item / a.split : 0;
    const int part = active ? item % a.split : 0;
    const unsigned seq = token / a.length, l = token - seq * a.length;
    const unsigned o = seq / a.inner, i = seq - o * a.inner;
    const bool inside = a.lens == nullptr || (int)l < a.lens[seq];
    double p = (double)l;
    if (a.positions) {
      const long long at_p = seq * a.pos_stride + l;
      p = a.pos64 ? (double)static_cast<const long long*>(a.positions)[at_p]
                  : (double)static_cast<const int*>(a.positions)[at_p];
    }
    rot.make(a, at, freqs, p);
    heads_of<T, LAYOUT, G, NORM, BWD, U>(a, a.side[0], at, rot, gamma[0], token, o, i, l, part, active, inside, dq);
    heads_of<T, LAYOUT, G, NORM, BWD, U>(a, a.side[1], at, rot, gamma[NORM ? 1 : 0], token, o, i, l, part, active,
                                         inside, dk);
  }
  if constexpr (NORM && BWD) {
    if (a.part == nullptr) return;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int team = threadIdx.x / G;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        red[team * (G * VEC) + (LAYOUT == ANY ? c + 32 * j : c * VEC + j)] = k ? dk[j] : dq[j];
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

// What a call launches: teams of G lanes, `split` of them to a token, `grid` CTAs.
struct Plan {
  int layout, lanes, split;
  unsigned grid, items;
};

bool heads_ok(const UnblendHeadStrides& s, const void* x, const UnblendRotaryParams* p, int heads, int elem) {
  return aligned16(x) && (p->outer <= 1 || s.outer * elem % 16 == 0) && (p->inner <= 1 || s.inner * elem % 16 == 0) &&
         (p->length <= 1 || s.row * elem % 16 == 0) && (heads <= 1 || s.head * elem % 16 == 0);
}

// Enough teams for all SMs come first: a token's heads are divided among teams, which compute its cosines each for
// itself, until there are about 1024 threads per SM. Larger calls keep a token's heads together.
Plan make_plan(const UnblendRotaryParams* p, bool vectors, bool sums) {
  Plan r;
  r.layout = !vectors ? ANY : p->half ? PAIRS_HALF : PAIRS_ADJACENT;
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
  const long long cap = ub::kNumSMs * (sums ? 4 : 8);
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

template <typename T, int LAYOUT, int G, bool NORM, bool BWD>
int launch(const Args& a, const Plan& pl, cudaStream_t st) {
  rotary_kernel<T, LAYOUT, G, NORM, BWD><<<pl.grid, THREADS, 0, st>>>(a);
  UB_CHECK_LAUNCH();
  return 0;
}

template <typename T, bool NORM, bool BWD>
int launch_layout(const Args& a, const Plan& pl, cudaStream_t st) {
  if (pl.layout == ANY) return launch<T, ANY, 32, NORM, BWD>(a, pl, st);
  const bool half = pl.layout == PAIRS_HALF;
  switch (pl.lanes) {
    case 4: return half ? launch<T, PAIRS_HALF, 4, NORM, BWD>(a, pl, st) : launch<T, PAIRS_ADJACENT, 4, NORM, BWD>(a, pl, st);
    case 8: return half ? launch<T, PAIRS_HALF, 8, NORM, BWD>(a, pl, st) : launch<T, PAIRS_ADJACENT, 8, NORM, BWD>(a, pl, st);
    case 16: return half ? launch<T, PAIRS_HALF, 16, NORM, BWD>(a, pl, st) : launch<T, PAIRS_ADJACENT, 16, NORM, BWD>(a, pl, st);
    default: return half ? launch<T, PAIRS_HALF, 32, NORM, BWD>(a, pl, st) : launch<T, PAIRS_ADJACENT, 32, NORM, BWD>(a, pl, st);
  }
}

template <bool NORM, bool BWD>
int run(Args& a, const UnblendRotaryParams* p, const void* q, const void* k, const void* q0, const void* k0, void* qo,
        void* ko, bool inverse, Plan& pl, cudaStream_t st) {
  a.side[0] = Side{q, q0, qo, p->q, p->q0, NORM ? p->gamma_q : nullptr, p->heads};
  a.side[1] = Side{k, k0, ko, p->k, p->k0, NORM ? p->gamma_k : nullptr, p->k_heads};
  a.freqs = p->freqs;
  a.positions = p->positions;
  a.lens = NORM ? p->lens : nullptr;
  a.pos_stride = p->positions_stride;
  a.tokens = (unsigned)((long long)p->outer * p->inner * p->length);
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
  a.w_is_t = NORM && p->w_dtype == p->dtype && p->dtype != UNBLEND_F32;
  switch (p->dtype) {
    case UNBLEND_F32: return launch_layout<float, NORM, BWD>(a, pl, st);
    case UNBLEND_BF16: return launch_layout<__nv_bfloat16, NORM, BWD>(a, pl, st);
    default: return launch_layout<__half, NORM, BWD>(a, pl, st);
  }
}

// Whether every row is whole 16-byte chunks of eight dims whose partners are in a chunk too.
bool vectors_ok(const UnblendRotaryParams* p, const void* q, const void* k, const void* q0, const void* k0,
                const void* qo, const void* ko) {
  const int e = elem_size(p->dtype);
  if (p->hd % VEC || (p->half && p->pairs % VEC)) return false;
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
  Plan pl = make_plan(p, vectors_ok(p, q, k, nullptr, nullptr, q_out, k_out), false);
  Args a{};
  return run<false, false>(a, p, q, k, nullptr, nullptr, q_out, k_out, inverse, pl, ub::as_stream(stream));
}

extern "C" int unblend_qk_norm_rotary_forward(const void* q, const void* k, void* q_out, void* k_out,
                                              const UnblendRotaryParams* p, void* stream) {
  UB_REQUIRE(params_ok(p) && norm_ok(p) && q && q_out && (p->k_heads == 0 || (k && k_out)));
  Plan pl = make_plan(p, vectors_ok(p, q, k, nullptr, nullptr, q_out, k_out), false);
  Args a{};
  return run<true, false>(a, p, q, k, nullptr, nullptr, q_out, k_out, false, pl, ub::as_stream(stream));
}

extern "C" int unblend_qk_norm_rotary_grad_workspace(const UnblendRotaryParams* p, long long* bytes) {
  UB_REQUIRE(params_ok(p) && bytes);
  const unsigned a = make_plan(p, true, true).grid, b = make_plan(p, false, true).grid;  // alignment is not known here
  *bytes = (long long)(a > b ? a : b) * 2 * p->hd * (long long)sizeof(float);
  return 0;
}

extern "C" int unblend_qk_norm_rotary_backward(const void* dq, const void* dk, const void* q, const void* k,
                                               void* dq_out, void* dk_out, void* dgamma_q, void* dgamma_k, float* work,
                                               const UnblendRotaryParams* p, void* stream) {
  UB_REQUIRE(params_ok(p) && norm_ok(p) && dq && q && dq_out && (p->k_heads == 0 || (dk && k && dk_out)));
  UB_REQUIRE((dgamma_q == nullptr) == (dgamma_k == nullptr) && (dgamma_q == nullptr || work != nullptr));
  Plan pl = make_plan(p, vectors_ok(p, dq, dk, q, k, dq_out, dk_out), dgamma_q != nullptr);
  Args a{};
  a.part = dgamma_q ? work : nullptr;
  cudaStream_t st = ub::as_stream(stream);
  const int rc = run<true, true>(a, p, dq, dk, q, k, dq_out, dk_out, true, pl, st);
  if (rc || !dgamma_q) return rc;
  switch (p->w_dtype) {
    case UNBLEND_F32: return launch_column_sums<float>(work, pl.grid, p->hd, 2, dgamma_q, dgamma_k, st);
    case UNBLEND_BF16: return launch_column_sums<__nv_bfloat16>(work, pl.grid, p->hd, 2, dgamma_q, dgamma_k, st);
    default: return launch_column_sums<__half>(work, pl.grid, p->hd, 2, dgamma_q, dgamma_k, st);
  }
}
