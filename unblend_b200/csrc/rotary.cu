// Rotary positions of queries and keys, and their RMS norm per head with the rotation in the same pass, with gradients:
//
//   y = rot(x * r * gamma),   r = (mean(x^2) + eps)^-1/2 over a head's dims (rotation alone: y = rot(x))
//   g = rot^T(dy),  dgamma = sum g x r,  h = g gamma,  dx = r (h - x r mean(h x r))
//
// rot turns pair i of the first 2n dims by position * freqs[i] and multiplies it by `scale`; the dims behind stay. It is
// linear, so its backward pass is the transposed rotation of the gradients alone; the norm's backward pass reads x again
// and takes r from it, as the row is in registers anyway.
//
// Bound: HBM (2 passes over the tensors per direction, 3 for the norm's backward pass) for many heads per token; issue slots
// for few, as each token's angles and addresses are shared by fewer rows. A team of lanes (the next power of two of hd / 8)
// keeps a token and walks over its heads, so that cosines and sines are computed once per token and lane and not read from
// a table. Rows come through shared memory a batch of heads ahead (cp.async): with loads to registers alone too few bytes
// were in flight (norm, 801 x 62 x 16 heads of 64: 119 us a step, now 100). Pairs are kept whole in a lane and worked on two
// at a time in packed fp32; as single floats the arithmetic bound the kernels (142 us).
//
// Measured, bf16: 62 x 801 tokens x 16 heads of 64, rotation 29 us per direction (6.9 TB/s), norm 801 x 62 35 us forward
// (5.8 TB/s) and 57 us backward (5.4); 20018 x 40 heads of 128 in half layout 68 us (6.0 TB/s) and 111 us (5.5). Forward and
// backward of 3 x 16381 x 20 heads of 128, 64 dims turned, fp16: 174 us (5.8 TB/s). Rows that have to go through shared memory:
// 32000 x 32 heads of 128 with 25 pairs in half layout 304 us (3.5 TB/s). Others would lose by it: the first two of these cases
// 131 instead of 78 us and 206 instead of 100 (both directions), as elements are picked one by one.
#include <cmath>

#include "train_common.cuh"

namespace {

using namespace ub::train;

constexpr int THREADS = 256;
constexpr int MAX_HD = 256;
constexpr int VEC = 8;

enum Mode { ROTATE = 0, NORM = 1, NORM_BACKWARD = 2 };

// How a row comes into registers: ADJACENT and HALF pairs straight from memory, where a lane's pairs are whole 8- or 16-byte
// pieces of it; any other row by way of shared memory.
enum Layout { ADJACENT = 0, HALF = 1, STAGED = 2 };

// CTAs per SM that the registers have to allow, and that are launched.
constexpr int resident(int layout, int elem, int mode) {
  if (layout == STAGED) return mode == NORM_BACKWARD ? 2 : 3;
  return (mode == NORM_BACKWARD ? 3 : 4) - (elem == 4);
}

// Heads of a team in flight.
constexpr int batch(int layout, int elem, int mode) {
  const int most = layout == STAGED ? 2 : elem == 4 ? 2 : 4;
  return mode == NORM_BACKWARD ? most / 2 : most;
}

struct Side {  // q or k
  const void* x;   // input; backward: the output's gradient
  const void* x0;  // backward of the norm: the forward's input
  void* out;       // contiguous
  UnblendHeadStrides s, s0;
  const void* gamma;
  int heads;
  int rounds;  // of a team's batches, the same for all of a token's teams
};

// n / d for n < 2^31 without a division, as a product with a rounded-up reciprocal of 31 + l bits behind the point, where
// 2^l is the first power of two that is not below d:
//
//   m = floor(2^(31 + l) / d) + 1, so m d = 2^(31 + l) + e with 0 < e <= d <= 2^l, and
//   n m / 2^(31 + l) = n / d + (n e / 2^(31 + l)) / d
//
// The last term is below 1 / d, as n e < 2^31 2^l: it never reaches the next integer. m is below 2^32, because d is above
// 2^(l - 1) (m = 2^31 + 1 for powers of two). The upper half of 2 n m, which fits 64 bits, takes 32 of the 32 + l places.
struct Divisor {
  unsigned d, m, l;

  Divisor() = default;
  explicit Divisor(unsigned by) : d(by), l(0) {
    while ((1ull << l) < d) ++l;
    m = (unsigned)((1ull << (31 + l)) / d + 1);
  }
  __device__ __forceinline__ unsigned operator()(unsigned n) const { return __umulhi(2 * n, m) >> l; }
};

struct Args {
  Side side[2];
  const void* freqs;
  const void* positions;
  const int* lens;
  float* part;  // backward of the norm: [gridDim.x][2 hd] sums for the weights' gradients, may be null
  long long pos_stride;  // of a sequence
  Divisor length, inner, parts;  // parts: teams that share a token's heads
  unsigned items;
  int split;  // parts again
  int hd, pairs, half;
  float scale, eps, sign;
  bool f64, pos64, w_is_t, pieces;
};

// Cosine and sine of position p times a frequency, times scale. The frequency comes in turns, as the sum of two doubles,
// and the whole turns are taken off the product before anything is rounded to fp32: the error is that of the final
// functions for every integer below 2^53. 16-bit tensors take the hardware's functions, off by 2^-21 within half a turn:
// a 500th of what rounding the results to fp16 costs, and an eighth of the instructions.
template <typename T>
__device__ __forceinline__ void turn(double p, double2 f, float scale, float& c, float& s) {
  const double hi = p * f.x;
  const double lo = fma(p, f.y, fma(p, f.x, -hi));
  double t = (hi - rint(hi)) + lo;  // beyond 2^53 turns the low part has whole ones too
  t -= rint(t);
  if (sizeof(T) == 2)
    __sincosf(6.283185307f * (float)t, &s, &c);
  else
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
    token = active ? a.parts(item) : 0;
    part = active ? (int)(item - token * a.split) : 0;
    const unsigned seq = a.length(token);
    l = token - seq * a.length.d;
    o = a.inner(seq), i = seq - o * a.inner.d;
    inside = a.lens == nullptr || (int)l < a.lens[seq];
    p = (double)l;
    if (a.positions) {
      const long long at = seq * a.pos_stride + l;
      p = a.pos64 ? (double)static_cast<const long long*>(a.positions)[at]
                  : (double)static_cast<const int*>(a.positions)[at];
    }
  }
};

// A lane's four pairs (a, b) as packed fp32: A = (a0, a1), (a2, a3), B likewise.
struct Pairs {
  float2 A[2], B[2];
};

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 neg(float2 v) { return make_float2(-v.x, -v.y); }
__device__ __forceinline__ float& part_of(float2 (&v)[2], int j) { return j & 1 ? v[j >> 1].y : v[j >> 1].x; }

// A lane's place in its row. Its pairs are number 4 c + j of the row's; behind the turned ones they are two neighbours, so that
// hd / 2 of them (rounded up) make a row for any number of turned pairs. For ADJACENT and HALF they lie in two groups of four
// elements at off0 and off1: consecutive for 16-bit adjacent pairs (one 16-byte access), half a row apart for fp32 ones (whole
// lines per access), the pairs' first and second members for HALF.
template <typename T, int LAYOUT>
struct Place {
  int off0, off1, c;
  bool has;
  unsigned turned;  // bit j: pair j turns

  __device__ __forceinline__ Place(const Args& a, int lane) {
    c = lane;
    has = c * VEC < a.hd;
    off0 = VEC * c, off1 = off0 + 4;
    if (LAYOUT == HALF && 4 * c < a.pairs) off0 = 4 * c, off1 = a.pairs + 4 * c;
    if (LAYOUT == ADJACENT && sizeof(T) == 4) off0 = 4 * c, off1 = a.hd / 2 + 4 * c;
    turned = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (has && pair(a, j) < a.pairs) turned |= 1u << j;
  }
  __device__ __forceinline__ int pair(const Args& a, int j) const {
    if (LAYOUT == ADJACENT) return ((j < 2 ? off0 : off1 - 4) >> 1) + j;
    return 4 * c + j;
  }
  // element that A (b = 0) or B (b = 1) holds of pair j; STAGED: may be hd, behind a row of odd width
  __device__ __forceinline__ int element(const Args& a, int j, int b) const {
    if (LAYOUT == HALF) return (b ? off1 : off0) + j;
    if (LAYOUT == ADJACENT) return (j < 2 ? off0 : off1 - 4) + 2 * j + b;
    const int p = 4 * c + j;
    return a.half && p < a.pairs ? p + b * a.pairs : 2 * p + b;
  }
};

// Eight elements of a row as they lie in memory: groups of four at off0 and off1.
template <typename T, int LAYOUT>
struct Piece {
  uint32_t w[2 * sizeof(T)];

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
        if (LAYOUT == HALF) {
          r.A[k] = make_float2(f[2 * k], f[2 * k + 1]);
          r.B[k] = make_float2(f[4 + 2 * k], f[5 + 2 * k]);
        } else {
          r.A[k] = make_float2(f[4 * k], f[4 * k + 2]);
          r.B[k] = make_float2(f[4 * k + 1], f[4 * k + 3]);
        }
      } else if (LAYOUT == HALF) {
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
        if (LAYOUT == HALF) {
          f[2 * k] = r.A[k].x, f[2 * k + 1] = r.A[k].y, f[4 + 2 * k] = r.B[k].x, f[5 + 2 * k] = r.B[k].y;
        } else {
          f[4 * k] = r.A[k].x, f[4 * k + 1] = r.B[k].x, f[4 * k + 2] = r.A[k].y, f[4 * k + 3] = r.B[k].y;
        }
      } else if (LAYOUT == HALF) {
        w[k] = word(r.A[k].x, r.A[k].y, T());
        w[2 + k] = word(r.B[k].x, r.B[k].y, T());
      } else {
        w[2 * k] = word(r.A[k].x, r.B[k].x, T());
        w[2 * k + 1] = word(r.A[k].y, r.B[k].y, T());
      }
    }
  }

  __device__ __forceinline__ void store(T* row, int off0, int off1) const {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<uint4*>(row + off0) = make_uint4(w[0], w[1], w[2], w[3]);
      *reinterpret_cast<uint4*>(row + off1) = make_uint4(w[4], w[5], w[6], w[7]);
    } else if constexpr (LAYOUT == ADJACENT) {
      *reinterpret_cast<uint4*>(row + off0) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      *reinterpret_cast<uint2*>(row + off0) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(row + off1) = make_uint2(w[2], w[3]);
    }
  }

  // On its way to the thread's own place in shared memory, which no other thread reads: no barrier is needed. Not `on`: zeros.
  __device__ __forceinline__ static void fetch(uint32_t* to, const T* row, int off0, int off1, bool on) {
    const uint32_t dst = (uint32_t)__cvta_generic_to_shared(to);
    if constexpr (sizeof(T) == 4) {
      const int n = on ? 16 : 0;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(row + off0), "r"(n) : "memory");
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + THREADS * 16), "l"(row + off1), "r"(n)
                   : "memory");
    } else if constexpr (LAYOUT == ADJACENT) {
      const int n = on ? 16 : 0;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(row + off0), "r"(n) : "memory");
    } else {
      const int n = on ? 8 : 0;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(row + off0), "r"(n) : "memory");
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst + 8), "l"(row + off1), "r"(n) : "memory");
    }
  }
  __device__ __forceinline__ void read(const uint32_t* from) {
    const uint4 u = *reinterpret_cast<const uint4*>(from);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    if constexpr (sizeof(T) == 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(from + THREADS * 4);
      w[4] = v.x, w[5] = v.y, w[6] = v.z, w[7] = v.w;
    }
  }
};

// A row by way of shared memory, [G * VEC] elements for each team: in 16-byte pieces, asynchronously, where it lies on such
// boundaries, else element by element; zeros behind hd.
template <typename T, int G>
__device__ __forceinline__ void stage(T* buf, const T* row, int c, int hd, bool on, bool pieces) {
  if (pieces) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      const int e = (i * G + c) * (16 / (int)sizeof(T));
      const bool has = on && e < hd;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(buf + e)),
                   "l"(row + e), "r"(has ? 16 : 0)
                   : "memory");
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int e = i * G + c;
      buf[e] = on && e < hd ? row[e] : from_f<T>(0.f);
    }
  }
}
template <typename T, int G>
__device__ __forceinline__ void unstage(const T* buf, T* row, int c, int hd, bool pieces) {
  if (pieces) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      const int e = (i * G + c) * (16 / (int)sizeof(T));
      if (e < hd) *reinterpret_cast<uint4*>(row + e) = *reinterpret_cast<const uint4*>(buf + e);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int e = i * G + c;
      if (e < hd) row[e] = buf[e];
    }
  }
}

// What a team's arithmetic needs for one token and side: cosines and sines, for the norm's forward pass times gamma.
template <int MODE>
struct Factors {
  float2 CA[2], SA[2], CB[2], SB[2];
  Pairs gamma;
};

// 1 / sqrt(x); the function is off by two ulp, which fp32 results would show: one Newton step more for them.
template <typename T>
__device__ __forceinline__ float reciprocal_root(float x) {
  const float r = rsqrtf(x);
  if (sizeof(T) == 2 || !(x >= 1e-30f && x <= 1e30f)) return r;
  return fmaf(0.5f * r, fmaf(-x * r, r, 1.f), r);
}

// The arithmetic on a lane's pairs of one row: v the input (the output's gradient), w the forward's input for its gradient.
// live: whether the row counts for the weights' gradients.
template <typename T, int LAYOUT, int G, int MODE>
__device__ __forceinline__ Pairs compute(const Args& a, const Factors<MODE>& f, unsigned turned, float inv_hd, Pairs v,
                                         const Pairs& w, bool live, Pairs& dgamma) {
  Pairs y;
  // What does not turn is x, not 1 a - 0 b: b may be infinite.
  const auto keep = [&](Pairs x) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool turns = LAYOUT == HALF ? turned != 0 : turned >> j & 1;  // HALF: all of a lane's pairs or none
      part_of(y.A, j) = turns ? part_of(y.A, j) : part_of(x.A, j);
      part_of(y.B, j) = turns ? part_of(y.B, j) : part_of(x.B, j);
    }
  };
  if constexpr (MODE == NORM) {
    float2 ss = mul2(v.A[0], v.A[0]);
    ss = ub::fma2(v.A[1], v.A[1], ss);
    ss = ub::fma2(v.B[0], v.B[0], ss);
    ss = ub::fma2(v.B[1], v.B[1], ss);
    const float2 rstd = both(reciprocal_root<T>(team_sum<G>(ss.x + ss.y) * inv_hd + a.eps));
    Pairs x;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float2 A = mul2(v.A[k], rstd), B = mul2(v.B[k], rstd);
      x.A[k] = mul2(f.CA[k], A);
      x.B[k] = mul2(f.CB[k], B);
      y.A[k] = ub::fma2(f.SB[k], B, x.A[k]);
      y.B[k] = ub::fma2(f.SA[k], A, x.B[k]);
    }
    if (2 * a.pairs != a.hd) keep(x);
  } else {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      y.A[k] = ub::fma2(f.SB[k], v.B[k], mul2(f.CA[k], v.A[k]));
      y.B[k] = ub::fma2(f.SA[k], v.A[k], mul2(f.CB[k], v.B[k]));
    }
    if (2 * a.pairs != a.hd) keep(v);
  }
  if constexpr (MODE == NORM_BACKWARD) {
    const Pairs g = y;
    float2 ss = both(0.f), dot = both(0.f);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      y.A[k] = mul2(g.A[k], f.gamma.A[k]);
      y.B[k] = mul2(g.B[k], f.gamma.B[k]);
      ss = ub::fma2(w.A[k], w.A[k], ss);
      dot = ub::fma2(y.A[k], w.A[k], dot);
      ss = ub::fma2(w.B[k], w.B[k], ss);
      dot = ub::fma2(y.B[k], w.B[k], dot);
    }
    const float rstd = reciprocal_root<T>(team_sum<G>(ss.x + ss.y) * inv_hd + a.eps);
    const float2 m = both(-team_sum<G>(dot.x + dot.y) * rstd * inv_hd);
    // Rows that do not count: not 0 * x r, as their r may be infinite.
    const float2 rs = both(rstd), counts = both(live ? rstd : 0.f);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      dgamma.A[k] = ub::fma2(g.A[k], mul2(w.A[k], counts), dgamma.A[k]);
      dgamma.B[k] = ub::fma2(g.B[k], mul2(w.B[k], counts), dgamma.B[k]);
      y.A[k] = mul2(rs, ub::fma2(mul2(w.A[k], rs), m, y.A[k]));
      y.B[k] = mul2(rs, ub::fma2(mul2(w.B[k], rs), m, y.B[k]));
    }
  }
  return y;
}

// Where a team's rows of one side and token come from.
template <typename T, int MODE>
struct Source {
  const T *x, *x0;
  long long step, step0;  // to the team's next head
  int left;               // heads from the current one on
  bool on;

  __device__ __forceinline__ Source(const Args& a, const Side& sd, const Token& t) {
    x = static_cast<const T*>(sd.x) + (t.o * sd.s.outer + t.i * sd.s.inner + t.l * sd.s.row + t.part * sd.s.head);
    step = sd.s.head * a.split;
    x0 = nullptr, step0 = 0;
    if constexpr (MODE == NORM_BACKWARD) {
      x0 = static_cast<const T*>(sd.x0) + (t.o * sd.s0.outer + t.i * sd.s0.inner + t.l * sd.s0.row + t.part * sd.s0.head);
      step0 = sd.s0.head * a.split;
    }
    left = sd.heads - t.part;
    on = t.active && t.inside;
  }
};

template <typename T, int LAYOUT, int G, int MODE>
__global__ void __launch_bounds__(THREADS, resident(LAYOUT, sizeof(T), MODE)) rotary_kernel(
    const __grid_constant__ Args a) {
  constexpr int TEAMS = THREADS / G, U = batch(LAYOUT, sizeof(T), MODE), PIECES = MODE == NORM_BACKWARD ? 2 * U : U;
  constexpr int PIECE = THREADS * VEC * (int)sizeof(T) / 4;  // words of a piece of all threads
  __shared__ double2 freqs[MAX_HD / 2];
  __shared__ float gamma[2][MODE != ROTATE ? MAX_HD : 1];
  // Pieces on their way, in two halves; at the end the sums for the weights' gradients.
  __shared__ __align__(16) uint32_t ring[2 * PIECES * PIECE];
  static_assert(MODE != NORM_BACKWARD || sizeof(ring) >= THREADS * VEC * sizeof(float), "the sums use the ring");
  load_tables<T, MODE>(a, freqs, reinterpret_cast<float (*)[MAX_HD]>(gamma));
  const Place<T, LAYOUT> at(a, threadIdx.x % G);
  const float inv_hd = 1.f / (float)a.hd;
  Pairs d[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) d[0].A[k] = d[0].B[k] = d[1].A[k] = d[1].B[k] = both(0.f);

  float2 C[2], S[2];
  const auto factors = [&](int side) {
    Factors<MODE> f;
    if constexpr (MODE != ROTATE) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int ea = at.element(a, j, 0), eb = at.element(a, j, 1);
        part_of(f.gamma.A, j) = at.has && ea < a.hd ? gamma[side][ea] : 0.f;
        part_of(f.gamma.B, j) = at.has && eb < a.hd ? gamma[side][eb] : 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      f.CA[k] = MODE == NORM ? mul2(C[k], f.gamma.A[k]) : C[k];
      f.CB[k] = MODE == NORM ? mul2(C[k], f.gamma.B[k]) : C[k];
      f.SA[k] = MODE == NORM ? mul2(S[k], f.gamma.A[k]) : S[k];
      f.SB[k] = neg(MODE == NORM ? mul2(S[k], f.gamma.B[k]) : S[k]);
    }
    return f;
  };
  const auto cosines = [&](const Token& t) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float c = 1.f, s = 0.f;
      if (at.turned >> j & 1) turn<T>(t.p, freqs[at.pair(a, j)], a.scale, c, s);
      part_of(C, j) = c;
      part_of(S, j) = s * a.sign;
    }
  };

  const long long stride = (long long)gridDim.x * TEAMS;
  const int per_round = U * a.split;
  uint32_t* const mine = ring + threadIdx.x * 4;  // the thread's own pieces; STAGED: the team's rows
  T* const rows = reinterpret_cast<T*>(ring) + (threadIdx.x / G) * (G * VEC);
  constexpr int ROW = THREADS * VEC;  // elements from piece to piece
  int half = 0;
  const auto fetch = [&](Source<T, MODE>& s) {  // the next heads into the other half
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool on = s.on && u * a.split < s.left;
      const T* const x = s.x + u * s.step;  // behind the last head nothing is read from it
      [[maybe_unused]] const T* const x0 = s.x0 + u * s.step0;
      const int to = half * PIECES + u;
      if constexpr (LAYOUT == STAGED) {
        stage<T, G>(rows + to * ROW, x, at.c, a.hd, on, a.pieces);
        if constexpr (MODE == NORM_BACKWARD) stage<T, G>(rows + (to + U) * ROW, x0, at.c, a.hd, on, a.pieces);
      } else {
        const bool has = on && at.has;
        Piece<T, LAYOUT>::fetch(mine + to * PIECE, x, at.off0, at.off1, has);
        if constexpr (MODE == NORM_BACKWARD)
          Piece<T, LAYOUT>::fetch(mine + (to + U) * PIECE, x0, at.off0, at.off1, has);
      }
    }
    cp_commit();
    half ^= 1;
    s.x += U * s.step;
    if constexpr (MODE == NORM_BACKWARD) s.x0 += U * s.step0;
    s.left -= per_round;
  };
  // A lane's pairs of a row in flight. STAGED: elements behind hd are zeros (hd is below G * VEC where it is odd).
  const auto pairs = [&](int from) {
    if constexpr (LAYOUT == STAGED) {
      Pairs v;
      const T* const row = rows + from * ROW;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int ea = at.element(a, j, 0), eb = at.element(a, j, 1);
        part_of(v.A, j) = at.has ? to_f(row[ea]) : 0.f;
        part_of(v.B, j) = at.has ? to_f(row[eb]) : 0.f;
      }
      return v;
    } else {
      Piece<T, LAYOUT> r;
      r.read(mine + from * PIECE);
      return r.get();
    }
  };
  const auto zeros = [](Pairs& y) {
#pragma unroll
    for (int k = 0; k < 2; ++k) y.A[k] = y.B[k] = both(0.f);
  };

  long long base = (long long)blockIdx.x * TEAMS;
  Token t(a, (unsigned)base + threadIdx.x / G);
  Source<T, MODE> src(a, a.side[0], t);
  fetch(src);
  for (; base < a.items; base += stride) {
    cosines(t);
    const Token next(a, base + stride < a.items ? (unsigned)(base + stride) + threadIdx.x / G : a.items);
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const Side& sd = a.side[side];
      const Factors<MODE> f = factors(side);
      T* out = static_cast<T*>(sd.out) + ((long long)t.token * sd.heads + t.part) * a.hd;
      int left = sd.heads - t.part;
      for (int rounds = sd.rounds; rounds > 0; --rounds) {
        if (rounds == 1) {  // the next heads are the other side's, or the next token's
          if (side == 0 && a.side[1].heads > 0)
            src = Source<T, MODE>(a, a.side[1], t);
          else
            src = Source<T, MODE>(a, a.side[0], next);
        }
        fetch(src);
        cp_wait<1>();
        const int from = half * PIECES;
        if constexpr (LAYOUT == STAGED) {
          __syncwarp();
          Pairs v[U], w[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            v[u] = pairs(from + u);
            if constexpr (MODE == NORM_BACKWARD) w[u] = pairs(from + U + u);
          }
          __syncwarp();
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const bool row = t.active && u * a.split < left;
            Pairs y = compute<T, LAYOUT, G, MODE>(a, f, at.turned, inv_hd, v[u], w[u], row && t.inside, d[side]);
            if (MODE != ROTATE && !t.inside) zeros(y);
            T* const to = rows + (from + u) * ROW;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (at.has) {
                to[at.element(a, j, 0)] = from_f<T>(part_of(y.A, j));
                to[at.element(a, j, 1)] = from_f<T>(part_of(y.B, j));
              }
            }
          }
          __syncwarp();
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (t.active && u * a.split < left)
              unstage<T, G>(rows + (from + u) * ROW, out + (long long)u * a.split * a.hd, at.c, a.hd, a.pieces);
          __syncwarp();
        } else {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const Pairs v = pairs(from + u);
            Pairs w;
            if constexpr (MODE == NORM_BACKWARD) w = pairs(from + U + u);
            const bool row = t.active && u * a.split < left;
            Pairs y = compute<T, LAYOUT, G, MODE>(a, f, at.turned, inv_hd, v, w, row && t.inside, d[side]);
            if (row && at.has) {
              if (MODE != ROTATE && !t.inside) zeros(y);
              Piece<T, LAYOUT> r;
              r.set(y);
              r.store(out + (long long)u * a.split * a.hd, at.off0, at.off1);
            }
          }
        }
        out += (long long)per_round * a.hd;
        left -= per_round;
      }
    }
    t = next;
  }
  cp_wait<0>();
  if constexpr (MODE == NORM_BACKWARD) {
    if (a.part == nullptr) return;
    float* const red = reinterpret_cast<float*>(ring);
    const int team = threadIdx.x / G;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      __syncthreads();
      if (at.has) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          red[team * (G * VEC) + at.element(a, j, 0)] = part_of(d[k].A, j);
          red[team * (G * VEC) + at.element(a, j, 1)] = part_of(d[k].B, j);
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

// What a call launches: teams of G lanes, `split` of them to a token, `grid` CTAs.
struct Plan {
  int layout;
  bool pieces;  // STAGED: rows are whole 16-byte pieces
  int lanes, split;
  unsigned grid, items;
};

bool heads_ok(const UnblendHeadStrides& s, const void* x, const UnblendRotaryParams* p, int heads, int elem) {
  return aligned16(x) && (p->outer <= 1 || s.outer * elem % 16 == 0) && (p->inner <= 1 || s.inner * elem % 16 == 0) &&
         (p->length <= 1 || s.row * elem % 16 == 0) && (heads <= 1 || s.head * elem % 16 == 0);
}

// Enough teams for all SMs come first: a token's heads are divided among teams, which compute its cosines each for itself,
// until there are 256 threads per SM; larger calls keep a token's heads together. Both sides, a forward and a backward call waited
// for: 62 tokens x 16 heads of 64, fp32, divided 27 us, undivided 28; norm of 8058 padded tokens x 16 heads of 48, fp32, divided
// by three 41 us among other calls, undivided 37; 1025 tokens x 64 heads of 96 by way of shared memory (16 lanes: by three) 68,
// by ten 64.
Plan make_plan(const UnblendRotaryParams* p, bool aligned, int mode) {
  Plan r;
  r.pieces = aligned && p->hd % VEC == 0;
  r.layout = !r.pieces || (p->half && p->pairs % 4) ? STAGED : p->half ? HALF : ADJACENT;
  r.lanes = 4;
  while (r.lanes * VEC < p->hd) r.lanes *= 2;
  const long long tokens = (long long)p->outer * p->inner * p->length;
  const int most = p->heads > p->k_heads ? p->heads : p->k_heads;
  long long split = (ub::kNumSMs * 256LL + tokens * r.lanes - 1) / (tokens * r.lanes);
  if (split > most) split = most;
  r.split = (int)split;
  r.items = (unsigned)(tokens * split);
  const long long teams = THREADS / r.lanes, ctas = (r.items + teams - 1) / teams;
  const long long cap = ub::kNumSMs * resident(r.layout, elem_size(p->dtype), mode);
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

template <typename T, int LAYOUT, int MODE>
int launch_lanes(Args& a, const Plan& pl, cudaStream_t st) {
  const int per_round = batch(LAYOUT, sizeof(T), MODE) * pl.split;
  for (Side& s : a.side) s.rounds = (s.heads + per_round - 1) / per_round;
  switch (pl.lanes) {
    case 4: rotary_kernel<T, LAYOUT, 4, MODE><<<pl.grid, THREADS, 0, st>>>(a); break;
    case 8: rotary_kernel<T, LAYOUT, 8, MODE><<<pl.grid, THREADS, 0, st>>>(a); break;
    case 16: rotary_kernel<T, LAYOUT, 16, MODE><<<pl.grid, THREADS, 0, st>>>(a); break;
    default: rotary_kernel<T, LAYOUT, 32, MODE><<<pl.grid, THREADS, 0, st>>>(a); break;
  }
  UB_CHECK_LAUNCH();
  return 0;
}

template <typename T, int MODE>
int launch_layout(Args& a, const Plan& pl, cudaStream_t st) {
  switch (pl.layout) {
    case ADJACENT: return launch_lanes<T, ADJACENT, MODE>(a, pl, st);
    case HALF: return launch_lanes<T, HALF, MODE>(a, pl, st);
    default: return launch_lanes<T, STAGED, MODE>(a, pl, st);
  }
}

// Teams form the addresses of heads behind the last one too (and copy nothing from them), which have to be aligned like
// the others. The stride of a single head is used for nothing else and may be any number: 0 in its place.
UnblendHeadStrides steps(UnblendHeadStrides s, int heads) {
  if (heads <= 1) s.head = 0;
  return s;
}

template <int MODE>
int run(Args& a, const UnblendRotaryParams* p, const void* q, const void* k, const void* q0, const void* k0, void* qo,
        void* ko, bool inverse, Plan& pl, cudaStream_t st) {
  a.side[0] = Side{q, q0, qo, steps(p->q, p->heads), steps(p->q0, p->heads), MODE != ROTATE ? p->gamma_q : nullptr,
                   p->heads, 0};
  a.side[1] = Side{k, k0, ko, steps(p->k, p->k_heads), steps(p->k0, p->k_heads), MODE != ROTATE ? p->gamma_k : nullptr,
                   p->k_heads, 0};
  a.freqs = p->freqs;
  a.positions = p->positions;
  a.lens = MODE != ROTATE ? p->lens : nullptr;
  a.pos_stride = p->positions_stride;
  a.length = Divisor((unsigned)p->length);
  a.inner = Divisor((unsigned)p->inner);
  a.parts = Divisor((unsigned)pl.split);
  a.items = pl.items;
  a.split = pl.split;
  a.hd = p->hd;
  a.pairs = p->pairs;
  a.half = p->half;
  a.pieces = pl.pieces;
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

// Whether every row starts on a 16-byte boundary.
bool rows_aligned16(const UnblendRotaryParams* p, const void* q, const void* k, const void* q0, const void* k0,
                const void* qo, const void* ko) {
  const int e = elem_size(p->dtype);
  if (p->hd % VEC) return false;  // nor would the outputs' rows
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
  Plan pl = make_plan(p, rows_aligned16(p, q, k, nullptr, nullptr, q_out, k_out), ROTATE);
  Args a{};
  return run<ROTATE>(a, p, q, k, nullptr, nullptr, q_out, k_out, inverse, pl, ub::as_stream(stream));
}

extern "C" int unblend_qk_norm_rotary_forward(const void* q, const void* k, void* q_out, void* k_out,
                                              const UnblendRotaryParams* p, void* stream) {
  UB_REQUIRE(params_ok(p) && norm_ok(p) && q && q_out && (p->k_heads == 0 || (k && k_out)));
  Plan pl = make_plan(p, rows_aligned16(p, q, k, nullptr, nullptr, q_out, k_out), NORM);
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
  Plan pl = make_plan(p, rows_aligned16(p, dq, dk, q, k, dq_out, dk_out), NORM_BACKWARD);
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
