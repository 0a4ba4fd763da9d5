// An AdamW step over many tensors in one launch, its moments in fp32 or 8 bits, and the 2-norm of many tensors.
//
//   g' = c g,  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
//   p  = (1 - lr wd) p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// The moments of all tensors lie in one array each; every tensor starts at a block of 256 elements of its own. A warp
// takes a block at a time and finds its tensor in the table of the launch (kernel parameters: nothing is copied to the
// device, and a captured graph keeps them) by bisection.
//
// In 32 bits HBM bounds it: 28 bytes per fp32 element, 6.5 TB/s (134 M parameters in 675 tensors: 575 us). In 8 bits 10 + 1/16
// bytes per 16-bit element are few beside the codes' arithmetic, about 63 instructions per element of which half are the
// integer pipe's (118 M bf16 parameters: 297 us, 3.8 TB/s, issue slots 73 % and integer pipe 54 % busy; 509 us with scalar
// floats and 32-bit patterns for the codes). What helped: two floats, and two codes as bf16, per instruction; runs of
// consecutive blocks per warp, as the search took 10 instructions per element; the next block's loads ahead of a block's
// arithmetic. Handing out the values: 180 us for the same (6.2 TB/s).
//
// 8 bits: a block has two scales, the largest |m| and the largest u = sqrt(v). u is kept instead of v because its range is
// half as many octaves. Codes are small floats relative to the scale, whose largest code is 1: m has a sign, 3 bits of
// mantissa and 15.9 octaves, u 4 bits and 15.9 octaves. Both are the leading bits of the fp32 pattern, rounded to
// nearest even (a step is 2^-3, 2^-4 of the octave's start). An m below half the smallest magnitude is 0; a u that is not
// 0 never becomes 0, since the update divides by it. The update itself uses m and v before they are rounded. What decides
// a code is computed in fp32 one operation at a time (no fused multiply-add), so that the codes are defined bit for bit.
// A value that is not finite makes its block's scale infinite or NaN, and with it every moment of the block.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "train_common.cuh"

namespace {

using namespace ub::train;

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int BLOCK = 256;            // elements that share scales
// CTAs per SM that the registers allow: in 8 bits a warp has two blocks in flight, for fp32 tensors of twice the size (134 M fp32
// parameters with values: 616 us with two CTAs, 658 with three and spills).
constexpr int FULL_CTAS = 4;
constexpr int eight_ctas(int elem, int grad_elem) { return elem + grad_elem > 4 ? 2 : 3; }
constexpr int SMALL = 64, MIDDLE = 256, LARGE = 896;  // tensors of a launch: 2.3, 9 or 32 KB of kernel parameters

template <int N>
struct Table {
  UnblendAdamWTensor t[N];
  unsigned start[N];  // first of the launch's units of each tensor
  int count;
  unsigned total;
};

// The tensor that a unit belongs to.
template <int N>
__device__ __forceinline__ int tensor_of(const Table<N>& tab, unsigned unit) {
  int lo = 0, hi = tab.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (tab.start[mid] <= unit)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

struct StepArgs {
  void* m;
  void* v;
  float2* scales;
  const float* grad_scale;
  const long long* step;  // device: the bias corrections and factors below are computed from it
  const float* lr;        // device
  double b1d, b2d, lrd, wdd;
  float b1, c1, b2, c2, eps, one;
  unsigned run;  // consecutive blocks of a warp
  float decay, size, root;  // 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
};

// Codes travel two at a time as bf16: a code's value is the bf16 pattern (c + 889) << 4 for m and (c + 1777) << 3 for u (code
// 1 is 2^-16 * 1.25 and 2^-16 * 1.125), which the packed 16-bit pipes decode and zero with half the integer instructions that
// 32-bit patterns take; those had bound the kernel.
constexpr unsigned M_BIAS = (889u << 4) * 0x10001u, U_BIAS = (1777u << 3) * 0x10001u;
constexpr float M_ONE = 1.25f / 65536.f;

__device__ __forceinline__ __nv_bfloat162 as_bf2(unsigned w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
__device__ __forceinline__ unsigned as_word(__nv_bfloat162 h) { return *reinterpret_cast<unsigned*>(&h); }
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 wide(unsigned w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// The values of codes 2 I and 2 I + 1 of four, relative to their scale.
template <int I>
__device__ __forceinline__ float2 m_values(unsigned w) {
  const unsigned x = __byte_perm(w, 0, I ? 0x4342 : 0x4140), c = x & 0x007f007fu;
  const __nv_bfloat162 there = __hne2(as_bf2(c), as_bf2(0));  // 1 or 0
  return wide(as_word(__hmul2(as_bf2(c * 16u + M_BIAS), there)) | (x << 8 & 0x80008000u));
}
template <int I>
__device__ __forceinline__ float2 u_values(unsigned w) {
  const unsigned x = __byte_perm(w, 0, I ? 0x4342 : 0x4140);
  const __nv_bfloat162 there = __hne2(as_bf2(x), as_bf2(0));
  return wide(as_word(__hmul2(as_bf2(x * 8u + U_BIAS), there)));
}

// Rounds to BITS bits of mantissa (the leading one not counted) by Veltkamp's splitting (Dekker, "A floating-point technique
// for extending the available precision", 1971); in radix 2 and for these lengths that is to nearest even for every
// mantissa. `one` is a factor of 1 that the compiler does not know: it would fuse the product into the sums.
template <int BITS>
__device__ __forceinline__ float2 rounded(float2 r, float one) {
  const float2 p = mul2(r, both((float)(1 << (23 - BITS)) + 1.f));
  const float2 q = ub::fma2(p, both(-one), r);
  return ub::fma2(p, both(one), q);
}

// Upper halves of two patterns: the floats as bf16, cut off.
__device__ __forceinline__ unsigned upper(float2 v) {
  return __byte_perm(__float_as_uint(v.x), __float_as_uint(v.y), 0x7632);
}

// Codes of two values relative to their block's largest, in the upper bytes of the halves.
__device__ __forceinline__ unsigned m_codes(float2 r, float one) {
  float2 a = make_float2(fmaxf(fabsf(r.x), M_ONE), fmaxf(fabsf(r.y), M_ONE));
  a.x = fabsf(r.x) > 0.5f * M_ONE ? a.x : 0.f;
  a.y = fabsf(r.y) > 0.5f * M_ONE ? a.y : 0.f;
  const unsigned c = __vmaxu2(upper(rounded<3>(a, one)), M_BIAS) - M_BIAS;
  return c * 16u | (upper(r) & 0x80008000u);
}
// What is not 0 has code 1 or more (the mask looks at the bf16 pattern: above 2^-133 of the largest).
__device__ __forceinline__ unsigned u_codes(float2 r, float one) {
  const unsigned there = __hne2_mask(as_bf2(upper(r)), as_bf2(0));
  return (__vmaxu2(upper(rounded<4>(r, one)), U_BIAS + 0x00080008u) - U_BIAS & there) * 32u;
}

// Largest magnitude of three, NaN if one is.
__device__ __forceinline__ float top3(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 1 / x to within an ulp for normal x.
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// 1 / top, 0 for a block of zeros (or below the normal range, where 1 / top could overflow).
__device__ __forceinline__ float inverse(float top) { return top >= 1.17549435e-38f ? __frcp_rn(top) : 0.f; }

// What a lane holds of a block, as read: eight elements in two groups of four.
template <typename T>
struct Eight {
  alignas(16) T e[8];

  // `one`: the groups follow one another; full: the block is whole and p on a boundary of four elements (one: of eight)
  __device__ __forceinline__ void load(const T* p, int gap, bool one, bool full, int left) {
    if (full) {
      if (sizeof(T) == 2 && one) {
        *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(p);
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if constexpr (sizeof(T) == 2)
            *reinterpret_cast<uint2*>(e + 4 * j) = *reinterpret_cast<const uint2*>(p + j * gap);
          else
            *reinterpret_cast<uint4*>(e + 4 * j) = *reinterpret_cast<const uint4*>(p + j * gap);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = (i & 3) + (i >> 2) * gap;
        e[i] = at < left ? p[at] : from_f<T>(0.f);
      }
    }
  }
  __device__ __forceinline__ void store(T* p, int gap, bool one, bool full, int left) const {
    if (full) {
      if (sizeof(T) == 2 && one) {
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(e);
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if constexpr (sizeof(T) == 2)
            *reinterpret_cast<uint2*>(p + j * gap) = *reinterpret_cast<const uint2*>(e + 4 * j);
          else
            *reinterpret_cast<uint4*>(p + j * gap) = *reinterpret_cast<const uint4*>(e + 4 * j);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = (i & 3) + (i >> 2) * gap;
        if (at < left) p[at] = e[i];
      }
    }
  }
  __device__ __forceinline__ void get(float2 (&v)[4]) const {
    if constexpr (sizeof(T) == 2) {
      unpack16(*reinterpret_cast<const uint4*>(e), v, T());
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = make_float2(e[2 * i], e[2 * i + 1]);
    }
  }
  __device__ __forceinline__ void set(const float2 (&v)[4]) {
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(e) = pack16(v, T());
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) e[2 * i] = v[i].x, e[2 * i + 1] = v[i].y;
    }
  }
};

// Largest of non-negative values by their patterns: NaN is above infinity.
__device__ __forceinline__ float warp_top(float v) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v))); }

// A lane's part of a block of one tensor. In 8 bits its elements are consecutive for 16-bit tensors (accesses of 16 and 8
// bytes); otherwise two groups of four 128 elements apart (whole lines per access).
template <typename T, typename TG, bool EIGHT, int N>
struct Unit {
  static constexpr bool ONE = EIGHT && sizeof(T) == 2 && sizeof(TG) == 2;
  static constexpr int GAP = ONE ? 4 : 128;
  T* p;
  long long at;  // of the moments
  int left;      // elements of the tensor from the lane's first on
  bool full;
  Eight<T> param;
  Eight<TG> grad;
  unsigned mc[2], uc[2];  // 8 bits: codes and scales
  float2 scale;

  __device__ __forceinline__ void fetch(const Table<N>& tab, const StepArgs& a, int k, unsigned unit, int lane) {
    const long long local = unit - tab.start[k], n = tab.t[k].n - local * BLOCK;
    const int mine = lane * (ONE ? 8 : 4);
    p = static_cast<T*>(tab.t[k].param) + local * BLOCK;
    const TG* g = static_cast<const TG*>(tab.t[k].grad) + local * BLOCK;
    full = n >= BLOCK && reinterpret_cast<uintptr_t>(p) % ((ONE ? 8 : 4) * sizeof(T)) == 0 &&
           reinterpret_cast<uintptr_t>(g) % ((ONE ? 8 : 4) * sizeof(TG)) == 0;
    left = (int)min(n, (long long)BLOCK) - mine;
    p += mine;
    const long long block = tab.t[k].block + local;
    at = block * BLOCK + mine;
    if constexpr (EIGHT) {
      scale = a.scales[block];
      if constexpr (ONE) {
        const uint2 m = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.m) + at);
        const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.v) + at);
        mc[0] = m.x, mc[1] = m.y, uc[0] = u.x, uc[1] = u.y;
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          mc[j] = *reinterpret_cast<const unsigned*>(static_cast<const uint8_t*>(a.m) + at + j * GAP);
          uc[j] = *reinterpret_cast<const unsigned*>(static_cast<const uint8_t*>(a.v) + at + j * GAP);
        }
      }
    }
    param.load(p, GAP, ONE, full, left);
    grad.load(g + mine, GAP, ONE, full, left);
  }
};

struct Factors {
  float decay, size, root, grad;
};

// The update of a lane's part of a block.
template <typename T, typename TG, bool EIGHT, int N>
__device__ __forceinline__ void update(Unit<T, TG, EIGHT, N>& x, const StepArgs& a, const Factors& f, int lane) {
  using U = Unit<T, TG, EIGHT, N>;
  float2 pv[4], gv[4], mv[4], uv[4];  // uv: v, in 8 bits u as the codes are read
  if constexpr (EIGHT) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      mv[2 * j] = mul2(m_values<0>(x.mc[j]), both(x.scale.x));
      mv[2 * j + 1] = mul2(m_values<1>(x.mc[j]), both(x.scale.x));
      uv[2 * j] = mul2(u_values<0>(x.uc[j]), both(x.scale.y));
      uv[2 * j + 1] = mul2(u_values<1>(x.uc[j]), both(x.scale.y));
    }
  } else {
    Eight<float> w;
    w.load(static_cast<const float*>(a.m) + x.at, U::GAP, false, true, 0);
    w.get(mv);
    w.load(static_cast<const float*>(a.v) + x.at, U::GAP, false, true, 0);
    w.get(uv);
  }
  x.param.get(pv);
  x.grad.get(gv);
  // Sums as fma with the factor `one`: a packed product would be fused into them.
  const auto moments = [&](int i) {
    const float2 gr = mul2(gv[i], both(f.grad));
    mv[i] = ub::fma2(mul2(mv[i], both(a.b1)), both(a.one), mul2(gr, both(a.c1)));
    uv[i] = ub::fma2(mul2(uv[i], both(a.b2)), both(a.one), mul2(mul2(gr, gr), both(a.c2)));
  };
  const auto param = [&](int i, float2 u) {
    const float2 denom = ub::fma2(u, both(f.root), both(a.eps));
    const float2 step = mul2(mv[i], make_float2(reciprocal(denom.x), reciprocal(denom.y)));
    pv[i] = ub::fma2(step, both(-f.size), mul2(pv[i], both(f.decay)));
  };
  [[maybe_unused]] float top_m = 0.f, top_u = 0.f;
  [[maybe_unused]] float2 root_v[4];
  if constexpr (EIGHT) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uv[i] = mul2(uv[i], uv[i]);
      moments(i);
      top_m = top3(top_m, mv[i].x, mv[i].y);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      root_v[i] = make_float2(__fsqrt_rn(uv[i].x), __fsqrt_rn(uv[i].y));
      top_u = top3(top_u, root_v[i].x, root_v[i].y);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) param(i, root_v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      moments(i);
      param(i, make_float2(__fsqrt_rn(uv[i].x), __fsqrt_rn(uv[i].y)));
    }
  }
  x.param.set(pv);
  x.param.store(x.p, U::GAP, U::ONE, x.full, x.left);
  if constexpr (EIGHT) {
    top_m = warp_top(top_m), top_u = warp_top(top_u);
    const float inv_m = inverse(top_m), inv_u = inverse(top_u);
    unsigned cm[2], cu[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      cm[j] = __byte_perm(m_codes(mul2(mv[2 * j], both(inv_m)), a.one),
                          m_codes(mul2(mv[2 * j + 1], both(inv_m)), a.one), 0x7531);
      cu[j] = __byte_perm(u_codes(mul2(root_v[2 * j], both(inv_u)), a.one),
                          u_codes(mul2(root_v[2 * j + 1], both(inv_u)), a.one), 0x7531);
    }
    uint8_t *pm = static_cast<uint8_t*>(a.m) + x.at, *pu = static_cast<uint8_t*>(a.v) + x.at;
    if constexpr (U::ONE) {
      *reinterpret_cast<uint2*>(pm) = make_uint2(cm[0], cm[1]);
      *reinterpret_cast<uint2*>(pu) = make_uint2(cu[0], cu[1]);
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        *reinterpret_cast<unsigned*>(pm + j * U::GAP) = cm[j];
        *reinterpret_cast<unsigned*>(pu + j * U::GAP) = cu[j];
      }
    }
    if (lane == 0) a.scales[x.at / BLOCK] = make_float2(top_m, top_u);
  } else {
    Eight<float> w;
    w.set(mv);
    w.store(static_cast<float*>(a.m) + x.at, U::GAP, false, true, 0);
    w.set(uv);
    w.store(static_cast<float*>(a.v) + x.at, U::GAP, false, true, 0);
  }
}

template <typename T, typename TG, bool EIGHT, int N>
__global__ void __launch_bounds__(THREADS, EIGHT ? eight_ctas(sizeof(T), sizeof(TG)) : FULL_CTAS) adamw_kernel(
    const __grid_constant__ Table<N> tab, const __grid_constant__ StepArgs a) {
  Factors f{a.decay, a.size, a.root, a.grad_scale ? *a.grad_scale : 1.f};
  if (!isfinite(f.grad)) return;  // an overflow somewhere in the gradients: nothing changes
  if (a.step || a.lr) {
    __shared__ float computed[3];
    if (threadIdx.x == 0) {
      const double lr = a.lr ? (double)*a.lr : a.lrd;
      computed[0] = (float)(1.0 - lr * a.wdd);
      if (a.step) {
        const double t = (double)max(*a.step, 1LL);
        computed[1] = (float)(lr / (1.0 - pow(a.b1d, t)));
        computed[2] = (float)(1.0 / sqrt(1.0 - pow(a.b2d, t)));
      } else {  // size is 1 / (1 - b1^t) here
        computed[1] = (float)(lr * (double)f.size);
        computed[2] = f.root;
      }
    }
    __syncthreads();
    f.decay = computed[0], f.size = computed[1], f.root = computed[2];
  }
  const int lane = threadIdx.x & 31;
  const unsigned warps = gridDim.x * WARPS;
  unsigned run = blockIdx.x * WARPS + (threadIdx.x >> 5);
  if (run >= tab.total) return;
  if constexpr (!EIGHT) {
    for (unsigned unit = run; unit < tab.total; unit += warps) {
      Unit<T, TG, EIGHT, N> x;
      x.fetch(tab, a, tensor_of(tab, unit), unit, lane);
      update(x, a, f, lane);
    }
  } else {
    // Runs of a.run blocks per warp: the tensor is searched for at the first, and followed from there.
    unsigned unit = run * a.run, end = min(unit + a.run, tab.total);
    if (unit >= tab.total) return;
    const unsigned last = (tab.total - 1) / a.run;
    int k = tensor_of(tab, unit);
    const auto advance = [&] {  // whether there is another block
      if (++unit < end) {
        while (k + 1 < tab.count && unit >= tab.start[k + 1]) ++k;
        return true;
      }
      run += warps;
      if (run > last) return false;
      unit = run * a.run;
      end = min(unit + a.run, tab.total);
      k = tensor_of(tab, unit);
      return true;
    };
    // The arithmetic is long: the next block is on its way meanwhile.
    Unit<T, TG, EIGHT, N> x, y;
    x.fetch(tab, a, k, unit, lane);
    for (;;) {
      bool more = advance();
      if (more) y.fetch(tab, a, k, unit, lane);
      update(x, a, f, lane);
      if (!more) return;
      more = advance();
      if (more) x.fetch(tab, a, k, unit, lane);
      update(y, a, f, lane);
      if (!more) return;
    }
  }
}

// The values that 8-bit moments stand for: 4096 of them per CTA, four times four per thread, all loads first.
constexpr int VALUES = 4;

__global__ void __launch_bounds__(THREADS) adamw_values_kernel(const uint8_t* m, const uint8_t* u, const float2* scales,
                                                               float* m_out, float* v_out, long long n) {
  const long long first = blockIdx.x * (long long)(VALUES * THREADS * 4) + threadIdx.x * 4;
  unsigned mc[VALUES], uc[VALUES];
  float2 sc[VALUES];
#pragma unroll
  for (int i = 0; i < VALUES; ++i) {
    const long long at = first + i * (THREADS * 4);
    if (at < n) {
      mc[i] = *reinterpret_cast<const unsigned*>(m + at);
      uc[i] = *reinterpret_cast<const unsigned*>(u + at);
      sc[i] = scales[at / BLOCK];
    }
  }
#pragma unroll
  for (int i = 0; i < VALUES; ++i) {
    const long long at = first + i * (THREADS * 4);
    if (at < n) {
      const float2 m0 = mul2(m_values<0>(mc[i]), both(sc[i].x)), m1 = mul2(m_values<1>(mc[i]), both(sc[i].x));
      float2 u0 = mul2(u_values<0>(uc[i]), both(sc[i].y)), u1 = mul2(u_values<1>(uc[i]), both(sc[i].y));
      u0 = mul2(u0, u0), u1 = mul2(u1, u1);
      *reinterpret_cast<float4*>(m_out + at) = make_float4(m0.x, m0.y, m1.x, m1.y);
      *reinterpret_cast<float4*>(v_out + at) = make_float4(u0.x, u0.y, u1.x, u1.y);
    }
  }
}

// Sums of squares in double: exact products, and neither overflow nor underflow for any fp32 value. Warps take runs of
// 1024 elements; CTAs leave a sum each, and one CTA adds those in a fixed order. Up to FEW runs one cluster of eight CTAs does
// both, which saves a launch (90 fp16 tensors of 0.6 M elements: 23 us with two launches).
constexpr int RUN = 1024, FEW = 1024, CLUSTER = 8, CLUSTER_THREADS = 512;

template <typename T>
__device__ __forceinline__ void add_squares(const T* g, long long left, int lane, double (&s)[4]) {
  constexpr int VEC = 16 / (int)sizeof(T), LOADS = RUN / 32 / VEC;
  const int n = (int)min(left, (long long)RUN);
  const auto add = [&](float x, int i) { s[i] = fma((double)x, (double)x, s[i]); };
  if (reinterpret_cast<uintptr_t>(g) % 16 == 0) {
    uint4 w[LOADS];
    if (n == RUN) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) w[j] = reinterpret_cast<const uint4*>(g)[j * 32 + lane];
    } else {
#pragma unroll
      for (int j = 0; j < LOADS; ++j)
        w[j] = (j * 32 + lane + 1) * VEC <= n ? reinterpret_cast<const uint4*>(g)[j * 32 + lane] : make_uint4(0, 0, 0, 0);
      const int rest = n / VEC * VEC + lane;
      if (rest < n) add(to_f(g[rest]), 0);
    }
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      float2 v[VEC / 2];
      unpack16(w[j], v, T());
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) add(v[i].x, (2 * i) % 4), add(v[i].y, (2 * i + 1) % 4);
    }
  } else {
#pragma unroll 1
    for (int at = lane; at < n; at += 8 * 32) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = at + 32 * j < n ? to_f(g[at + 32 * j]) : 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) add(v[j], j % 4);
    }
  }
}

// The sum of the runs that a CTA's warps take, in thread 0.
template <typename T, int N, int WARPS_>
__device__ __forceinline__ double cta_squares(const Table<N>& tab) {
  __shared__ double red[WARPS_];
  const int lane = threadIdx.x & 31;
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  for (unsigned unit = blockIdx.x * WARPS_ + (threadIdx.x >> 5); unit < tab.total; unit += gridDim.x * WARPS_) {
    const int k = tensor_of(tab, unit);
    const long long at = (long long)(unit - tab.start[k]) * RUN;
    add_squares(static_cast<const T*>(tab.t[k].grad) + at, tab.t[k].n - at, lane, s);
  }
  double t = ub::warp_sum_d((s[0] + s[1]) + (s[2] + s[3]));
  if (lane == 0) red[threadIdx.x >> 5] = t;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int w = 1; w < WARPS_; ++w) t += red[w];
  return t;
}

__device__ __forceinline__ void norm_out(double sum, float max_norm, float* norm, float* scale) {
  const double r = sqrt(sum);
  const float given = (float)r;  // infinite from half a step above the largest fp32 number on
  *norm = given;
  if (scale) *scale = !isfinite(given) ? given - given : r > max_norm ? (float)(max_norm / r) : 1.f;
}

template <typename T, int N>
__global__ void __launch_bounds__(THREADS) square_sums_kernel(const __grid_constant__ Table<N> tab, double* part) {
  const double t = cta_squares<T, N, WARPS>(tab);
  if (threadIdx.x == 0) part[blockIdx.x] = t;
}

__global__ void __launch_bounds__(1024) norm_join_kernel(const double* part, int n, float max_norm, float* norm,
                                                         float* scale) {
  __shared__ double red[32];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) s += part[i];
  s = ub::warp_sum_d(s);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = ub::warp_sum_d(red[threadIdx.x]);
    if (threadIdx.x == 0) norm_out(s, max_norm, norm, scale);
  }
}

template <typename T, int N>
__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(CLUSTER_THREADS)
    few_squares_kernel(const __grid_constant__ Table<N> tab, float max_norm, float* norm, float* scale) {
  __shared__ double sums[CLUSTER];  // in the first CTA
  cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  cluster.barrier_arrive();
  const double t = cta_squares<T, N, CLUSTER_THREADS / 32>(tab);
  cluster.barrier_wait();  // the first CTA is there
  if (threadIdx.x == 0) *cluster.map_shared_rank(&sums[blockIdx.x], 0) = t;
  cluster.sync();
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    double s = sums[0];
    for (int i = 1; i < CLUSTER; ++i) s += sums[i];
    norm_out(s, max_norm, norm, scale);
  }
}

template <int N>
Table<N> make_table(const UnblendAdamWTensor* t, int count, int unit) {
  Table<N> tab;
  tab.count = count;
  unsigned at = 0;
  for (int i = 0; i < count; ++i) {
    tab.t[i] = t[i];
    tab.start[i] = at;
    at += (unsigned)((t[i].n + unit - 1) / unit);
  }
  tab.total = at;
  return tab;
}

bool tensors_ok(const UnblendAdamWTensor* t, int count, bool params, int elem, int grad_elem) {
  if (!t || count < 1) return false;
  long long units = 0;
  for (int i = 0; i < count; ++i) {
    if (t[i].n < 1 || t[i].n >= (1LL << 39) || !t[i].grad || reinterpret_cast<uintptr_t>(t[i].grad) % grad_elem)
      return false;
    if (params && (!t[i].param || reinterpret_cast<uintptr_t>(t[i].param) % elem || t[i].block < 0 ||
                   t[i].block >= (1LL << 31)))
      return false;
    units += (t[i].n + BLOCK - 1) / BLOCK;
  }
  return units < (1LL << 31);
}

struct Span {
  uintptr_t from, to;
};
bool before(const Span& x, const Span& y) { return x.from < y.from; }

// The spans of `list` in order, those up to `mid` and those from there each usually being so already.
void in_order(std::vector<Span>& list, size_t mid) {
  const auto parts = {list.begin(), list.begin() + mid, list.end()};
  for (auto p = parts.begin(); p + 1 != parts.end(); ++p)
    if (!std::is_sorted(p[0], p[1], before)) std::sort(p[0], p[1], before);
  std::inplace_merge(list.begin(), list.begin() + mid, list.end(), before);
}

// Whether what the call writes (parameters, moments, scales) shares memory neither within itself nor with what else it reads
// (gradients, numbers on the device).
bool apart(const UnblendAdamWTensor* t, int count, int elem, int grad_elem, int bits, const void* m, const void* v,
           const void* scales, const UnblendAdamWParams* p) {
  std::vector<Span> written, only_read, blocks;  // blocks: of the moments, joined where tensors follow one another
  written.reserve((size_t)count + 3);
  only_read.reserve((size_t)count + 3);
  const auto span = [](const void* x, uintptr_t bytes) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(x);
    return Span{at, at + bytes};
  };
  bool ordered = true;
  for (int i = 0; i < count; ++i) {
    written.push_back(span(t[i].param, (uintptr_t)t[i].n * elem));
    only_read.push_back(span(t[i].grad, (uintptr_t)t[i].n * grad_elem));
    const uintptr_t from = (uintptr_t)t[i].block, to = from + (uintptr_t)((t[i].n + BLOCK - 1) / BLOCK);
    if (!blocks.empty() && from == blocks.back().to) {
      blocks.back().to = to;
    } else {
      ordered &= blocks.empty() || from > blocks.back().to;
      blocks.push_back(Span{from, to});
    }
  }
  if (!ordered) {
    std::sort(blocks.begin(), blocks.end(), before);
    for (size_t i = 1; i < blocks.size(); ++i)
      if (blocks[i].from < blocks[i - 1].to) return false;
  }
  const auto moments = [&](const void* base, uintptr_t bytes) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(base);
    for (const Span& b : blocks) written.push_back(Span{at + b.from * bytes, at + b.to * bytes});
  };
  moments(m, BLOCK * bits / 8);
  moments(v, BLOCK * bits / 8);
  if (bits == 8) moments(scales, sizeof(float2));
  if (p->step_device) only_read.push_back(span(p->step_device, sizeof(long long)));
  if (p->lr_device) only_read.push_back(span(p->lr_device, sizeof(float)));
  if (p->grad_scale) only_read.push_back(span(p->grad_scale, sizeof(float)));
  in_order(written, count);
  in_order(only_read, count);
  const Span *w = written.data(), *w_end = w + written.size(), *r = only_read.data(), *r_end = r + only_read.size();
  uintptr_t end = 0, seen = 0;  // of what is written, and of all, so far
  while (w < w_end || r < r_end) {
    const bool write = r == r_end || (w < w_end && w->from <= r->from);
    const Span& x = write ? *w++ : *r++;
    if (x.from < (write ? seen : end)) return false;
    if (write) end = std::max(end, x.to);
    seen = std::max(seen, x.to);
  }
  return true;
}

unsigned grid_of(unsigned units, int per_sm) {
  const unsigned ctas = (units + WARPS - 1) / WARPS, cap = ub::kNumSMs * per_sm;
  return ctas < cap ? ctas : cap;
}

template <typename T, typename TG, bool EIGHT, int N>
int launch_table(const UnblendAdamWTensor* t, int count, StepArgs a, cudaStream_t st) {
  const Table<N> tab = make_table<N>(t, count, BLOCK);
  const unsigned grid = grid_of(tab.total, EIGHT ? eight_ctas(sizeof(T), sizeof(TG)) : 2 * FULL_CTAS);
  if (EIGHT) a.run = std::min(16u, std::max(1u, tab.total / (grid * WARPS * 4)));  // four runs per warp at least
  adamw_kernel<T, TG, EIGHT, N><<<grid, THREADS, 0, st>>>(tab, a);
  UB_CHECK_LAUNCH();
  return 0;
}

template <typename T, typename TG, bool EIGHT>
int launch_step(const UnblendAdamWTensor* t, int count, const StepArgs& a, cudaStream_t st) {
  for (int i = 0; i < count; i += LARGE) {
    const int n = std::min(LARGE, count - i);
    const int rc = n <= SMALL    ? launch_table<T, TG, EIGHT, SMALL>(t + i, n, a, st)
                   : n <= MIDDLE ? launch_table<T, TG, EIGHT, MIDDLE>(t + i, n, a, st)
                                 : launch_table<T, TG, EIGHT, LARGE>(t + i, n, a, st);
    if (rc) return rc;
  }
  return 0;
}

template <typename T, typename TG>
int launch_bits(const UnblendAdamWTensor* t, int count, int bits, const StepArgs& a, cudaStream_t st) {
  return bits == 8 ? launch_step<T, TG, true>(t, count, a, st) : launch_step<T, TG, false>(t, count, a, st);
}

template <typename T>
int launch_grad(const UnblendAdamWTensor* t, int count, int grad_dtype, int bits, const StepArgs& a, cudaStream_t st) {
  switch (grad_dtype) {
    case UNBLEND_F32: return launch_bits<T, float>(t, count, bits, a, st);
    case UNBLEND_BF16: return launch_bits<T, __nv_bfloat16>(t, count, bits, a, st);
    default: return launch_bits<T, __half>(t, count, bits, a, st);
  }
}

constexpr int NORM_CTAS = 8;  // per SM

template <typename T, int N>
int launch_few(const UnblendAdamWTensor* t, int count, float max_norm, float* norm, float* scale, cudaStream_t st) {
  few_squares_kernel<T, N><<<CLUSTER, CLUSTER_THREADS, 0, st>>>(make_table<N>(t, count, RUN), max_norm, norm, scale);
  UB_CHECK_LAUNCH();
  return 0;
}

template <typename T, int N>
int launch_sums(const UnblendAdamWTensor* t, int count, double* part, int* used, cudaStream_t st) {
  const Table<N> tab = make_table<N>(t, count, RUN);
  const unsigned grid = grid_of(tab.total, NORM_CTAS);
  square_sums_kernel<T, N><<<grid, THREADS, 0, st>>>(tab, part + *used);
  UB_CHECK_LAUNCH();
  *used += (int)grid;
  return 0;
}

// All tensors of one type. Few: the norm itself; else partial sums.
template <typename T>
int launch_squares(const UnblendAdamWTensor* t, int count, bool few, float max_norm, float* norm, float* scale,
                   double* part, int* used, cudaStream_t st) {
  if (few)
    return count <= SMALL    ? launch_few<T, SMALL>(t, count, max_norm, norm, scale, st)
           : count <= MIDDLE ? launch_few<T, MIDDLE>(t, count, max_norm, norm, scale, st)
                             : launch_few<T, LARGE>(t, count, max_norm, norm, scale, st);
  for (int i = 0; i < count; i += LARGE) {
    const int n = std::min(LARGE, count - i);
    const int rc = n <= SMALL    ? launch_sums<T, SMALL>(t + i, n, part, used, st)
                   : n <= MIDDLE ? launch_sums<T, MIDDLE>(t + i, n, part, used, st)
                                 : launch_sums<T, LARGE>(t + i, n, part, used, st);
    if (rc) return rc;
  }
  return 0;
}

// The update multiplies by an approximate reciprocal, which takes normal numbers only; the root of v is 0 or above 2^-75.
bool eps_ok(double eps) { return eps == 0 || (eps >= 1.17549435e-38 && eps <= 1e30); }

}  // namespace

extern "C" int unblend_adamw_step(const UnblendAdamWTensor* tensors, int count, void* exp_avg, void* exp_avg_sq,
                                  float* scales, int bits, int dtype, int grad_dtype, const UnblendAdamWParams* p,
                                  void* stream) {
  UB_REQUIRE(p && known_type(dtype) && known_type(grad_dtype) && (bits == 32 || bits == 8));
  UB_REQUIRE(exp_avg && exp_avg_sq && aligned16(exp_avg) && aligned16(exp_avg_sq));
  UB_REQUIRE(bits == 32 || (scales && reinterpret_cast<uintptr_t>(scales) % 8 == 0));
  UB_REQUIRE(p->beta1 >= 0 && p->beta1 < 1 && p->beta2 >= 0 && p->beta2 < 1 && eps_ok(p->eps));
  UB_REQUIRE(std::fabs(p->weight_decay) <= 1e18 && (p->lr_device || std::fabs(p->lr) <= 1e18));
  UB_REQUIRE(p->step_device || p->step >= 1);
  UB_REQUIRE(reinterpret_cast<uintptr_t>(p->step_device) % 8 == 0 && reinterpret_cast<uintptr_t>(p->lr_device) % 4 == 0 &&
             reinterpret_cast<uintptr_t>(p->grad_scale) % 4 == 0);
  UB_REQUIRE(tensors_ok(tensors, count, true, elem_size(dtype), elem_size(grad_dtype)));
  try {
    if (!apart(tensors, count, elem_size(dtype), elem_size(grad_dtype), bits, exp_avg, exp_avg_sq, scales, p))
      return UNBLEND_ERR_OVERLAP;
  } catch (const std::bad_alloc&) {
    return (int)cudaErrorMemoryAllocation;
  }
  StepArgs a{};
  a.run = 1;
  a.m = exp_avg;
  a.v = exp_avg_sq;
  a.scales = reinterpret_cast<float2*>(scales);
  a.grad_scale = p->grad_scale;
  a.step = p->step_device;
  a.lr = p->lr_device;
  a.b1d = p->beta1;
  a.b2d = p->beta2;
  a.lrd = p->lr;
  a.wdd = p->weight_decay;
  a.b1 = (float)p->beta1;
  a.c1 = (float)(1.0 - p->beta1);
  a.b2 = (float)p->beta2;
  a.c2 = (float)(1.0 - p->beta2);
  a.eps = (float)p->eps;
  a.one = 1.f;
  const double t = p->step_device ? 1.0 : (double)p->step;
  const double correction = 1.0 - std::pow(p->beta1, t);
  a.decay = (float)(1.0 - p->lr * p->weight_decay);
  a.size = (float)((p->lr_device ? 1.0 : p->lr) / correction);
  a.root = (float)(1.0 / std::sqrt(1.0 - std::pow(p->beta2, t)));
  cudaStream_t st = ub::as_stream(stream);
  switch (dtype) {
    case UNBLEND_F32: return launch_grad<float>(tensors, count, grad_dtype, bits, a, st);
    case UNBLEND_BF16: return launch_grad<__nv_bfloat16>(tensors, count, grad_dtype, bits, a, st);
    default: return launch_grad<__half>(tensors, count, grad_dtype, bits, a, st);
  }
}

extern "C" int unblend_adamw_values(const void* exp_avg, const void* exp_avg_sq, const float* scales, float* m, float* v,
                                    long long blocks, void* stream) {
  UB_REQUIRE(exp_avg && exp_avg_sq && scales && m && v && blocks >= 1 && blocks < (1LL << 31));
  UB_REQUIRE(aligned16(exp_avg) && aligned16(exp_avg_sq) && aligned16(m) && aligned16(v) &&
             reinterpret_cast<uintptr_t>(scales) % 8 == 0);
  const long long n = blocks * BLOCK, per_cta = VALUES * THREADS * 4;
  adamw_values_kernel<<<(unsigned)((n + per_cta - 1) / per_cta), THREADS, 0, ub::as_stream(stream)>>>(
      static_cast<const uint8_t*>(exp_avg), static_cast<const uint8_t*>(exp_avg_sq),
      reinterpret_cast<const float2*>(scales), m, v, n);
  UB_CHECK_LAUNCH();
  return 0;
}

extern "C" int unblend_grad_norm_workspace(int count, long long* bytes) {
  UB_REQUIRE(count >= 1 && bytes);
  // A launch for every LARGE tensors of each of the three types.
  *bytes = ((count + LARGE - 1) / LARGE + 2LL) * (ub::kNumSMs * NORM_CTAS) * (long long)sizeof(double);
  return 0;
}

extern "C" int unblend_grad_norm(const UnblendAdamWTensor* tensors, const int* counts, float max_norm, float* norm,
                                 float* scale, double* work, void* stream) {
  UB_REQUIRE(tensors && counts && norm && work && reinterpret_cast<uintptr_t>(work) % 8 == 0);
  UB_REQUIRE(!scale || (max_norm > 0.f && std::isfinite(max_norm)));
  long long runs = 0;
  int first = 0, used = 0, kinds = 0;
  for (int t = 0; t < 3; ++t) {
    UB_REQUIRE(counts[t] >= 0);
    UB_REQUIRE(counts[t] == 0 || tensors_ok(tensors + first, counts[t], false, 1, elem_size(t)));
    for (int i = first; i < first + counts[t]; ++i) runs += (tensors[i].n + RUN - 1) / RUN;
    first += counts[t];
    kinds += counts[t] > 0;
  }
  const bool few = kinds == 1 && first <= LARGE && runs <= FEW;
  cudaStream_t st = ub::as_stream(stream);
  first = 0;
  for (int t = 0; t < 3; ++t) {
    if (counts[t] == 0) continue;
    const UnblendAdamWTensor* mine = tensors + first;
    const int rc =
        t == UNBLEND_F32 ? launch_squares<float>(mine, counts[t], few, max_norm, norm, scale, work, &used, st)
        : t == UNBLEND_BF16
            ? launch_squares<__nv_bfloat16>(mine, counts[t], few, max_norm, norm, scale, work, &used, st)
            : launch_squares<__half>(mine, counts[t], few, max_norm, norm, scale, work, &used, st);
    if (rc) return rc;
    first += counts[t];
  }
  if (few) return 0;
  norm_join_kernel<<<1, 1024, 0, st>>>(work, used, max_norm, norm, scale);
  UB_CHECK_LAUNCH();
  return 0;
}
