// LayerNorm with gradients: forward that leaves each row's (mean, rstd), backward for the input and the weights.
//
//   y = xhat * gamma + beta,  xhat = (x - mean) * rstd,  rstd = 1 / sqrt(var + eps)
//   gy = dy * gamma
//   dx = rstd * (gy - mean(gy) - xhat * mean(gy * xhat))
//   dgamma = sum_rows dy * xhat,  dbeta = sum_rows dy
//
// Statistics, sums and all arithmetic are fp32; x, y, dy and dx are fp32, bf16 or fp16.
// Floor of both directions: one read of each input and one write of each output. The forward pass of wide 16-bit rows
// stops at the L1 path before HBM (78 and 39 % of their rates at 65536 x 1024 bf16): each row reads the weights again.
//
// A row of up to 1024 columns belongs to one warp (no barrier), a wider one up to 8192 to a CTA, 16 values per thread;
// wider rows are read again for every reduction. Rows come through shared memory by cp.async, several in flight per
// warp, and the arithmetic goes two values at a time: at HBM's rate an SM has some 180 cycles for a row of 1024 bf16
// columns, and both latency (one row per warp in flight) and issue slots (scalar arithmetic) had been the bound.
//
// Rows that do not start on 16-byte boundaries (odd widths, slices) move by aligned 16-byte chunks as well: a thread
// takes its values out of its own chunk and its neighbour's. A chunk at the end of a row holds values of the next one,
// or of the gap between them; only chunks that reach in front of the tensor's first row or behind its last are put
// together value by value (a load that the thread waits for: done at every row's ends it cost half the bandwidth).
//
// Measured (forward, backward with all gradients): 86016 x 512 fp32 71 and 94 us (4.9 and 5.6 TB/s), 262147 x 1024 bf16
// 239 and 284 us (4.5 and 5.7 TB/s), 50000 x 4096 bf16 252 and 307 us (3.2 and 4.0 TB/s: a CTA's barriers show),
// 3333 x 5003 fp16 in wider rows 34 and 78 us (1.9 and 1.3 TB/s), 20000 x 12000 bf16 714 and 1566 us (three passes).
//
// The weights' gradients are summed in registers over the rows that a group walks, joined across the CTA in shared
// memory, and the CTAs' partial rows added in a fixed order by a second kernel: the result is the same on every run.
#include "train_common.cuh"

namespace {

using namespace ub::train;

constexpr int WARP_COLS = 1024;   // widest row of a warp
constexpr int CTA_COLS = 8192;    // widest row held in a CTA's registers
// Backward calls of up to so many narrow rows run in one CTA of 16 warps, without partial sums and their kernel.
constexpr int ONE_CTA_ROWS = 64;

struct NormArgs {
  const void* x;
  const void* dy;
  const void* gamma;
  const void* beta;
  void* y;       // forward output, or dx
  float* stats;  // [rows][2]
  float* part;   // [gridDim.x][2][cols], or null when one CTA writes the sums itself
  void *dgamma, *dbeta;
  RowMap xm, dym;
  unsigned rows;
  int cols;
  int w_vec;  // the weights' base is aligned for 16-byte loads
  const void *x_lo, *x_hi, *dy_lo, *dy_hi;  // the memory from the first row's first value to the last one's end
  float eps;
};

// Sum of N values over the threads of a row: a warp or the CTA. CTA rows alternate between two shared arrays: an array
// is written again only after the barrier of the reduction in between, which every reader of it has passed.
template <bool WARP, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* red, int& phase) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = ub::warp_sum(v[i]);
  if constexpr (!WARP) {
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;  // at most 16
    float* r = red + phase * 16 * N;
    phase ^= 1;
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) r[(threadIdx.x >> 5) * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = lane < warps ? r[lane * N + i] : 0.f;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      v[i] = __shfl_sync(0xffffffffu, s, 0);
    }
  }
}

// The eight words (a, then b) from byte `shift` on (a multiple of the element size), 16 bytes of them.
__device__ __forceinline__ uint4 take16(const uint4& a, const uint4& b, int shift) {
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  if (shift & 8) {
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  }
  if (shift & 4) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  if (shift & 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint4 shfl_down1(const uint4& v) {
  return make_uint4(__shfl_down_sync(0xffffffffu, v.x, 1), __shfl_down_sync(0xffffffffu, v.y, 1),
                    __shfl_down_sync(0xffffffffu, v.z, 1), __shfl_down_sync(0xffffffffu, v.w, 1));
}

// A run of VEC consecutive values of a row on its way through shared memory: the aligned chunk that holds the first of
// them and, for the last lane of a warp, the chunk behind it (other lanes get that from their neighbour). A thread
// reads what it copied itself, so no barrier is needed. `g` is the number of the run.
template <typename T, bool ALIGNED>
struct Run {
  static constexpr int VEC = 16 / (int)sizeof(T);

  __device__ __forceinline__ static int shift(const T* row) { return (int)(reinterpret_cast<uintptr_t>(row) & 15); }

  __device__ __forceinline__ static void chunk(uint4* dst, const T* row, int first, int cols, const void* lo,
                                               const void* hi) {
    const T* p = row + first;
    if (first >= cols) return;
    if (p >= static_cast<const T*>(lo) && p + VEC <= static_cast<const T*>(hi)) {
      cp_async16(dst, p);
    } else {
      uint4 v = make_uint4(0, 0, 0, 0);
      T* e = reinterpret_cast<T*>(&v);
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (first + i >= 0 && first + i < cols) e[i] = p[i];
      *dst = v;
    }
  }

  __device__ __forceinline__ static void fetch(uint4* a, uint4* b, const T* row, int g, int cols, const void* lo,
                                               const void* hi) {
    if constexpr (ALIGNED) {
      if (g * VEC < cols) cp_async16(a, row + g * VEC);
    } else {
      const int first = g * VEC - shift(row) / (int)sizeof(T);
      chunk(a, row, first, cols, lo, hi);
      if ((threadIdx.x & 31) == 31 && shift(row)) chunk(b, row, first + VEC, cols, lo, hi);
    }
  }

  // All lanes of a warp together. Values past the row are 0.
  __device__ __forceinline__ static void read(const uint4* a, const uint4* b, int row_shift, int g, int cols,
                                              float2 (&v)[VEC / 2]) {
    uint4 w = *a;
    if constexpr (!ALIGNED) {
      if (row_shift) {
        uint4 n = shfl_down1(w);
        if ((threadIdx.x & 31) == 31) n = *b;
        w = take16(w, n, row_shift);
      }
    }
    unpack16(w, v, T());
    const int left = cols - g * VEC;
    if (left < VEC) {
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) {
        if (2 * i >= left) v[i].x = 0.f;
        if (2 * i + 1 >= left) v[i].y = 0.f;
      }
    }
  }
};

// The rows in flight of a thread: STAGES x RUNS chunks of its own and of its warp's last lane.
template <int STAGES, int RUNS, bool ALIGNED>
struct Ring {
  static constexpr int bytes(int threads) { return STAGES * RUNS * 16 * (threads + (ALIGNED ? 0 : threads / 32)); }
  uint4* base;
  __device__ __forceinline__ uint4* a(int stage, int k) const {
    return base + (stage * RUNS + k) * blockDim.x + threadIdx.x;
  }
  __device__ __forceinline__ uint4* b(int stage, int k) const {
    return base + STAGES * RUNS * blockDim.x + (stage * RUNS + k) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  }
};

// Rows in flight: 4, less where they would leave room for one CTA only (a warp per row) or for none (a CTA per row).
template <typename T, int NV, int TENSORS, bool WARP>
constexpr int stages_of() {
  const int one = (WARP ? 256 : 528) * NV * TENSORS * 16;
  if (WARP) return 4 * one > 112 * 1024 ? 2 : 4;
  return 4 * one > 208 * 1024 ? 3 : 4;
}

// Stores VEC values of every lane (runs g of consecutive lanes follow one another) to a row that starts anywhere. The
// aligned chunk that starts in a lane's values ends in the next lane's.
template <typename T, bool ALIGNED>
__device__ __forceinline__ void store_run(T* row, int g, int cols, const float2 (&o)[8 / sizeof(T)]) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const uint4 w = pack16(o, T());
  const int c = g * VEC;
  if constexpr (ALIGNED) {
    if (c < cols) *reinterpret_cast<uint4*>(row + c) = w;
  } else {
    const int lane = threadIdx.x & 31;
    const int mis = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    const int h = mis ? VEC - mis : 0;  // values of a run in front of the chunk that starts in it
    const uint4 n = shfl_down1(w);
    const bool whole = c + h + VEC <= cols && (lane < 31 || h == 0);
    if (whole) *reinterpret_cast<uint4*>(row + c + h) = take16(w, n, h * (int)sizeof(T));
    // Values that no whole chunk takes: in front of a warp's first chunk, behind its last, around the row's end.
    const bool front = lane == 0 || c + h > cols;
    if (front || !whole) {
      const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (c + i < cols && (i < h ? front : !whole)) row[c + i] = e[i];
    }
  }
}

// Weights of run g as fp32 pairs, `none` without weights and past the row.
template <typename TW, int VEC>
__device__ __forceinline__ void load_weights(const NormArgs& a, const void* w, float none, int g,
                                             float2 (&v)[VEC / 2]) {
  const int c = g * VEC;
  const TW* p = static_cast<const TW*>(w) + c;
  if (w && a.w_vec && c + VEC <= a.cols) {
    load_vec<TW, VEC>(p, reinterpret_cast<float(&)[VEC]>(v));
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      v[i].x = w && c + 2 * i < a.cols ? to_f(p[2 * i]) : none;
      v[i].y = w && c + 2 * i + 1 < a.cols ? to_f(p[2 * i + 1]) : none;
    }
  }
}

template <typename T, typename TW, int NV, bool ALIGNED, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 512, WARP ? 2 : 1)
    layer_norm_fwd_kernel(const __grid_constant__ NormArgs a) {
  constexpr int VEC = 16 / (int)sizeof(T);
  constexpr int ST = stages_of<T, NV, 1, WARP>();
  using R = Run<T, ALIGNED>;
  __shared__ float red[32];
  extern __shared__ uint4 dyn[];
  const Ring<ST, NV, ALIGNED> ring{dyn};
  int phase = 0;
  const int tpr = WARP ? 32 : blockDim.x;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int group = WARP ? threadIdx.x >> 5 : 0, groups = WARP ? blockDim.x >> 5 : 1;
  const float inv_c = 1.f / (float)a.cols;
  const long long step = (long long)gridDim.x * groups;
  const T* xb = static_cast<const T*>(a.x);
  auto fetch = [&](int stage, long long r) {
    if (r < a.rows) {
      const T* x = xb + row_offset(a.xm, (unsigned)r);
#pragma unroll
      for (int k = 0; k < NV; ++k) R::fetch(ring.a(stage, k), ring.b(stage, k), x, k * tpr + t, a.cols, a.x_lo, a.x_hi);
    }
    cp_commit();
  };
  long long row = (long long)blockIdx.x * groups + group;
#pragma unroll
  for (int i = 0; i < ST - 1; ++i) fetch(i, row + i * step);
  for (int stage = 0; row < a.rows; row += step, stage = (stage + 1) % ST) {
    fetch((stage + ST - 1) % ST, row + (ST - 1) * step);
    cp_wait<ST - 1>();
    const int shift = ALIGNED ? 0 : R::shift(xb + row_offset(a.xm, (unsigned)row));
    float2 v[NV][VEC / 2], acc = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (ALIGNED && (k * tpr + t) * VEC >= a.cols) {
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) v[k][i] = make_float2(0.f, 0.f);
      } else {
        R::read(ring.a(stage, k), ring.b(stage, k), shift, k * tpr + t, ALIGNED ? 1 << 30 : a.cols, v[k]);
      }
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) acc = add2(acc, v[k][i]);
    }
    float s[1] = {acc.x + acc.y};
    row_sum<WARP, 1>(s, red, phase);
    const float mean = s[0] * inv_c;
    const float2 minus = make_float2(-mean, -mean);
    acc = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int left = a.cols - (k * tpr + t) * VEC;
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) {
        v[k][i] = add2(v[k][i], minus);
        if (left < VEC) {
          if (2 * i >= left) v[k][i].x = 0.f;
          if (2 * i + 1 >= left) v[k][i].y = 0.f;
        }
        acc = ub::fma2(v[k][i], v[k][i], acc);
      }
    }
    s[0] = acc.x + acc.y;
    row_sum<WARP, 1>(s, red, phase);
    const float rstd = 1.f / sqrtf(s[0] * inv_c + a.eps);
    const float2 r2 = make_float2(rstd, rstd);
    T* y = static_cast<T*>(a.y) + row * a.cols;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float2 g[VEC / 2], b[VEC / 2];
      load_weights<TW, VEC>(a, a.gamma, 1.f, k * tpr + t, g);
      load_weights<TW, VEC>(a, a.beta, 0.f, k * tpr + t, b);
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) b[i] = ub::fma2(mul2(v[k][i], r2), g[i], b[i]);
      store_run<T, ALIGNED>(y, k * tpr + t, a.cols, b);
    }
    if (t == 0) reinterpret_cast<float2*>(a.stats)[row] = make_float2(mean, rstd);
  }
}

// The sums of the weights' gradients take the registers: a warp reads its row's x and dy again for the second pass, a
// CTA's thread, with 16 values, keeps them.
template <typename T, typename TW, int NV, bool ALIGNED, bool WARP>
__global__ void __launch_bounds__(512)
    layer_norm_bwd_kernel(const __grid_constant__ NormArgs a) {
  constexpr int VEC = 16 / (int)sizeof(T);
  constexpr int ST = stages_of<T, NV, 2, WARP>();
  constexpr bool KEEP = !WARP;
  using R = Run<T, ALIGNED>;
  __shared__ float red[64];
  extern __shared__ uint4 dyn[];
  const Ring<ST, 2 * NV, ALIGNED> ring{dyn};
  float* sums = reinterpret_cast<float*>(dyn);  // after the rows: [warps][cols]
  int phase = 0;
  const int tpr = WARP ? 32 : blockDim.x;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int group = WARP ? threadIdx.x >> 5 : 0, groups = WARP ? blockDim.x >> 5 : 1;
  const float inv_c = 1.f / (float)a.cols;
  const long long step = (long long)gridDim.x * groups;
  const T *xb = static_cast<const T*>(a.x), *dyb = static_cast<const T*>(a.dy);
  const float2* stats = reinterpret_cast<const float2*>(a.stats);
  float2 dg[NV][VEC / 2], db[NV][VEC / 2];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) dg[k][i] = db[k][i] = make_float2(0.f, 0.f);
  auto fetch = [&](int stage, long long r) {
    if (r < a.rows) {
      const T* x = xb + row_offset(a.xm, (unsigned)r);
      const T* dy = dyb + row_offset(a.dym, (unsigned)r);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        R::fetch(ring.a(stage, k), ring.b(stage, k), x, k * tpr + t, a.cols, a.x_lo, a.x_hi);
        R::fetch(ring.a(stage, NV + k), ring.b(stage, NV + k), dy, k * tpr + t, a.cols, a.dy_lo, a.dy_hi);
      }
    }
    cp_commit();
  };
  long long row = (long long)blockIdx.x * groups + group;
#pragma unroll
  for (int i = 0; i < ST - 1; ++i) fetch(i, row + i * step);
  float2 st_ahead = row < a.rows ? stats[row] : make_float2(0.f, 0.f);
  for (int stage = 0; row < a.rows; row += step, stage = (stage + 1) % ST) {
    fetch((stage + ST - 1) % ST, row + (ST - 1) * step);
    const float2 st = st_ahead;
    if (row + step < a.rows) st_ahead = stats[row + step];
    cp_wait<ST - 1>();
    int sx = 0, sd = 0;
    if constexpr (!ALIGNED) {
      sx = R::shift(xb + row_offset(a.xm, (unsigned)row));
      sd = R::shift(dyb + row_offset(a.dym, (unsigned)row));
    }
    const float2 r2 = make_float2(st.y, st.y), shift2 = make_float2(-st.x, -st.x);
    float2 s0 = make_float2(0.f, 0.f), s1 = s0;
    // xhat and gy = dy * gamma of run k; dy is 0 past the row.
    auto values = [&](int k, float2 (&xh)[VEC / 2], float2 (&d)[VEC / 2], float2 (&gy)[VEC / 2]) {
      const int g = k * tpr + t, cols = ALIGNED ? 1 << 30 : a.cols;
      R::read(ring.a(stage, k), ring.b(stage, k), sx, g, cols, xh);
      R::read(ring.a(stage, NV + k), ring.b(stage, NV + k), sd, g, cols, d);
      float2 gm[VEC / 2];
      load_weights<TW, VEC>(a, a.gamma, 1.f, g, gm);
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) {
        xh[i] = mul2(add2(xh[i], shift2), r2);
        gy[i] = mul2(d[i], gm[i]);
      }
    };
    float2 xh[KEEP ? NV : 1][VEC / 2], gy[KEEP ? NV : 1][VEC / 2];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (ALIGNED && (k * tpr + t) * VEC >= a.cols) break;
      float2 d[VEC / 2];
      const int at = KEEP ? k : 0;
      values(k, xh[at], d, gy[at]);
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) {
        dg[k][i] = ub::fma2(d[i], xh[at][i], dg[k][i]);
        db[k][i] = add2(db[k][i], d[i]);
        s0 = add2(s0, gy[at][i]);
        s1 = ub::fma2(gy[at][i], xh[at][i], s1);
      }
    }
    float s[2] = {s0.x + s0.y, s1.x + s1.y};
    row_sum<WARP, 2>(s, red, phase);
    // dx = rstd gy - rstd m0 - xhat rstd m1
    const float m0 = -st.y * (s[0] * inv_c), m1 = -st.y * (s[1] * inv_c);
    const float2 c0 = make_float2(m0, m0), c1 = make_float2(m1, m1);
    T* dx = static_cast<T*>(a.y) + row * a.cols;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (ALIGNED && (k * tpr + t) * VEC >= a.cols) break;
      const int at = KEEP ? k : 0;
      if (!KEEP) {
        float2 d[VEC / 2];
        values(k, xh[at], d, gy[at]);
      }
      float2 o[VEC / 2];
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) o[i] = ub::fma2(xh[at][i], c1, ub::fma2(gy[at][i], r2, c0));
      store_run<T, ALIGNED>(dx, k * tpr + t, a.cols, o);
    }
  }
  if (a.dgamma == nullptr) return;
  // Warps leave their sums behind one another in shared memory; the threads add them by column, in warp order.
  cp_wait<0>();
  for (int which = 0; which < 2; ++which) {
    auto put = [&](int c, float v) {
      if (a.part)
        a.part[((long long)blockIdx.x * 2 + which) * a.cols + c] = v;
      else
        static_cast<TW*>(which ? a.dbeta : a.dgamma)[c] = from_f<TW>(v);
    };
    if (WARP) __syncthreads();
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int c = (k * tpr + t) * VEC + i;
        const float2 p = which ? db[k][i / 2] : dg[k][i / 2];
        const float v = i & 1 ? p.y : p.x;
        if (c < a.cols) {
          if (WARP)
            sums[group * a.cols + c] = v;
          else
            put(c, v);
        }
      }
    if (!WARP) continue;
    __syncthreads();
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
      float v = 0.f;
      for (int w = 0; w < groups; ++w) v += sums[w * a.cols + c];
      put(c, v);
    }
  }
}

// Rows wider than the registers of a CTA: three passes over the row (the second and third hit L2).
template <typename T, typename TW>
__global__ void __launch_bounds__(512) layer_norm_fwd_wide_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[64];
  int phase = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row_offset(a.xm, (unsigned)row);
    float s[1] = {0.f}, q[1] = {0.f};
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) s[0] += to_f(x[c]);
    row_sum<false, 1>(s, red, phase);
    const float mean = s[0] / (float)a.cols;
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
      const float d = to_f(x[c]) - mean;
      q[0] = fmaf(d, d, q[0]);
    }
    row_sum<false, 1>(q, red, phase);
    const float rstd = 1.f / sqrtf(q[0] / (float)a.cols + a.eps);
    T* y = static_cast<T*>(a.y) + row * a.cols;
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
      const float g = a.gamma ? to_f(static_cast<const TW*>(a.gamma)[c]) : 1.f;
      const float b = a.beta ? to_f(static_cast<const TW*>(a.beta)[c]) : 0.f;
      y[c] = from_f<T>(fmaf((to_f(x[c]) - mean) * rstd, g, b));
    }
    if (threadIdx.x == 0) reinterpret_cast<float2*>(a.stats)[row] = make_float2(mean, rstd);
  }
}

// Input gradient of rows wider than the registers of a CTA: two passes over the row.
template <typename T, typename TW>
__global__ void __launch_bounds__(512) layer_norm_dx_wide_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[64];
  int phase = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row_offset(a.xm, (unsigned)row);
    const T* dy = static_cast<const T*>(a.dy) + row_offset(a.dym, (unsigned)row);
    const float2 st = reinterpret_cast<const float2*>(a.stats)[row];
    float s[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
      const float gy = to_f(dy[c]) * (a.gamma ? to_f(static_cast<const TW*>(a.gamma)[c]) : 1.f);
      s[0] += gy;
      s[1] = fmaf(gy, (to_f(x[c]) - st.x) * st.y, s[1]);
    }
    row_sum<false, 2>(s, red, phase);
    const float m0 = s[0] / (float)a.cols, m1 = s[1] / (float)a.cols;
    T* dx = static_cast<T*>(a.y) + row * a.cols;
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
      const float gy = to_f(dy[c]) * (a.gamma ? to_f(static_cast<const TW*>(a.gamma)[c]) : 1.f);
      dx[c] = from_f<T>(st.y * (gy - m0 - (to_f(x[c]) - st.x) * st.y * m1));
    }
  }
}

// Weight gradients of wide rows: CTA (x, y) sums columns [256 x, 256 x + 256) over rows y, y + gridDim.y, ...
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_dw_wide_kernel(const __grid_constant__ NormArgs a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.cols) return;
  float dg = 0.f, db = 0.f;
  for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float2 st = reinterpret_cast<const float2*>(a.stats)[row];
    const float d = to_f((static_cast<const T*>(a.dy) + row_offset(a.dym, (unsigned)row))[c]);
    const float x = to_f((static_cast<const T*>(a.x) + row_offset(a.xm, (unsigned)row))[c]);
    dg = fmaf(d, (x - st.x) * st.y, dg);
    db += d;
  }
  float* part = a.part + (long long)blockIdx.y * 2 * a.cols;
  part[c] = dg;
  part[a.cols + c] = db;
}

// CTAs of the backward kernel, each of which leaves one partial row of the weights' gradients; 1: none are needed.
int bwd_ctas(long long rows, int cols) {
  if (cols <= WARP_COLS && rows <= ONE_CTA_ROWS) return 1;
  const long long units = cols <= WARP_COLS ? (rows + 7) / 8 : rows;
  const long long most = 2LL * ub::kNumSMs;
  return (int)(units < most ? units : most);
}

// A wide row's sums always take the second kernel.
bool joins(long long rows, int cols) { return cols > CTA_COLS || bwd_ctas(rows, cols) > 1; }

template <typename T, typename TW, int NV, bool ALIGNED, bool WARP>
int launch_one(const NormArgs& a, bool backward, cudaStream_t st) {
  constexpr int PER = NV * 16 / (int)sizeof(T);  // values per thread
  int threads = WARP ? 256 : ((a.cols + PER - 1) / PER + 31) / 32 * 32;
  if (backward) {
    constexpr auto kern = layer_norm_bwd_kernel<T, TW, NV, ALIGNED, WARP>;
    using Rows = Ring<stages_of<T, NV, 2, WARP>(), 2 * NV, ALIGNED>;
    // A call of one CTA takes 16 warps where their rows fit shared memory.
    constexpr int MOST_THREADS = !WARP || Rows::bytes(512) <= 200 * 1024 ? 512 : 256;
    if (WARP && bwd_ctas(a.rows, a.cols) == 1) threads = MOST_THREADS;
    // The most of any width, allowed once: the rows in flight, or the warps' sums.
    constexpr int JOIN = WARP ? MOST_THREADS / 32 * 4 * 32 * PER : 0;
    constexpr int MOST = Rows::bytes(MOST_THREADS) > JOIN ? Rows::bytes(MOST_THREADS) : JOIN;
    if (MOST > 40 * 1024 && allow_smem<kern>(MOST) != cudaSuccess) return (int)cudaGetLastError();
    const int rows = Rows::bytes(threads), join = WARP ? threads / 32 * 4 * a.cols : 0;
    kern<<<bwd_ctas(a.rows, a.cols), threads, rows > join ? rows : join, st>>>(a);
  } else {
    constexpr auto kern = layer_norm_fwd_kernel<T, TW, NV, ALIGNED, WARP>;
    using Rows = Ring<stages_of<T, NV, 1, WARP>(), NV, ALIGNED>;
    constexpr int MOST = Rows::bytes(WARP ? 256 : 512);
    if (MOST > 40 * 1024 && allow_smem<kern>(MOST) != cudaSuccess) return (int)cudaGetLastError();
    const int smem = Rows::bytes(threads);
    // As many CTAs as run at once: each walks the same number of rows, a partial second wave would cost a whole one.
    int per_sm = 1;
    if ((a.rows + 7) / 8 > ub::kNumSMs) cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, smem);
    kern<<<ub::grid_1d(a.rows, WARP ? 8 : 1, (long long)per_sm * ub::kNumSMs), threads, smem, st>>>(a);
  }
  UB_CHECK_LAUNCH();
  return 0;
}

template <typename T, typename TW, bool ALIGNED>
int launch_cols(const NormArgs& a, bool backward, cudaStream_t st) {
  constexpr int N8 = sizeof(T) / 2;  // 16-byte runs of 8 values
  if (a.cols <= 256) return launch_one<T, TW, N8, ALIGNED, true>(a, backward, st);
  if (a.cols <= 512) return launch_one<T, TW, 2 * N8, ALIGNED, true>(a, backward, st);
  if (a.cols <= 768) return launch_one<T, TW, 3 * N8, ALIGNED, true>(a, backward, st);
  if (a.cols <= WARP_COLS) return launch_one<T, TW, 4 * N8, ALIGNED, true>(a, backward, st);
  return launch_one<T, TW, 2 * N8, ALIGNED, false>(a, backward, st);
}

template <typename T, typename TW>
int launch_types(const NormArgs& a, bool vec, bool backward, cudaStream_t st) {
  if (a.cols > CTA_COLS) {
    const unsigned grid = ub::grid_1d(a.rows, 1, 4LL * ub::kNumSMs);
    if (!backward) {
      layer_norm_fwd_wide_kernel<T, TW><<<grid, 512, 0, st>>>(a);
      UB_CHECK_LAUNCH();
      return 0;
    }
    layer_norm_dx_wide_kernel<T, TW><<<grid, 512, 0, st>>>(a);
    UB_CHECK_LAUNCH();
    if (a.dgamma) {
      const dim3 g((a.cols + 255) / 256, bwd_ctas(a.rows, a.cols));
      layer_norm_dw_wide_kernel<T><<<g, 256, 0, st>>>(a);
      UB_CHECK_LAUNCH();
    }
    return 0;
  }
  return vec ? launch_cols<T, TW, true>(a, backward, st) : launch_cols<T, TW, false>(a, backward, st);
}

int launch(const NormArgs& a, int dtype, int w_dtype, bool vec, bool backward, cudaStream_t st) {
  if (dtype == UNBLEND_F32) return launch_types<float, float>(a, vec, backward, st);
  if (dtype == UNBLEND_BF16)
    return w_dtype == UNBLEND_F32 ? launch_types<__nv_bfloat16, float>(a, vec, backward, st)
                                  : launch_types<__nv_bfloat16, __nv_bfloat16>(a, vec, backward, st);
  return w_dtype == UNBLEND_F32 ? launch_types<__half, float>(a, vec, backward, st)
                                : launch_types<__half, __half>(a, vec, backward, st);
}

// The bytes from the first to behind the last value of a tensor's rows.
void span(const void* base, const RowMap& m, long long outer, int cols, int elem, const void** lo, const void** hi) {
  long long first = 0, last = 0;
  for (const long long d : {(outer - 1) * m.so, ((long long)m.inner - 1) * m.si}) (d < 0 ? first : last) += d;
  *lo = static_cast<const char*>(base) + first * elem;
  *hi = static_cast<const char*>(base) + (last + cols) * elem;
}

bool types_ok(int dtype, int w_dtype) {
  return known_type(dtype) && (w_dtype == UNBLEND_F32 || w_dtype == dtype);
}

}  // namespace

extern "C" int unblend_layer_norm_grad_workspace(long long rows, int cols, long long* bytes) {
  UB_REQUIRE(bytes && rows_ok(1, rows, cols));
  *bytes = joins(rows, cols) ? (long long)bwd_ctas(rows, cols) * 2 * cols * (long long)sizeof(float) : 0;
  return 0;
}

extern "C" int unblend_layer_norm_forward(const void* x, long long x_so, long long x_si, void* y, float* stats,
                                          const void* gamma, const void* beta, float eps, long long outer,
                                          long long inner, int cols, int dtype, int w_dtype, void* stream) {
  UB_REQUIRE(x && y && stats && rows_ok(outer, inner, cols) && types_ok(dtype, w_dtype) && eps >= 0.f);
  UB_REQUIRE(reinterpret_cast<uintptr_t>(stats) % sizeof(float2) == 0);
  NormArgs a{};
  a.x = x;
  a.y = y;
  a.stats = stats;
  a.gamma = gamma;
  a.beta = beta;
  a.eps = eps;
  a.xm = row_map(x_so, x_si, inner);
  a.rows = (unsigned)(outer * inner);
  a.cols = cols;
  const int es = elem_size(dtype);
  const bool vec = cols % (16 / es) == 0 && rows_aligned(x, a.xm, outer, es, 16) && aligned16(y);
  a.w_vec = aligned16(gamma) && aligned16(beta);
  span(x, a.xm, outer, cols, es, &a.x_lo, &a.x_hi);
  return launch(a, dtype, w_dtype, vec, false, ub::as_stream(stream));
}

extern "C" int unblend_layer_norm_backward(const void* dy, long long dy_so, long long dy_si, const void* x,
                                           long long x_so, long long x_si, const float* stats, const void* gamma,
                                           void* dx, void* dgamma, void* dbeta, float* work, long long outer,
                                           long long inner, int cols, int dtype, int w_dtype, void* stream) {
  UB_REQUIRE(dy && x && stats && dx && rows_ok(outer, inner, cols) && types_ok(dtype, w_dtype));
  UB_REQUIRE(reinterpret_cast<uintptr_t>(stats) % sizeof(float2) == 0);
  UB_REQUIRE((dgamma != nullptr) == (dbeta != nullptr) && (!dgamma || work || !joins(outer * inner, cols)));
  NormArgs a{};
  a.x = x;
  a.dy = dy;
  a.y = dx;
  a.stats = const_cast<float*>(stats);
  a.gamma = gamma;
  a.dgamma = dgamma;
  a.dbeta = dbeta;
  a.part = dgamma && joins(outer * inner, cols) ? work : nullptr;
  a.xm = row_map(x_so, x_si, inner);
  a.dym = row_map(dy_so, dy_si, inner);
  a.rows = (unsigned)(outer * inner);
  a.cols = cols;
  const int es = elem_size(dtype);
  const bool vec = cols % (16 / es) == 0 && rows_aligned(x, a.xm, outer, es, 16) &&
                   rows_aligned(dy, a.dym, outer, es, 16) && aligned16(dx);
  a.w_vec = aligned16(gamma);
  span(x, a.xm, outer, cols, es, &a.x_lo, &a.x_hi);
  span(dy, a.dym, outer, cols, es, &a.dy_lo, &a.dy_hi);
  cudaStream_t st = ub::as_stream(stream);
  const int rc = launch(a, dtype, w_dtype, vec, true, st);
  if (rc || !a.part) return rc;
  const int parts = bwd_ctas(a.rows, cols);
  if (w_dtype == UNBLEND_F32) return launch_column_sums<float>(work, parts, cols, 2, dgamma, dbeta, st);
  if (w_dtype == UNBLEND_BF16) return launch_column_sums<__nv_bfloat16>(work, parts, cols, 2, dgamma, dbeta, st);
  return launch_column_sums<__half>(work, parts, cols, 2, dgamma, dbeta, st);
}
