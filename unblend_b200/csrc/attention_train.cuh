// Shared by the attention kernels with gradients: arguments, addressing, the visible range of a tile and the kernels
// that join the parts of a split axis.
#pragma once

#include "train_common.cuh"

namespace ub {
namespace train {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

struct AttnArgs {
  const void *q, *k, *v, *dout;
  const void* out_in;  // forward output, read by the backward pass
  void *out, *dq, *dk, *dv;
  float* lse;
  float* dsum;  // [rows] rowsum(dout * out) (CUDA cores), or [rows][2] row statistics (tensor cores)
  float* dnorm;     // [rows] norms of the rows of dout (tensor cores, fp16)
  unsigned* range;  // [seqs * kv_heads][4] bits of the largest norm of a row of v and of dout, and |D| (the same)
  UnblendHeadStrides q_s, k_s, v_s, out_s, dout_s, dq_s, dk_s, dv_s;
  const int *q_lens, *k_lens;
  int seqs, inner, heads, kv_heads, group, lq, lk, hd, causal;
  int all_keys;  // backward: lse and out are of these keys alone
  float scale;
  int splits;       // parts of the streamed axis
  float* part;      // [splits][rows][hd] (dk / dv: two of them), null when splits == 1
  float* part_lse;  // [splits][rows], forward
};

struct Bounds {
  int ql, kl, off;  // valid queries and keys; causal: query i sees keys j <= i + off
};

__device__ __forceinline__ Bounds bounds_of(const AttnArgs& a, int seq) {
  Bounds b;
  b.ql = a.q_lens ? min(max(a.q_lens[seq], 0), a.lq) : a.lq;
  b.kl = a.k_lens ? min(max(a.k_lens[seq], 0), a.lk) : a.lk;
  b.off = b.kl - b.ql;
  return b;
}

// Keys [0, end) that some query of [i0, i0 + n) sees.
__device__ __forceinline__ int key_end(const AttnArgs& a, const Bounds& b, int i0, int n) {
  const int last = min(i0 + n, b.ql) - 1;
  if (last < i0) return 0;
  return a.causal ? max(0, min(b.kl, last + b.off + 1)) : b.kl;
}

// First query that sees some key of [j0, ...): queries [begin, b.ql) do.
__device__ __forceinline__ int query_begin(const AttnArgs& a, const Bounds& b, int j0) {
  if (j0 >= b.kl) return b.ql;
  return a.causal ? max(0, j0 - b.off) : 0;
}

// Query i sees keys [0, limit).
__device__ __forceinline__ int key_limit(const AttnArgs& a, const Bounds& b, int i) {
  return i < b.ql ? (a.causal ? min(b.kl, i + b.off + 1) : b.kl) : 0;
}

__device__ __forceinline__ long long head_offset(const UnblendHeadStrides& s, const AttnArgs& a, int seq, int h) {
  const int o = seq / a.inner;
  return (long long)o * s.outer + (long long)(seq - o * a.inner) * s.inner + (long long)h * s.head;
}

// 2^x, the hardware approximation (2 ulp).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// dS = P (dP - D) of fp16 calls is stored times a power of two: unscaled, the gradients of a loss averaged over tokens
// would sink into fp16's subnormals (dout of size 1e-4 over 8192 keys: dq off by 10 %), those of a loss scaled up pass
// its largest value. For values of size `bound` (0 up to infinity; as bits) this is the k for which bound 2^k lies in
// [2^14, 2^15); 40 at most, so that fp32 sums times 2^k stay finite, and 0 where the bound is infinite or NaN.
__device__ __forceinline__ int fp16_shift(unsigned bound_bits) {
  const int e = (int)(bound_bits >> 23) - 127;
  return e > 127 ? 0 : min(14 - e, 40);
}
__device__ __forceinline__ float pow2(int k) { return __uint_as_float((unsigned)(127 + k) << 23); }

// n / d for n < 2^31 by a multiplication: with 2^s >= d and m = floor(2^(31 + s) / d) + 1, floor(n m / 2^(31 + s)) is
// exact because n (m d - 2^(31 + s)) < 2^(31 + s). A hardware division takes a hundred cycles, which short
// units of work do not hide.
struct FastDiv {
  uint32_t d, m, shift;
  __device__ __forceinline__ int operator()(int n) const { return (int)(((uint64_t)(uint32_t)n * m) >> shift); }
};

inline FastDiv fast_div(long long d) {
  FastDiv f;
  uint32_t s = 0;
  while ((1LL << s) < d) ++s;
  f.d = (uint32_t)d;
  f.shift = 31 + s;
  f.m = (uint32_t)((1ULL << f.shift) / (uint64_t)d + 1);
  return f;
}

// Joins the forward parts of each row (at most 32): out = sum_s exp(lse_s - lse) out_s. W warps per row (8 from five
// parts on); lane s weighs part s, warp w adds parts w, w + W, ... (at most 4) and the warps' sums are added in order:
// the loads of all parts are in flight at once. Latency of two dependent loads: 3 us for 64 rows of 32 parts.
constexpr int MAX_PARTS = 32, JOIN_WARPS = 8;

template <typename T, int W>
__global__ void __launch_bounds__(32 * JOIN_WARPS) attention_join_kernel(const __grid_constant__ AttnArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long rows = (long long)a.seqs * a.heads * a.lq;
  const long long row = blockIdx.x * (long long)(JOIN_WARPS / W) + warp / W;
  if (row >= rows) return;  // W = 1: whole warps, no barrier below
  const float l = lane < a.splits ? a.part_lse[lane * rows + row] : -INFINITY;
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, v[4][4];
  const float* part = a.part + row * a.hd + lane;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int s = x * W + warp % W;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      v[x][k] = s < a.splits && 32 * k + lane < a.hd ? part[s * rows * a.hd + 32 * k] : 0.f;
  }
  const bool nan = __any_sync(0xffffffffu, l != l);
  float top = l;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (nan) top = NAN;
  const float w = top == -INFINITY || l == -INFINITY ? 0.f : expf(l - top);
  const float total = ub::warp_sum(w);
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const float ws = __shfl_sync(0xffffffffu, w, x * W + warp % W);
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] = fmaf(ws, v[x][k], acc[k]);
  }
  const float inv = top == -INFINITY ? 0.f : 1.f / total;
  const int i = (int)(row % a.lq);
  const long long sh = row / a.lq;
  const int h = (int)(sh % a.heads), seq = (int)(sh / a.heads);
  T* out = static_cast<T*>(a.out) + head_offset(a.out_s, a, seq, h) + i * a.out_s.row;
  if constexpr (W == 1) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (32 * k + lane < a.hd) out[32 * k + lane] = from_f<T>(acc[k] * inv);
    if (a.lse && lane == 0) a.lse[row] = top == -INFINITY ? top : top + logf(total);
  } else {
    static_assert(W == JOIN_WARPS, "one row per CTA");
    __shared__ float sums[W][128];
#pragma unroll
    for (int k = 0; k < 4; ++k) sums[warp][32 * k + lane] = acc[k];
    __syncthreads();
    if (threadIdx.x < a.hd) {
      float t = 0.f;
#pragma unroll
      for (int x = 0; x < W; ++x) t += sums[x][threadIdx.x];
      out[threadIdx.x] = from_f<T>(t * inv);
    }
    if (a.lse && threadIdx.x == 0) a.lse[row] = top == -INFINITY ? top : top + logf(total);
  }
}

// Adds the parts of the gradients row by row: part [splits][seqs * heads * len][hd] -> out, up to three tensors.
struct SumArgs {
  struct One {
    const float* part;
    void* out;
    UnblendHeadStrides to;
    int splits, heads, len;
    long long rows;
  } of[3];
  long long rows;  // of all
};

template <typename T>
__global__ void __launch_bounds__(256)
    attention_sum_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ SumArgs s) {
  const int lane = threadIdx.x & 31;
  long long row = blockIdx.x * 8LL + (threadIdx.x >> 5);
  if (row >= s.rows) return;
  int w = 0;
  while (row >= s.of[w].rows) row -= s.of[w++].rows;
  const SumArgs::One& x = s.of[w];
  const long long sh = row / x.len;
  const int i = (int)(row - sh * x.len);
  const int h = (int)(sh % x.heads), seq = (int)(sh / x.heads);
  T* o = static_cast<T*>(x.out) + head_offset(x.to, a, seq, h) + i * x.to.row;
  for (int d = lane; d < a.hd; d += 32) {
    float t = 0.f;
#pragma unroll 4
    for (int p = 0; p < x.splits; ++p) t += x.part[(p * x.rows + row) * a.hd + d];
    o[d] = from_f<T>(t);
  }
}

// The tensor-core kernels (attention_train_tc.cu). `sizes`: whether they take a call of this type, head dim and scale;
// `fits`: and can address its n tensors.
bool attention_tc_sizes(const UnblendAttnTrainParams& p);
bool attention_tc_fits(const UnblendAttnTrainParams& p, const void* const* ptrs, const UnblendHeadStrides* strides,
                       const int* heads, const int* rows, int n);
int attention_fwd_tc(const AttnArgs& a, const UnblendAttnTrainParams& p, int rows_per_cta, cudaStream_t st);
int attention_stats_tc(const AttnArgs& a, const UnblendAttnTrainParams& p, cudaStream_t st);
int attention_dq_tc(const AttnArgs& a, const UnblendAttnTrainParams& p, int splits, float* part, cudaStream_t st);
int attention_dkv_tc(const AttnArgs& a, const UnblendAttnTrainParams& p, int splits, float* part, cudaStream_t st);

// Sequences of one tile (attention_train_small.cu), of calls that `attention_tc_fits`.
bool attention_is_small(const UnblendAttnTrainParams& p, bool backward);
int attention_small_forward(const AttnArgs& a, const UnblendAttnTrainParams& p, cudaStream_t st);
int attention_small_backward(const AttnArgs& a, const UnblendAttnTrainParams& p, cudaStream_t st);

}  // namespace train
}  // namespace ub
