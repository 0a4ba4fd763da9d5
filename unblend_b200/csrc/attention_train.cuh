// Shared by the attention kernels with gradients: arguments, addressing, the visible range of a tile and the kernels
// that join the parts of a split axis.
#pragma once

#include "train_common.cuh"

namespace ub {
namespace train {

struct AttnArgs {
  const void *q, *k, *v, *dout;
  const void* out_in;  // forward output, read by the backward pass
  void *out, *dq, *dk, *dv;
  float* lse;
  float* dsum;  // [rows] rowsum(dout * out) (CUDA cores), or [rows][2] row statistics (tensor cores)
  UnblendHeadStrides q_s, k_s, v_s, out_s, dout_s, dq_s, dk_s, dv_s;
  const int *q_lens, *k_lens;
  int seqs, inner, heads, kv_heads, group, lq, lk, hd, causal;
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

__device__ __forceinline__ bool sees(const AttnArgs& a, const Bounds& b, int i, int j) {
  return i < b.ql && j < b.kl && (!a.causal || j <= i + b.off);
}

__device__ __forceinline__ long long head_offset(const UnblendHeadStrides& s, const AttnArgs& a, int seq, int h) {
  const int o = seq / a.inner;
  return (long long)o * s.outer + (long long)(seq - o * a.inner) * s.inner + (long long)h * s.head;
}

// Joins the forward parts of each row: out = sum_s exp(lse_s - lse) out_s. One warp per row, parts in order.
template <typename T>
__global__ void __launch_bounds__(256) attention_join_kernel(const __grid_constant__ AttnArgs a) {
  const int lane = threadIdx.x & 31;
  const long long rows = (long long)a.seqs * a.heads * a.lq;
  const long long row = blockIdx.x * 8LL + (threadIdx.x >> 5);
  if (row >= rows) return;
  float top = -INFINITY;
  for (int s = 0; s < a.splits; ++s) {
    const float l = a.part_lse[s * rows + row];
    if (l > top || l != l) top = l;  // a NaN stays
  }
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, total = 0.f;
  if (top != -INFINITY) {
    for (int s = 0; s < a.splits; ++s) {
      const float l = a.part_lse[s * rows + row];
      if (l == -INFINITY) continue;
      const float w = expf(l - top);
      total += w;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int d = 32 * k + lane;
        if (d < a.hd) acc[k] = fmaf(w, a.part[(s * rows + row) * a.hd + d], acc[k]);
      }
    }
  }
  const float inv = total > 0.f ? 1.f / total : (top != -INFINITY ? total : 0.f);
  const int i = (int)(row % a.lq);
  const long long sh = row / a.lq;
  const int h = (int)(sh % a.heads), seq = (int)(sh / a.heads);
  T* out = static_cast<T*>(a.out) + head_offset(a.out_s, a, seq, h) + i * a.out_s.row;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int d = 32 * k + lane;
    if (d < a.hd) out[d] = from_f<T>(acc[k] * inv);
  }
  if (a.lse && lane == 0) a.lse[row] = top == -INFINITY ? top : top + logf(total);
}

// Adds the parts of a gradient row by row: part [splits][seqs * heads * len][hd] -> out.
template <typename T>
__global__ void __launch_bounds__(256)
    attention_sum_kernel(const __grid_constant__ AttnArgs a, const float* part, int splits, int heads, int len,
                         void* out, const __grid_constant__ UnblendHeadStrides st) {
  const int lane = threadIdx.x & 31;
  const long long rows = (long long)a.seqs * heads * len;
  const long long row = blockIdx.x * 8LL + (threadIdx.x >> 5);
  if (row >= rows) return;
  const long long sh = row / len;
  const int i = (int)(row - sh * len);
  const int h = (int)(sh % heads), seq = (int)(sh / heads);
  T* o = static_cast<T*>(out) + head_offset(st, a, seq, h) + i * st.row;
  for (int d = lane; d < a.hd; d += 32) {
    float t = 0.f;
    for (int s = 0; s < splits; ++s) t += part[(s * rows + row) * a.hd + d];
    o[d] = from_f<T>(t);
  }
}


// The tensor-core kernels (attention_train_tc.cu). `fits`: whether they can address the n tensors of a call.
bool attention_tc_fits(const UnblendAttnTrainParams& p, const void* const* ptrs, const UnblendHeadStrides* strides,
                       const int* heads, const int* rows, int n);
int attention_fwd_tc(const AttnArgs& a, const UnblendAttnTrainParams& p, int rows_per_cta, cudaStream_t st);
int attention_stats_tc(const AttnArgs& a, const UnblendAttnTrainParams& p, cudaStream_t st);
int attention_dq_tc(const AttnArgs& a, const UnblendAttnTrainParams& p, int splits, float* part, cudaStream_t st);
int attention_dkv_tc(const AttnArgs& a, const UnblendAttnTrainParams& p, int splits, float* part, cudaStream_t st);

}  // namespace train
}  // namespace ub
