// Attention with gradients: entry points, and the fp32 CUDA-core kernels.
//
//   S = scale Q K^T (masked),  lse = log sum_j exp S,  P = exp(S - lse),  O = P V
//   D = rowsum(dO * O),  dV = P^T dO,  dS = P * (dO V^T - D),  dQ = scale dS K,  dK = scale dS^T Q
//
// Nothing of size lq x lk is stored: the forward pass keeps a running maximum and sum per query and leaves lse, the
// backward pass computes P again from it. The backward pass is two kernels, one walking the keys for a tile of
// queries (dQ, and D on the way), one walking the queries of all heads of a group for a tile of keys (dK, dV); each
// output element belongs to one CTA, so nothing is added by atomics and the result is the same on every run, for two
// products more than the five that one kernel with atomics would need.
// When the tiles are too few to fill the GPU the walked axis is split and the parts joined in order by another kernel.
//
// The kernels here take every type, stride and alignment, and are the path of fp32: 64 x 64 score tiles on 256
// threads, 4 x 4 scores per thread, operands in shared memory as fp32 (transposed where the head axis is summed). Bound
// by the shared-memory reads that feed the FP32 pipes (89 % of their rate in the forward kernel, FMA 45 %): 8 x 1344 x
// 1344, 8 heads of 64, fp32 1.09 ms forward (27 TFLOP/s) and 3.32 ms backward (31 TFLOP/s). 4 x 8 scores on 128
// threads halve the reads, but with as few warps were only faster forward at head dim 64 (0.97 ms; backward 3.58 ms,
// at head dim 128 2.62 and 9.17 ms against 2.17 and 7.50 ms).
#include "attention_train.cuh"
#include "warp_mma.cuh"

namespace {

using namespace ub::train;

constexpr int TILE = 64;
constexpr int NT = 256;
constexpr int LD = TILE + 4;  // row pitch of [dim][row] tiles: 16-byte rows, 4-bank shift per dim

// Rows [r0, r0 + 64) of a head into shared memory: transposed [dim][LD] and / or as rows [row][HDP + 4]. Rows from
// `valid` on and dims from hd up to a multiple of 4 become 0. Lane = row, so the transposed stores do not conflict.
template <typename T, int HDP, bool TRANS, bool ROWS>
__device__ __forceinline__ void load_tile(const T* base, long long row_stride, int r0, int valid, int hd, bool vec,
                                          float* trans, float* rows) {
  const int row = threadIdx.x & 63, part = threadIdx.x >> 6;
  const bool in = r0 + row < valid;
  const T* p = base + (long long)(r0 + row) * row_stride;
  for (int d = part * 4; d < hd; d += 16) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (in) {
      if (vec) {
        load_vec<T, 4>(p + d, v);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < hd) v[e] = to_f(p[d + e]);
      }
    }
    if constexpr (TRANS) {
#pragma unroll
      for (int e = 0; e < 4; ++e) trans[(d + e) * LD + row] = v[e];
    }
    if constexpr (ROWS) *reinterpret_cast<float4*>(rows + row * (HDP + 4) + d) = make_float4(v[0], v[1], v[2], v[3]);
  }
}

// acc[r][c] = sum_d A[d][4 ty + r] * B[d][4 tx + c]
__device__ __forceinline__ void mm_nt(float2 (&acc)[4][2], const float* A, const float* B, int hd, int ty, int tx) {
#pragma unroll
  for (int r = 0; r < 4; ++r) acc[r][0] = acc[r][1] = make_float2(0.f, 0.f);
#pragma unroll 4
  for (int d = 0; d < hd; ++d) {
    const float4 a = *reinterpret_cast<const float4*>(A + d * LD + 4 * ty);
    const float4 b = *reinterpret_cast<const float4*>(B + d * LD + 4 * tx);
    const float ar[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float2 rr = make_float2(ar[r], ar[r]);
      acc[r][0] = ub::fma2(rr, make_float2(b.x, b.y), acc[r][0]);
      acc[r][1] = ub::fma2(rr, make_float2(b.z, b.w), acc[r][1]);
    }
  }
}

// acc[r][g] += sum_j W[j][4 ty + r] * B[j][64 g + 4 tx ..]
template <int HDP>
__device__ __forceinline__ void mm_wn(float2 (&acc)[4][HDP / 64][2], const float* W, const float* B, int ty, int tx) {
#pragma unroll 4
  for (int j = 0; j < TILE; ++j) {
    const float4 w = *reinterpret_cast<const float4*>(W + j * LD + 4 * ty);
    const float wr[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int g = 0; g < HDP / 64; ++g) {
      const float4 b = *reinterpret_cast<const float4*>(B + j * (HDP + 4) + 64 * g + 4 * tx);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float2 rr = make_float2(wr[r], wr[r]);
        acc[r][g][0] = ub::fma2(rr, make_float2(b.x, b.y), acc[r][g][0]);
        acc[r][g][1] = ub::fma2(rr, make_float2(b.z, b.w), acc[r][g][1]);
      }
    }
  }
}

template <int HDP>
__device__ __forceinline__ void zero(float2 (&acc)[4][HDP / 64][2]) {
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int g = 0; g < HDP / 64; ++g) acc[r][g][0] = acc[r][g][1] = make_float2(0.f, 0.f);
}

// A thread's 4 x 4 values transposed: S[4 tx + e][4 ty ..].
__device__ __forceinline__ void put_scores(float* S, const float (&v)[4][4], int ty, int tx) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    *reinterpret_cast<float4*>(S + (4 * tx + e) * LD + 4 * ty) = make_float4(v[0][e], v[1][e], v[2][e], v[3][e]);
}

// One accumulator row (64 g + 4 tx + e over all tx, g) times mul to out[d] (T) or to a fp32 part row.
template <typename T, int HDP>
__device__ __forceinline__ void store_row(const float2 (&acc)[HDP / 64][2], float mul, T* out, int hd, int tx) {
#pragma unroll
  for (int g = 0; g < HDP / 64; ++g) {
    const float v[4] = {acc[g][0].x * mul, acc[g][0].y * mul, acc[g][1].x * mul, acc[g][1].y * mul};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 64 * g + 4 * tx + e;
      if (d < hd) out[d] = from_f<T>(v[e]);
    }
  }
}

// Over the 16 lanes (tx) that share a row.
__device__ __forceinline__ float row_max16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float row_sum16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Unit {
  int seq, h, tile, split;
};

__device__ __forceinline__ Unit unit_of(int tiles, int heads, int splits) {
  unsigned u = blockIdx.x;
  Unit r;
  r.split = u % splits;
  u /= splits;
  r.tile = u % tiles;
  u /= tiles;
  r.h = u % heads;
  r.seq = u / heads;
  return r;
}

template <typename T, int HDP>
__global__ void __launch_bounds__(NT) attention_fwd_kernel(const __grid_constant__ AttnArgs a, int vec) {
  extern __shared__ float smem[];
  float* sQ = smem;                      // [HDP][LD]
  float* sK = sQ + HDP * LD;             // [HDP][LD]
  float* sV = sK + HDP * LD;             // [64][HDP + 4]
  float* sP = sV + TILE * (HDP + 4);     // [64 keys][LD]
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const Unit u = unit_of((a.lq + TILE - 1) / TILE, a.heads, a.splits);
  const Bounds b = bounds_of(a, u.seq);
  const int i0 = u.tile * TILE;
  const T* q = static_cast<const T*>(a.q) + head_offset(a.q_s, a, u.seq, u.h);
  const T* k = static_cast<const T*>(a.k) + head_offset(a.k_s, a, u.seq, u.h / a.group);
  const T* v = static_cast<const T*>(a.v) + head_offset(a.v_s, a, u.seq, u.h / a.group);
  const int tiles = (key_end(a, b, i0, TILE) + TILE - 1) / TILE;
  const int t0 = (int)((long long)tiles * u.split / a.splits), t1 = (int)((long long)tiles * (u.split + 1) / a.splits);
  float2 o[4][HDP / 64][2];
  zero<HDP>(o);
  float m[4], l[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) m[r] = -INFINITY, l[r] = 0.f;
  const float c = a.scale * LOG2E;
  const int hd = a.hd;
  if (t0 < t1) load_tile<T, HDP, true, false>(q, a.q_s.row, i0, b.ql, hd, vec, sQ, nullptr);
  for (int t = t0; t < t1; ++t) {
    const int j0 = t * TILE;
    __syncthreads();
    load_tile<T, HDP, true, false>(k, a.k_s.row, j0, b.kl, hd, vec, sK, nullptr);
    load_tile<T, HDP, false, true>(v, a.v_s.row, j0, b.kl, hd, vec, nullptr, sV);
    __syncthreads();
    float2 s[4][2];
    mm_nt(s, sQ, sK, hd, ty, tx);
    float p[4][4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int limit = key_limit(a, b, i0 + 4 * ty + r) - j0;
      float x[4] = {s[r][0].x * c, s[r][0].y * c, s[r][1].x * c, s[r][1].y * c};
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (4 * tx + e >= limit) x[e] = -INFINITY;
        top = fmaxf(top, x[e]);
      }
      top = fmaxf(row_max16(top), m[r]);
      const float base = top == -INFINITY ? 0.f : top;
      const float corr = exp2f(m[r] - base);
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[r][e] = exp2f(x[e] - base);
        sum += p[r][e];
      }
      l[r] = l[r] * corr + row_sum16(sum);
      m[r] = top;
#pragma unroll
      for (int g = 0; g < HDP / 64; ++g)
#pragma unroll
        for (int e = 0; e < 2; ++e) o[r][g][e].x *= corr, o[r][g][e].y *= corr;
    }
    put_scores(sP, p, ty, tx);
    __syncthreads();
    mm_wn<HDP>(o, sP, sV, ty, tx);
  }
  const long long rows = (long long)a.seqs * a.heads * a.lq;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = i0 + 4 * ty + r;
    if (i >= a.lq) continue;
    const long long row = ((long long)u.seq * a.heads + u.h) * a.lq + i;
    const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
    // Scores that are all NaN leave no maximum, but a sum of NaN.
    const float lse = l[r] == 0.f ? -INFINITY : (m[r] + log2f(l[r])) * LN2;
    if (a.splits > 1) {
      store_row<float, HDP>(o[r], inv, a.part + (u.split * rows + row) * hd, hd, tx);
      if (tx == 0) a.part_lse[u.split * rows + row] = lse;
    } else {
      store_row<T, HDP>(o[r], inv,
                        static_cast<T*>(a.out) + head_offset(a.out_s, a, u.seq, u.h) + (long long)i * a.out_s.row, hd,
                        tx);
      if (tx == 0 && a.lse) a.lse[row] = lse;
    }
  }
}

// dQ of 64 queries of one head; D = rowsum(dO * O) on the way (its first split leaves it for the dk / dv kernel).
template <typename T, int HDP>
__global__ void __launch_bounds__(NT) attention_dq_kernel(const __grid_constant__ AttnArgs a, int vec) {
  extern __shared__ float smem[];
  float* sQ = smem;                       // [HDP][LD]
  float* sO = sQ + HDP * LD;              // [HDP][LD] dO
  float* sV = sO + HDP * LD;              // [HDP][LD]
  float* sK = sV + HDP * LD;              // [HDP][LD]
  float* sKr = sK + HDP * LD;             // [64][HDP + 4]
  float* sS = sKr + TILE * (HDP + 4);     // [64 keys][LD]
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const Unit u = unit_of((a.lq + TILE - 1) / TILE, a.heads, a.splits);
  const Bounds b = bounds_of(a, u.seq);
  const int i0 = u.tile * TILE;
  const T* q = static_cast<const T*>(a.q) + head_offset(a.q_s, a, u.seq, u.h);
  const T* dout = static_cast<const T*>(a.dout) + head_offset(a.dout_s, a, u.seq, u.h);
  const T* out = static_cast<const T*>(a.out_in) + head_offset(a.out_s, a, u.seq, u.h);
  const T* k = static_cast<const T*>(a.k) + head_offset(a.k_s, a, u.seq, u.h / a.group);
  const T* v = static_cast<const T*>(a.v) + head_offset(a.v_s, a, u.seq, u.h / a.group);
  const long long row0 = ((long long)u.seq * a.heads + u.h) * a.lq;
  const int tiles = (key_end(a, b, i0, TILE) + TILE - 1) / TILE;
  const int t0 = (int)((long long)tiles * u.split / a.splits), t1 = (int)((long long)tiles * (u.split + 1) / a.splits);
  const int hd = a.hd;
  float D[4], lse[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = i0 + 4 * ty + r;
    float s = 0.f;
    lse[r] = -INFINITY;
    if (i < b.ql) {
      lse[r] = a.lse[row0 + i];
      if (lse[r] != -INFINITY)
        for (int d = tx; d < hd; d += 16)
          s = fmaf(to_f(dout[i * a.dout_s.row + d]), to_f(out[i * a.out_s.row + d]), s);
    }
    D[r] = row_sum16(s);
    if (i < a.lq && tx == 0 && u.split == 0) a.dsum[row0 + i] = D[r];
  }
  float2 acc[4][HDP / 64][2];
  zero<HDP>(acc);
  const float c = a.scale * LOG2E;
  if (t0 < t1) {
    load_tile<T, HDP, true, false>(q, a.q_s.row, i0, b.ql, hd, vec, sQ, nullptr);
    load_tile<T, HDP, true, false>(dout, a.dout_s.row, i0, b.ql, hd, vec, sO, nullptr);
  }
  for (int t = t0; t < t1; ++t) {
    const int j0 = t * TILE;
    __syncthreads();
    load_tile<T, HDP, true, true>(k, a.k_s.row, j0, b.kl, hd, vec, sK, sKr);
    load_tile<T, HDP, true, false>(v, a.v_s.row, j0, b.kl, hd, vec, sV, nullptr);
    __syncthreads();
    float2 s[4][2], dp[4][2];
    mm_nt(s, sQ, sK, hd, ty, tx);
    mm_nt(dp, sO, sV, hd, ty, tx);
    float ds[4][4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int limit = key_limit(a, b, i0 + 4 * ty + r) - j0;
      const float x[4] = {s[r][0].x, s[r][0].y, s[r][1].x, s[r][1].y};
      const float g[4] = {dp[r][0].x, dp[r][0].y, dp[r][1].x, dp[r][1].y};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        ds[r][e] = 4 * tx + e < limit ? exp2f(x[e] * c - lse[r] * LOG2E) * (g[e] - D[r]) : 0.f;
    }
    put_scores(sS, ds, ty, tx);
    __syncthreads();
    mm_wn<HDP>(acc, sS, sKr, ty, tx);
  }
  const long long rows = (long long)a.seqs * a.heads * a.lq;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = i0 + 4 * ty + r;
    if (i >= a.lq) continue;
    if (a.splits > 1)
      store_row<float, HDP>(acc[r], a.scale, a.part + (u.split * rows + row0 + i) * hd, hd, tx);
    else
      store_row<T, HDP>(acc[r], a.scale,
                        static_cast<T*>(a.dq) + head_offset(a.dq_s, a, u.seq, u.h) + (long long)i * a.dq_s.row, hd,
                        tx);
  }
}

// dK and dV of 64 keys of one key/value head: walks the (query head of the group, query tile) pairs.
template <typename T, int HDP>
__global__ void __launch_bounds__(NT) attention_dkv_kernel(const __grid_constant__ AttnArgs a, int vec) {
  extern __shared__ float smem[];
  float* sK = smem;                       // [HDP][LD]
  float* sV = sK + HDP * LD;              // [HDP][LD]
  float* sQ = sV + HDP * LD;              // [HDP][LD]
  float* sO = sQ + HDP * LD;              // [HDP][LD] dO
  float* sQr = sO + HDP * LD;             // [64][HDP + 4]
  float* sOr = sQr + TILE * (HDP + 4);    // [64][HDP + 4]
  float *sP = sQ, *sS = sO;               // [64 queries][LD] P^T and dS^T, once S^T and dP^T are there
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const Unit u = unit_of((a.lk + TILE - 1) / TILE, a.kv_heads, a.splits);
  const Bounds b = bounds_of(a, u.seq);
  const int j0 = u.tile * TILE;
  const T* k = static_cast<const T*>(a.k) + head_offset(a.k_s, a, u.seq, u.h);
  const T* v = static_cast<const T*>(a.v) + head_offset(a.v_s, a, u.seq, u.h);
  const int begin = query_begin(a, b, j0) / TILE;
  const int per_head = j0 < b.kl ? max(0, (b.ql + TILE - 1) / TILE - begin) : 0;
  const int total = per_head * a.group;
  const int t0 = (int)((long long)total * u.split / a.splits), t1 = (int)((long long)total * (u.split + 1) / a.splits);
  const int hd = a.hd;
  const float c = a.scale * LOG2E;
  float2 dk[4][HDP / 64][2], dv[4][HDP / 64][2];
  zero<HDP>(dk);
  zero<HDP>(dv);
  if (t0 < t1) {
    load_tile<T, HDP, true, false>(k, a.k_s.row, j0, b.kl, hd, vec, sK, nullptr);
    load_tile<T, HDP, true, false>(v, a.v_s.row, j0, b.kl, hd, vec, sV, nullptr);
  }
  // Rows that see no key have P = 0 whatever they hold: cut away, so that NaN in them stays out of the sums.
  const int first = a.causal ? max(0, -b.off) : 0;
  for (int t = t0; t < t1; ++t) {
    const int h = u.h * a.group + t / per_head;
    const int i0 = (begin + t % per_head) * TILE;
    const T* q = static_cast<const T*>(a.q) + head_offset(a.q_s, a, u.seq, h);
    const T* dout = static_cast<const T*>(a.dout) + head_offset(a.dout_s, a, u.seq, h);
    const long long row0 = ((long long)u.seq * a.heads + h) * a.lq;
    __syncthreads();
    load_tile<T, HDP, true, true>(q, a.q_s.row, i0, b.ql, hd, vec, sQ, sQr);
    load_tile<T, HDP, true, true>(dout, a.dout_s.row, i0, b.ql, hd, vec, sO, sOr);
    __syncthreads();
    if (i0 < first) {
      for (int e = threadIdx.x; e < (first - i0 < TILE ? first - i0 : TILE) * (HDP + 4); e += NT) sQr[e] = sOr[e] = 0.f;
      __syncthreads();
    }
    float2 s[4][2], dp[4][2];
    mm_nt(s, sK, sQ, hd, ty, tx);
    mm_nt(dp, sV, sO, hd, ty, tx);
    float p[4][4], ds[4][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = i0 + 4 * tx + e, limit = key_limit(a, b, i) - j0;
      const float lse = i < b.ql ? a.lse[row0 + i] * LOG2E : 0.f, D = i < b.ql ? a.dsum[row0 + i] : 0.f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float x = e & 1 ? s[r][e / 2].y : s[r][e / 2].x, g = e & 1 ? dp[r][e / 2].y : dp[r][e / 2].x;
        const bool on = 4 * ty + r < limit;
        p[r][e] = on ? exp2f(x * c - lse) : 0.f;
        ds[r][e] = on ? p[r][e] * (g - D) : 0.f;
      }
    }
    __syncthreads();
    put_scores(sP, p, ty, tx);
    put_scores(sS, ds, ty, tx);
    __syncthreads();
    mm_wn<HDP>(dv, sP, sOr, ty, tx);
    mm_wn<HDP>(dk, sS, sQr, ty, tx);
  }
  const long long rows = (long long)a.seqs * a.kv_heads * a.lk;
  const long long row0 = ((long long)u.seq * a.kv_heads + u.h) * a.lk;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int j = j0 + 4 * ty + r;
    if (j >= a.lk) continue;
    if (a.splits > 1) {
      store_row<float, HDP>(dk[r], a.scale, a.part + (u.split * rows + row0 + j) * hd, hd, tx);
      store_row<float, HDP>(dv[r], 1.f, a.part + ((a.splits + u.split) * rows + row0 + j) * hd, hd, tx);
    } else {
      store_row<T, HDP>(dk[r], a.scale,
                        static_cast<T*>(a.dk) + head_offset(a.dk_s, a, u.seq, u.h) + (long long)j * a.dk_s.row, hd,
                        tx);
      store_row<T, HDP>(dv[r], 1.f,
                        static_cast<T*>(a.dv) + head_offset(a.dv_s, a, u.seq, u.h) + (long long)j * a.dv_s.row, hd,
                        tx);
    }
  }
}

// ------------------------------------------------------------------------------------------- few queries
//
// Forward for at most 8 rows per key/value head (query heads of the group times queries), fp32: single new tokens over
// a long context. Bound by reading K and V once: a key's 8 hd bytes serve 4 hd flops per row, far too little for a tile
// of 128 rows. LANES lanes share a key, 8 dims each, so that O of all rows fits few registers and many warps an SM; a
// group of lanes holds FEW_KEYS keys of K and V in flight, sums their scores over its lanes and keeps its own running
// maximum, sum and O, joined at the end over the groups and warps. The key range is split over many CTAs;
// attention_join_kernel joins those. 4 x 8191 keys, 16 over 4 heads of 128, fp32: 40 us with the join (3.4 TB/s).
constexpr int FEW_ROWS = 8, FEW_NT = 128, FEW_KEYS = 4, FEW_STAGES = 3;

// K and V of a thread's keys in flight: FEW_STAGES x FEW_KEYS x (K, V) x 32 bytes.
constexpr int FEW_SMEM = FEW_STAGES * FEW_KEYS * 2 * 8 * (int)sizeof(float) * FEW_NT;

template <int HD, int R>
__global__ void __launch_bounds__(FEW_NT) attention_few_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int LANES = HD / 8, GROUPS = 32 / LANES;
  constexpr int V = 4, CH = 2;  // elements per chunk, chunks per lane
  constexpr int WARPS = FEW_NT / 32;
  __shared__ float sq[R][HD];
  __shared__ float so[WARPS][R][HD + 2];  // O, maximum, sum of each warp
  extern __shared__ uint4 ring[];  // [stage][key][chunk][K, V][thread]: a thread reads what it copied itself
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % LANES, grp = lane / LANES;
  const int split = blockIdx.x % a.splits, sh = blockIdx.x / a.splits;
  const int seq = sh / a.kv_heads, hk = sh - seq * a.kv_heads;
  const Bounds b = bounds_of(a, seq);
  const int n_rows = a.group * a.lq;  // row r: head hk * group + r / lq, query r % lq
  const float c = a.scale * LOG2E;
  for (int x = threadIdx.x; x < R * HD; x += FEW_NT) {
    const int r = x / HD, d = x - r * HD;
    float v = 0.f;
    if (r < n_rows && r % a.lq < b.ql && d < a.hd)
      v = (static_cast<const float*>(a.q) + head_offset(a.q_s, a, seq, hk * a.group + r / a.lq) +
           (long long)(r % a.lq) * a.q_s.row)[d] * c;
    sq[r][d] = v;
  }
  __syncthreads();
  const int keys = key_end(a, b, 0, a.lq);
  const int begin = (int)((long long)keys * split / a.splits), end = (int)((long long)keys * (split + 1) / a.splits);
  const float* k = static_cast<const float*>(a.k) + head_offset(a.k_s, a, seq, hk);
  const float* v = static_cast<const float*>(a.v) + head_offset(a.v_s, a, seq, hk);
  float o[R][CH * V], m[R], l[R];
  int limit[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
    const int i = r % a.lq;
    limit[r] = r < n_rows && i < b.ql ? (a.causal ? min(b.kl, i + b.off + 1) : b.kl) : 0;
#pragma unroll
    for (int e = 0; e < CH * V; ++e) o[r][e] = 0.f;
  }
  constexpr int STEP = WARPS * GROUPS * FEW_KEYS;
  auto at = [&](int stage, int u, int x, int kv) {
    return ring + (((stage * FEW_KEYS + u) * CH + x) * 2 + kv) * FEW_NT + threadIdx.x;
  };
  auto fetch = [&](int stage, int j0) {
#pragma unroll
    for (int u = 0; u < FEW_KEYS; ++u) {
      const int j = j0 + (u * WARPS + warp) * GROUPS + grp;
#pragma unroll
      for (int x = 0; x < CH; ++x) {
        const int d = (x * LANES + sub) * V;
        if (j < end && d < a.hd) {
          cp_async16(at(stage, u, x, 0), k + (long long)j * a.k_s.row + d);
          cp_async16(at(stage, u, x, 1), v + (long long)j * a.v_s.row + d);
        } else if (j0 < end) {
          *at(stage, u, x, 0) = *at(stage, u, x, 1) = make_uint4(0, 0, 0, 0);
        }
      }
    }
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < FEW_STAGES - 1; ++i) fetch(i, begin + i * STEP);
  for (int j0 = begin, stage = 0; j0 < end; j0 += STEP, stage = (stage + 1) % FEW_STAGES) {
    fetch((stage + FEW_STAGES - 1) % FEW_STAGES, j0 + (FEW_STAGES - 1) * STEP);
    cp_wait<FEW_STAGES - 1>();
    float s[FEW_KEYS][R];
#pragma unroll
    for (int u = 0; u < FEW_KEYS; ++u)
#pragma unroll
      for (int r = 0; r < R; ++r) s[u][r] = 0.f;
#pragma unroll
    for (int x = 0; x < CH; ++x)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float4 qw = *reinterpret_cast<const float4*>(&sq[r][(x * LANES + sub) * V]);
        const float q[V] = {qw.x, qw.y, qw.z, qw.w};
#pragma unroll
        for (int u = 0; u < FEW_KEYS; ++u) {
          const float4 w = *reinterpret_cast<const float4*>(at(stage, u, x, 0));
          const float e[V] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int i = 0; i < V; ++i) s[u][r] = fmaf(q[i], e[i], s[u][r]);
        }
      }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = m[r];
#pragma unroll
      for (int u = 0; u < FEW_KEYS; ++u) {
#pragma unroll
        for (int w = LANES / 2; w > 0; w >>= 1) s[u][r] += __shfl_xor_sync(0xffffffffu, s[u][r], w);
        const int j = j0 + (u * WARPS + warp) * GROUPS + grp;
        if (j >= end || j >= limit[r]) s[u][r] = -INFINITY;
        top = fmaxf(top, s[u][r]);
      }
      const float base = top == -INFINITY ? 0.f : top;
      const float corr = exp2f(m[r] - base);
      m[r] = top;
      l[r] *= corr;
#pragma unroll
      for (int e = 0; e < CH * V; ++e) o[r][e] *= corr;
#pragma unroll
      for (int u = 0; u < FEW_KEYS; ++u) {
        s[u][r] = exp2f(s[u][r] - base);
        l[r] += s[u][r];
      }
    }
#pragma unroll
    for (int u = 0; u < FEW_KEYS; ++u)
#pragma unroll
      for (int x = 0; x < CH; ++x) {
        const float4 w = *reinterpret_cast<const float4*>(at(stage, u, x, 1));
        const float e[V] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
          for (int r = 0; r < R; ++r) o[r][x * V + i] = fmaf(s[u][r], e[i], o[r][x * V + i]);
      }
  }
  // The groups of a warp, then the warps.
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float top = m[r];
#pragma unroll
    for (int w = LANES; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    const float f = m[r] == -INFINITY && l[r] == l[r] ? 0.f : exp2f(m[r] - (top == -INFINITY ? 0.f : top));
    l[r] *= f;
#pragma unroll
    for (int w = LANES; w < 32; w <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], w);
#pragma unroll
    for (int e = 0; e < CH * V; ++e) {
      float x = o[r][e] * f;
#pragma unroll
      for (int w = LANES; w < 32; w <<= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
      if (grp == 0) so[warp][r][((e / V) * LANES + sub) * V + e % V] = x;
    }
    if (lane == 0) {
      so[warp][r][HD] = top;
      so[warp][r][HD + 1] = l[r];
    }
  }
  __syncthreads();
  const long long rows = (long long)a.seqs * a.heads * a.lq;
  for (int x = threadIdx.x; x < n_rows * HD; x += FEW_NT) {
    const int r = x / HD, d = x - r * HD;
    float top = -INFINITY, total = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, so[w][r][HD]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float lw = so[w][r][HD + 1];
      const float f = so[w][r][HD] == -INFINITY && lw == lw ? 0.f : exp2f(so[w][r][HD] - base);
      total += lw * f;
      acc = fmaf(so[w][r][d], f, acc);
    }
    const int h = hk * a.group + r / a.lq, i = r % a.lq;
    const long long row = ((long long)seq * a.heads + h) * a.lq + i;
    const float out = total == 0.f ? 0.f : acc / total;
    const float lse = total == 0.f ? -INFINITY : (top + log2f(total)) * LN2;
    if (a.splits > 1) {
      if (d < a.hd) a.part[(split * rows + row) * a.hd + d] = out;
      if (d == 0) a.part_lse[split * rows + row] = lse;
    } else {
      if (d < a.hd)
        (static_cast<float*>(a.out) + head_offset(a.out_s, a, seq, h) + (long long)i * a.out_s.row)[d] = out;
      if (d == 0 && a.lse) a.lse[row] = lse;
    }
  }
}

// The same for 16-bit types on mma.sync, up to 16 rows per key/value head: on the CUDA cores the products and the sums
// over lanes took 170 instructions per key, which bound the kernel (22 us where the reads take 5); here 16 keys take
// about 90 (4 x 8191 keys, 16 over 4 heads of 128: 20 us and 3 for the join, 2.9 TB/s). Rows are the M = 16 of
// m16n8k16: Q stays in registers as A, K rows are B of the scores, P goes from the score fragments into A of P V as it
// is, V^T comes by transposing loads. tcgen05's 128 rows would leave most lanes idle and wants P in TMEM for tiles too
// small to hide that. Each warp has its own ring of 16-key tiles and its own maxima, sums and O: no barrier until the
// end. 16-byte chunk c of a row lies at c ^ (row & 7).
constexpr int MMA_ROWS = 16, MMA_STAGES = 3;
constexpr int few_mma_smem(int hd) { return (FEW_NT / 32) * MMA_STAGES * 2 * 16 * hd * 2; }

template <typename T, int HD>
__global__ void __launch_bounds__(FEW_NT) attention_few_mma_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int WARPS = FEW_NT / 32, CHUNKS = HD / 8, TILE_E = 16 * HD;  // a K or V tile: 16 keys
  extern __shared__ __align__(128) uint8_t few_smem_raw[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane >> 2, ql = lane & 3;
  T* tiles = reinterpret_cast<T*>(few_smem_raw) + warp * MMA_STAGES * 2 * TILE_E;
  const int split = blockIdx.x % a.splits, sh = blockIdx.x / a.splits;
  const int seq = sh / a.kv_heads, hk = sh - seq * a.kv_heads;
  const Bounds b = bounds_of(a, seq);
  const int n_rows = a.group * a.lq;  // row r: head hk * group + r / lq, query r % lq
  const int keys = key_end(a, b, 0, a.lq);
  const int begin = (int)((long long)keys * split / a.splits), end = (int)((long long)keys * (split + 1) / a.splits);
  const T* k = static_cast<const T*>(a.k) + head_offset(a.k_s, a, seq, hk);
  const T* v = static_cast<const T*>(a.v) + head_offset(a.v_s, a, seq, hk);
  auto fetch = [&](int stage, int j0) {  // keys j0 .. j0 + 15
    if (j0 < end) {
      T* d = tiles + stage * 2 * TILE_E;
#pragma unroll
      for (int x = 0; x < 16 * CHUNKS / 32; ++x) {
        const int id = x * 32 + lane, row = id / CHUNKS, c = id % CHUNKS, j = j0 + row;
        const bool in = j < end && 8 * c < a.hd;
        const int to = row * HD + ((c ^ (row & 7)) * 8);
        cp_async16_or_zero(smem_at(d + to), in ? k + (long long)j * a.k_s.row + 8 * c : k, in);
        cp_async16_or_zero(smem_at(d + TILE_E + to), in ? v + (long long)j * a.v_s.row + 8 * c : v, in);
      }
    }
    cp_commit();
  };
  constexpr int STEP = WARPS * 16;
  const int first = begin + warp * 16;
#pragma unroll
  for (int i = 0; i < MMA_STAGES - 1; ++i) fetch(i, first + i * STEP);
  // Q as A fragments: rows quad and quad + 8, dims 16 ks + 2 ql + {0, 1} and + 8.
  uint32_t qf[HD / 16][4];
  int limit[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int r = quad + 8 * x, i = r % a.lq;
    const bool in = r < n_rows && i < b.ql;
    limit[x] = in ? (a.causal ? min(b.kl, i + b.off + 1) : b.kl) : 0;
    const T* q = static_cast<const T*>(a.q) +
                 (in ? head_offset(a.q_s, a, seq, hk * a.group + r / a.lq) + (long long)i * a.q_s.row : 0);
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int d = 16 * ks + 8 * y + 2 * ql;
        alignas(4) T e[2] = {from_f<T>(0.f), from_f<T>(0.f)};
        if (in && d < a.hd) e[0] = q[d];
        if (in && d + 1 < a.hd) e[1] = q[d + 1];
        qf[ks][2 * y + x] = *reinterpret_cast<const uint32_t*>(e);
      }
  }
  const float c = a.scale * LOG2E;
  float o[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int n = 0; n < HD / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
  const int mi = lane >> 3, mr = lane & 7;  // matrix and row that this lane addresses
  for (int j0 = first, stage = 0; j0 < end; j0 += STEP, stage = (stage + 1) % MMA_STAGES) {
    fetch((stage + MMA_STAGES - 1) % MMA_STAGES, j0 + (MMA_STAGES - 1) * STEP);
    cp_wait<MMA_STAGES - 1>();
    __syncwarp();
    const T* tk = tiles + stage * 2 * TILE_E;
    const T* tv = tk + TILE_E;
    float s[2][4];  // keys 8 n + 2 ql + {0, 1} of rows quad, quad + 8
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) {
      const int row = (mi >> 1) * 8 + mr;
      uint32_t f[4];
      ldmatrix4(f, smem_at(tk + row * HD + (((2 * ks + (mi & 1)) ^ mr) * 8)));
      mma16(s[0], qf[ks], f[0], f[1], T());
      mma16(s[1], qf[ks], f[2], f[3], T());
    }
    float p[2][4];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float top = m[x];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = j0 + 8 * n + 2 * ql + e;
          float& z = s[n][2 * x + e];
          z = j < end && j < limit[x] ? z * c : -INFINITY;
          top = fmaxf(top, z);
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float base = top == -INFINITY ? 0.f : top;
      const float corr = exp2f(m[x] - base);
      m[x] = top;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          p[n][2 * x + e] = exp2f(s[n][2 * x + e] - base);
          sum += p[n][2 * x + e];
        }
      l[x] = l[x] * corr + sum;  // this lane's keys
#pragma unroll
      for (int n = 0; n < HD / 8; ++n) o[n][2 * x] *= corr, o[n][2 * x + 1] *= corr;
    }
    const uint32_t pf[4] = {pack_pair<T>(p[0][0], p[0][1]), pack_pair<T>(p[0][2], p[0][3]),
                            pack_pair<T>(p[1][0], p[1][1]), pack_pair<T>(p[1][2], p[1][3])};
#pragma unroll
    for (int d = 0; d < HD / 16; ++d) {
      const int row = (mi & 1) * 8 + mr;
      uint32_t f[4];
      ldmatrix4_trans(f, smem_at(tv + row * HD + (((2 * d + (mi >> 1)) ^ mr) * 8)));
      mma16(o[2 * d], pf, f[0], f[1], T());
      mma16(o[2 * d + 1], pf, f[2], f[3], T());
    }
    __syncwarp();  // the tile is overwritten by the next but one fetch
  }
  // Warps join through shared memory, over the tiles: [warp][row][HD + 2].
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  float* so = reinterpret_cast<float*>(few_smem_raw);
  auto at = [&](int w, int r) { return so + (w * MMA_ROWS + r) * (HD + 2); };
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    float* to = at(warp, quad + 8 * x);
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) {
      to[8 * n + 2 * ql] = o[n][2 * x];
      to[8 * n + 2 * ql + 1] = o[n][2 * x + 1];
    }
    if (ql == 0) {
      to[HD] = m[x];
      to[HD + 1] = l[x];
    }
  }
  __syncthreads();
  const long long rows = (long long)a.seqs * a.heads * a.lq;
  for (int r = warp; r < n_rows; r += WARPS) {
    float top = -INFINITY, total = 0.f, f[WARPS];
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, at(w, r)[HD]);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float mw = at(w, r)[HD], lw = at(w, r)[HD + 1];
      f[w] = mw == -INFINITY && lw == lw ? 0.f : exp2f(mw - (top == -INFINITY ? 0.f : top));
      total += lw * f[w];
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const float lse = total == 0.f ? -INFINITY : (top + log2f(total)) * LN2;
    const int h = hk * a.group + r / a.lq, i = r % a.lq;
    const long long row = ((long long)seq * a.heads + h) * a.lq + i;
    T* out = static_cast<T*>(a.out) + head_offset(a.out_s, a, seq, h) + (long long)i * a.out_s.row;
    for (int d = lane; d < a.hd; d += 32) {
      float acc = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) acc = fmaf(at(w, r)[d], f[w], acc);
      if (a.splits > 1)
        a.part[(split * rows + row) * a.hd + d] = acc * inv;
      else
        out[d] = from_f<T>(acc * inv);
    }
    if (lane == 0) {
      if (a.splits > 1)
        a.part_lse[split * rows + row] = lse;
      else if (a.lse)
        a.lse[row] = lse;
    }
  }
}
static_assert(few_mma_smem(64) >= (FEW_NT / 32) * MMA_ROWS * (64 + 2) * 4, "the join uses the tiles' memory");

constexpr int fwd_smem(int hdp) { return 4 * (2 * hdp * LD + TILE * (hdp + 4) + TILE * LD); }
constexpr int dq_smem(int hdp) { return 4 * (4 * hdp * LD + TILE * (hdp + 4) + TILE * LD); }
constexpr int dkv_smem(int hdp) { return 4 * (4 * hdp * LD + 2 * TILE * (hdp + 4)); }
static_assert(dkv_smem(128) <= 227 * 1024 && dq_smem(128) <= 227 * 1024, "shared memory of one CTA");

long long div_up(long long a, long long b) { return (a + b - 1) / b; }

// Parts of the walked axis (`tiles` long) for units that do not fill the `slots` CTAs that run at once: as many as make
// the last CTA end first, fewer where that is equal.
int split_count(long long units, long long tiles, long long slots) {
  if (units >= slots || tiles <= 1) return 1;
  long long best = 1, least = tiles;
  const long long most = tiles < MAX_PARTS ? tiles : MAX_PARTS;
  for (int waves = 1; waves <= 4; ++waves) {
    const long long n = slots * waves / units, part = div_up(tiles, n < most ? n : most);  // n >= 1: units < slots
    if (waves * part < least) least = waves * part, best = div_up(tiles, part);
    if (n >= most) break;
  }
  return (int)best;
}

long long round4(long long n) { return (n + 3) / 4 * 4; }

// What a call runs on. A few rows per key/value head (forward): see attention_few_kernel. SMALL: sequences of one tile.
enum Path { CUDA_CORES = 0, TENSOR_CORES = 1, FEW = 2, SMALL = 3 };

// Work division of a call.
struct Plan {
  int fwd_rows;  // queries per CTA of the forward kernel
  int fwd_splits, dq_splits, dkv_splits;
  long long q_rows, k_rows;
};

Plan plan_of(const UnblendAttnTrainParams& p, Path path) {
  const bool tc = path == TENSOR_CORES;
  Plan n;
  const long long seqs = (long long)p.outer * p.inner, qh = seqs * p.heads, kh = seqs * p.kv_heads;
  const long long tile = tc ? 128 : TILE;
  const long long qt = div_up(p.lq, tile), kt = div_up(p.lk, tile);
  const long long sms = ub::kNumSMs, group = p.heads / p.kv_heads;
  n.q_rows = qh * p.lq;
  n.k_rows = kh * p.lk;
  n.fwd_splits = n.dq_splits = n.dkv_splits = 1;
  if (path == SMALL) return n;
  n.fwd_rows = (int)tile;
  // 256 queries per CTA halve the reads of K and V tiles, which only pays for wide heads and long rows: at head dim 128
  // 2048 x 2048 253 us against 267 us, 1536 169 against 170, 1024 88 against 86 (801: 134 against 118); at head dim 64
  // 8192 x 8192 448 against 414 us, 62 x 801 x 801 211 against 172 us (two CTAs per SM fill each other's waits).
  if (tc && p.hd > 64 && p.lk > 1024 && p.lq > 128 && qh * div_up(p.lq, 256) >= sms) n.fwd_rows = 256;
  n.fwd_splits = n.fwd_rows == 256 ? 1 : split_count(qh * qt, kt, 2 * sms);
  // Few rows: CTAs of 128 keys at least, twice as many as run at once, for sequences of unequal lengths.
  if (path == FEW) {
    const long long most = div_up(p.lk, 128), fill = div_up(4 * sms, kh);
    n.fwd_splits = (int)(fill < most ? (fill < MAX_PARTS ? fill : MAX_PARTS) : (most < MAX_PARTS ? most : MAX_PARTS));
  }
  n.dq_splits = split_count(qh * qt, kt, tc ? sms : 2 * sms);
  n.dkv_splits = split_count(kh * kt, qt * group, tc ? sms : 2 * sms);
  return n;
}

// Few rows per key/value head, of whole 16-byte chunks: what the sizes alone say.
bool few_rows_fit(const UnblendAttnTrainParams& p) {
  const int most = p.dtype == UNBLEND_F32 ? FEW_ROWS : MMA_ROWS;
  return (long long)p.heads / p.kv_heads * p.lq <= most && p.hd % (16 / elem_size(p.dtype)) == 0;
}

// Workspace: forward [parts][q_rows][hd] and [parts][q_rows] lse; backward D or row statistics [q_rows][2], for fp16
// norms [q_rows] and ranges [seqs * kv_heads][4], then the parts of dq and of dk and dv, which one kernel joins. Room
// for each kind of kernels that the sizes allow: which of them runs depends on the pointers too.
long long norm_floats(const UnblendAttnTrainParams& p, const Plan& n) {
  return p.dtype == UNBLEND_F16 ? round4(n.q_rows) : 0;
}

long long stats_floats(const UnblendAttnTrainParams& p, const Plan& n) {
  const long long ranges = p.dtype == UNBLEND_F16 ? 4LL * p.outer * p.inner * p.kv_heads : 0;
  return round4(2 * n.q_rows) + norm_floats(p, n) + ranges;
}

long long dq_part_floats(const UnblendAttnTrainParams& p, const Plan& n) {
  return n.dq_splits > 1 ? round4(n.dq_splits * n.q_rows * p.hd) : 0;
}

long long workspace_floats(const UnblendAttnTrainParams& p, bool backward) {
  long long most = 0;
  for (const Path path : {CUDA_CORES, TENSOR_CORES, FEW}) {
    if (path == TENSOR_CORES && !attention_tc_sizes(p)) continue;
    if (path == FEW && (backward || !few_rows_fit(p))) continue;
    const Plan n = plan_of(p, path);
    long long need;
    if (!backward) {
      need = n.fwd_splits > 1 ? n.fwd_splits * n.q_rows * (p.hd + 1LL) : 0;
    } else {
      need = stats_floats(p, n) + dq_part_floats(p, n);
      if (n.dkv_splits > 1) need += 2 * n.dkv_splits * n.k_rows * p.hd;
    }
    most = need > most ? need : most;
  }
  return most;
}

bool params_ok(const UnblendAttnTrainParams* p) {
  if (!p || !known_type(p->dtype)) return false;
  if (p->outer <= 0 || p->inner <= 0 || p->heads <= 0 || p->kv_heads <= 0 || p->lq <= 0 || p->lk <= 0) return false;
  if (p->hd <= 0 || p->hd > 128 || p->heads % p->kv_heads != 0) return false;
  if (p->lq >= (1 << 30) || p->lk >= (1 << 30)) return false;
  const long long seqs = (long long)p->outer * p->inner;
  if (seqs >= (1LL << 31)) return false;
  // CTAs of each kernel, splits included (at most 32).
  const long long qt = div_up(p->lq, TILE), kt = div_up(p->lk, TILE);
  return seqs <= (1LL << 31) / p->heads / qt / 32 && seqs <= (1LL << 31) / p->kv_heads / kt / 32 &&
         qt * (p->heads / p->kv_heads) < (1LL << 26) && seqs * p->lq <= (1LL << 38) / p->heads;
}

bool vec4_ok(const void* p, const UnblendHeadStrides& s, const UnblendAttnTrainParams& a) {
  const int w = 4 * elem_size(a.dtype);
  auto fits = [&](long long st, int n) { return n <= 1 || st % 4 == 0; };
  return reinterpret_cast<uintptr_t>(p) % w == 0 && fits(s.outer, a.outer) && fits(s.inner, a.inner) &&
         s.row % 4 == 0 && s.head % 4 == 0;
}

// Few rows per key/value head, K and V in 16-byte chunks.
bool few_fits(const UnblendAttnTrainParams& p, const void* k, const void* v) {
  const int e = 16 / elem_size(p.dtype);
  if (!few_rows_fit(p)) return false;
  for (const UnblendHeadStrides* s : {&p.k, &p.v})
    if ((p.lk > 1 && s->row % e != 0) || (p.kv_heads > 1 && s->head % e != 0) || (p.inner > 1 && s->inner % e != 0) ||
        (p.outer > 1 && s->outer % e != 0))
      return false;
  return aligned16(k) && aligned16(v);
}

AttnArgs args_of(const UnblendAttnTrainParams& p) {
  AttnArgs a{};
  a.q_s = p.q;
  a.k_s = p.k;
  a.v_s = p.v;
  a.out_s = p.out;
  a.dout_s = p.dout;
  a.dq_s = p.dq;
  a.dk_s = p.dk;
  a.dv_s = p.dv;
  a.q_lens = p.q_lens;
  a.k_lens = p.k_lens;
  a.seqs = p.outer * p.inner;
  a.inner = p.inner;
  a.heads = p.heads;
  a.kv_heads = p.kv_heads;
  a.group = p.heads / p.kv_heads;
  a.lq = p.lq;
  a.lk = p.lk;
  a.hd = p.hd;
  a.causal = p.causal ? 1 : 0;
  a.all_keys = p.all_keys ? 1 : 0;
  a.scale = p.scale;
  a.splits = 1;
  return a;
}

template <typename T, int HDP>
int simt_forward(const AttnArgs& a, bool vec, cudaStream_t st) {
  const long long units = (long long)a.seqs * a.heads * div_up(a.lq, TILE) * a.splits;
  if (allow_smem<attention_fwd_kernel<T, HDP>>(fwd_smem(HDP)) != cudaSuccess) return (int)cudaGetLastError();
  attention_fwd_kernel<T, HDP><<<(unsigned)units, NT, fwd_smem(HDP), st>>>(a, vec);
  UB_CHECK_LAUNCH();
  return 0;
}

template <typename T, int HDP>
int simt_dq(AttnArgs a, int splits, float* parts, bool vec, cudaStream_t st) {
  a.splits = splits;
  a.part = parts;
  const long long units = (long long)a.seqs * a.heads * div_up(a.lq, TILE) * splits;
  if (allow_smem<attention_dq_kernel<T, HDP>>(dq_smem(HDP)) != cudaSuccess) return (int)cudaGetLastError();
  attention_dq_kernel<T, HDP><<<(unsigned)units, NT, dq_smem(HDP), st>>>(a, vec);
  UB_CHECK_LAUNCH();
  return 0;
}

template <typename T, int HDP>
int simt_dkv(AttnArgs a, int splits, float* parts, bool vec, cudaStream_t st) {
  a.splits = splits;
  a.part = parts;
  const long long units = (long long)a.seqs * a.kv_heads * div_up(a.lk, TILE) * splits;
  if (allow_smem<attention_dkv_kernel<T, HDP>>(dkv_smem(HDP)) != cudaSuccess) return (int)cudaGetLastError();
  attention_dkv_kernel<T, HDP><<<(unsigned)units, NT, dkv_smem(HDP), st>>>(a, vec);
  UB_CHECK_LAUNCH();
  return 0;
}

template <int HD, int R>
int few_forward(const AttnArgs& a, cudaStream_t st) {
  const long long grid = (long long)a.seqs * a.kv_heads * a.splits;
  if (allow_smem<attention_few_kernel<HD, R>>(FEW_SMEM) != cudaSuccess) return (int)cudaGetLastError();
  attention_few_kernel<HD, R><<<(unsigned)grid, FEW_NT, FEW_SMEM, st>>>(a);
  UB_CHECK_LAUNCH();
  return 0;
}

template <int HD>
int few_rows(const AttnArgs& a, cudaStream_t st) {
  const int rows = a.group * a.lq;
  if (rows == 1) return few_forward<HD, 1>(a, st);
  if (rows == 2) return few_forward<HD, 2>(a, st);
  if (rows <= 4) return few_forward<HD, 4>(a, st);
  return few_forward<HD, 8>(a, st);
}

template <typename T, int HD>
int few_mma(const AttnArgs& a, cudaStream_t st) {
  const long long grid = (long long)a.seqs * a.kv_heads * a.splits;
  if (allow_smem<attention_few_mma_kernel<T, HD>>(few_mma_smem(HD)) != cudaSuccess) return (int)cudaGetLastError();
  attention_few_mma_kernel<T, HD><<<(unsigned)grid, FEW_NT, few_mma_smem(HD), st>>>(a);
  UB_CHECK_LAUNCH();
  return 0;
}

template <typename T>
int few_types(const AttnArgs& a, cudaStream_t st) {
  if constexpr (sizeof(T) == 4)
    return a.hd <= 64 ? few_rows<64>(a, st) : few_rows<128>(a, st);
  else
    return a.hd <= 64 ? few_mma<T, 64>(a, st) : few_mma<T, 128>(a, st);
}

template <typename T>
int forward_types(const AttnArgs& a, const UnblendAttnTrainParams& p, const Plan& n, Path path, bool vec,
                  cudaStream_t st) {
  int rc;
  if (path == FEW)
    rc = few_types<T>(a, st);
  else if (path == SMALL)
    rc = attention_small_forward(a, p, st);
  else if (path == TENSOR_CORES)
    rc = attention_fwd_tc(a, p, n.fwd_rows, st);
  else
    rc = a.hd <= 64 ? simt_forward<T, 64>(a, vec, st) : simt_forward<T, 128>(a, vec, st);
  if (rc || a.splits == 1) return rc;
  if (a.splits <= 4)
    attention_join_kernel<T, 1><<<(unsigned)div_up(n.q_rows, JOIN_WARPS), 32 * JOIN_WARPS, 0, st>>>(a);
  else
    attention_join_kernel<T, JOIN_WARPS><<<(unsigned)n.q_rows, 32 * JOIN_WARPS, 0, st>>>(a);
  UB_CHECK_LAUNCH();
  return 0;
}

template <typename T>
int backward_types(const AttnArgs& a, const UnblendAttnTrainParams& p, const Plan& n, float* parts, bool tc, bool vec,
                   cudaStream_t st) {
  int rc = tc ? attention_stats_tc(a, p, st) : 0;
  if (rc) return rc;
  if (tc)
    rc = attention_dq_tc(a, p, n.dq_splits, parts, st);
  else
    rc = a.hd <= 64 ? simt_dq<T, 64>(a, n.dq_splits, parts, vec, st) : simt_dq<T, 128>(a, n.dq_splits, parts, vec, st);
  if (rc) return rc;
  float* kv_parts = parts + dq_part_floats(p, n);
  if (tc)
    rc = attention_dkv_tc(a, p, n.dkv_splits, kv_parts, st);
  else
    rc = a.hd <= 64 ? simt_dkv<T, 64>(a, n.dkv_splits, kv_parts, vec, st)
                    : simt_dkv<T, 128>(a, n.dkv_splits, kv_parts, vec, st);
  if (rc || (n.dq_splits == 1 && n.dkv_splits == 1)) return rc;
  SumArgs sums{};
  int tensors = 0;
  auto add = [&](const float* part, int splits, int heads, int len, void* out, const UnblendHeadStrides& to) {
    SumArgs::One& x = sums.of[tensors++];
    x = SumArgs::One{part, out, to, splits, heads, len, (long long)a.seqs * heads * len};
    sums.rows += x.rows;
  };
  if (n.dq_splits > 1) add(parts, n.dq_splits, a.heads, a.lq, a.dq, a.dq_s);
  if (n.dkv_splits > 1) {
    add(kv_parts, n.dkv_splits, a.kv_heads, a.lk, a.dk, a.dk_s);
    add(kv_parts + n.dkv_splits * n.k_rows * a.hd, n.dkv_splits, a.kv_heads, a.lk, a.dv, a.dv_s);
  }
  attention_sum_kernel<T><<<(unsigned)div_up(sums.rows, 8), 256, 0, st>>>(a, sums);
  UB_CHECK_LAUNCH();
  return 0;
}

}  // namespace

extern "C" int unblend_attention_workspace(const UnblendAttnTrainParams* p, int backward, long long* bytes) {
  UB_REQUIRE(params_ok(p) && bytes);
  *bytes = 4 * workspace_floats(*p, backward != 0);
  return 0;
}

extern "C" int unblend_attention_forward(const void* q, const void* k, const void* v, void* out, float* lse,
                                         void* work, long long work_bytes, const UnblendAttnTrainParams* p,
                                         void* stream) {
  UB_REQUIRE(q && k && v && out && params_ok(p));
  const long long need = 4 * workspace_floats(*p, false);
  UB_REQUIRE(need == 0 || (aligned16(work) && work && work_bytes >= need));
  const void* ptrs[] = {q, k, v, out};
  const UnblendHeadStrides strides[] = {p->q, p->k, p->v, p->out};
  const int heads[] = {p->heads, p->kv_heads, p->kv_heads, p->heads}, rows[] = {p->lq, p->lk, p->lk, p->lq};
  Path path = attention_tc_fits(*p, ptrs, strides, heads, rows, 4) ? TENSOR_CORES : CUDA_CORES;
  if (path == TENSOR_CORES && attention_is_small(*p, false)) path = SMALL;
  // Few rows: shared heads read K and V once for the group (801 x 4 x 62, 8 over 2 heads of 64: 26 us, SMALL 33 us);
  // without them a short sequence is better off as one tile (801 x 16 x 62, 8 heads: 88 us, SMALL 36 us).
  if (few_fits(*p, k, v) && (path != SMALL || p->heads > p->kv_heads)) path = FEW;
  const Plan n = plan_of(*p, path);
  AttnArgs a = args_of(*p);
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.lse = lse;
  a.splits = n.fwd_splits;
  if (a.splits > 1) {
    a.part = static_cast<float*>(work);
    a.part_lse = a.part + a.splits * n.q_rows * p->hd;
  }
  cudaStream_t st = ub::as_stream(stream);
  const bool vec = p->hd % 4 == 0 && vec4_ok(q, p->q, *p) && vec4_ok(k, p->k, *p) && vec4_ok(v, p->v, *p);
  if (p->dtype == UNBLEND_F32) return forward_types<float>(a, *p, n, path, vec, st);
  if (p->dtype == UNBLEND_BF16) return forward_types<__nv_bfloat16>(a, *p, n, path, vec, st);
  return forward_types<__half>(a, *p, n, path, vec, st);
}

extern "C" int unblend_attention_backward(const void* dout, const void* q, const void* k, const void* v,
                                          const void* out, const float* lse, void* dq, void* dk, void* dv, void* work,
                                          long long work_bytes, const UnblendAttnTrainParams* p, void* stream) {
  UB_REQUIRE(dout && q && k && v && out && lse && dq && dk && dv && params_ok(p));
  UB_REQUIRE(work && aligned16(work) && work_bytes >= 4 * workspace_floats(*p, true));
  const void* ptrs[] = {q, k, v, out, dout, dq, dk, dv};
  const UnblendHeadStrides strides[] = {p->q, p->k, p->v, p->out, p->dout, p->dq, p->dk, p->dv};
  const int hq = p->heads, hk = p->kv_heads;
  const int heads[] = {hq, hk, hk, hq, hq, hq, hk, hk};
  const int rows[] = {p->lq, p->lk, p->lk, p->lq, p->lq, p->lq, p->lk, p->lk};
  const bool tc = attention_tc_fits(*p, ptrs, strides, heads, rows, 8);
  const Plan n = plan_of(*p, tc ? TENSOR_CORES : CUDA_CORES);
  AttnArgs a = args_of(*p);
  a.q = q;
  a.k = k;
  a.v = v;
  a.dout = dout;
  a.out_in = out;
  a.lse = const_cast<float*>(lse);
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  a.dsum = static_cast<float*>(work);
  a.dnorm = a.dsum + round4(2 * n.q_rows);
  a.range = reinterpret_cast<unsigned*>(a.dnorm + norm_floats(*p, n));
  float* parts = a.dsum + stats_floats(*p, n);
  cudaStream_t st = ub::as_stream(stream);
  if (tc && attention_is_small(*p, true)) return attention_small_backward(a, *p, st);
  const bool vec = p->hd % 4 == 0 && vec4_ok(q, p->q, *p) && vec4_ok(k, p->k, *p) && vec4_ok(v, p->v, *p) &&
                   vec4_ok(dout, p->dout, *p);
  if (p->dtype == UNBLEND_F32) return backward_types<float>(a, *p, n, parts, tc, vec, st);
  if (p->dtype == UNBLEND_BF16) return backward_types<__nv_bfloat16>(a, *p, n, parts, tc, vec, st);
  return backward_types<__half>(a, *p, n, parts, tc, vec, st);
}
