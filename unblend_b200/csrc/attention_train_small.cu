// Attention with gradients for sequences of one tile (up to 64 queries and 64 keys), bf16 and fp16: a CTA holds a whole
// sequence and head, so each tensor is read once and written once.
//
//   S = scale Q K^T, P = softmax(S), O = P V
//   dP = dO V^T, D = rowsum(P * dP) (= rowsum(dO * O)), dS = P * (dP - D)
//   dQ = scale dS K, dK = scale dS^T Q, dV = P^T dO
//
// With all keys of a row at hand D comes from P and dP in fp32: the output is not read. One kernel makes the three
// gradients, where the kernels for long rows need one for the statistics, one for dq and one for dk and dv, and read
// the inputs in each.
//
// Bound: HBM. A sequence and head gives 5 products of 64 x 64 x head dim for 7 tensors of 64 rows, far below what the
// tensor cores need per byte, so mma.sync is enough (m16n8k16, fp32 accumulators); tcgen05's 128 rows would be half
// empty, with one round trip through TMEM after the other and nothing to overlap it within a sequence. What hides
// latency here is several independent CTAs per SM.
//
// Four warps, 16 query rows each for S, dP and dQ; P and dS go through shared memory, and each warp takes 16 keys for dK
// and dV. P and dS are rounded to the inputs' type, as the tensor cores take both operands in one 16-bit type; P of fp16
// calls is kept times 2^12 there (small probabilities would be subnormal). Softmax, D and all sums are fp32. Results leave
// through shared memory in 16-byte chunks. 16-byte chunk c of a tile's row lies at c ^ (row & 7).
#include <type_traits>

#include "attention_train.cuh"
#include "warp_mma.cuh"

namespace {

using namespace ub::train;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr int ROWS = 64;  // of a tile
constexpr int NT = 128;

constexpr int fwd_smem(int hd) { return 3 * ROWS * hd * 2; }
constexpr int bwd_smem(int hd, bool grouped) { return ((grouped ? 5 : 4) * ROWS * hd + 2 * ROWS * ROWS) * 2; }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Rows [0, valid) of one head by cp.async; the rest of the tile is 0.
template <typename T, int HD>
__device__ __forceinline__ void fetch(T* tile, const T* src, long long stride, int valid, int hd) {
  constexpr int CH = HD / 8;
#pragma unroll
  for (int x = 0; x < ROWS * CH / NT; ++x) {
    const int id = x * NT + threadIdx.x, row = id / CH, c = id % CH;
    const bool in = row < valid && 8 * c < hd;
    cp_async16_or_zero(tile + row * HD + ((c ^ (row & 7)) * 8), in ? src + row * stride + 8 * c : src, in);
  }
}

// Address of a lane's row in ldmatrix: rows r0 .. r0 + 15 and chunks c, c + 1 of a tile, `down` of the four 8 x 8 blocks
// first.
template <typename T, int COLS>
__device__ __forceinline__ const T* block(const T* tile, int r0, int c, bool down) {
  const int lane = threadIdx.x & 31, m = lane >> 3, r = lane & 7;
  const int row = r0 + (down ? m & 1 : m >> 1) * 8 + r;
  return tile + row * COLS + (((c + (down ? m >> 1 : m & 1)) ^ r) * 8);
}

// d[16 x 64] = A[rows r0 ..][HD] B[64][HD]^T, both tiles as they lie.
template <typename T, int HD>
__device__ __forceinline__ void rows_dot(float (&d)[ROWS / 8][4], const T* ta, int r0, const T* tb) {
#pragma unroll
  for (int n = 0; n < ROWS / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) d[n][e] = 0.f;
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks) {
    uint32_t af[4], f[4];
    ldmatrix4(af, block<T, HD>(ta, r0, 2 * ks, true));
#pragma unroll
    for (int n = 0; n < ROWS / 16; ++n) {
      ldmatrix4(f, block<T, HD>(tb, 16 * n, 2 * ks, false));
      mma16(d[2 * n], af, f[0], f[1], T());
      mma16(d[2 * n + 1], af, f[2], f[3], T());
    }
  }
}

// d[16 x HD] += A[16][16] B[rows r0 .. r0 + 15][HD].
template <typename T, int HD>
__device__ __forceinline__ void rows_sum(float (&d)[HD / 8][4], const uint32_t (&af)[4], const T* tb, int r0) {
#pragma unroll
  for (int n = 0; n < HD / 16; ++n) {
    uint32_t f[4];
    ldmatrix4_trans(f, block<T, HD>(tb, r0, 2 * n, true));
    mma16(d[2 * n], af, f[0], f[1], T());
    mma16(d[2 * n + 1], af, f[2], f[3], T());
  }
}

template <int N>
__device__ __forceinline__ void clear(float (&d)[N][4]) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) d[n][e] = 0.f;
}

// A warp's 16 rows of results: rounded, through `stage` (the warp's own rows of a tile), to global memory.
template <typename T, int N>
__device__ __forceinline__ void pack_rows(uint32_t (&o)[N][2], const float (&d)[N][4], float f0, float f1) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    o[n][0] = pack_pair<T>(d[n][0] * f0, d[n][1] * f0);
    o[n][1] = pack_pair<T>(d[n][2] * f1, d[n][3] * f1);
  }
}
template <typename T, int HD>
__device__ __forceinline__ void put_rows(T* stage, const uint32_t (&o)[HD / 8][2], T* dst, long long stride, int r0,
                                         int rows, int hd) {
  constexpr int CH = HD / 8;
  const int lane = threadIdx.x & 31, quad = lane >> 2, ql = lane & 3;
  __syncwarp();
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int n = 0; n < CH; ++n)
      *reinterpret_cast<uint32_t*>(stage + (r0 + quad + 8 * x) * HD + ((n ^ quad) * 8) + 2 * ql) = o[n][x];
  __syncwarp();
#pragma unroll
  for (int x = 0; x < 16 * CH / 32; ++x) {
    const int id = x * 32 + lane, row = r0 + id / CH, c = id % CH;
    if (row < rows && 8 * c < hd)
      *reinterpret_cast<uint4*>(dst + row * stride + 8 * c) =
          *reinterpret_cast<const uint4*>(stage + row * HD + ((c ^ (row & 7)) * 8));
  }
}

// Keys [0, limit) are seen by query i.
__device__ __forceinline__ int key_limit(const AttnArgs& a, const Bounds& b, int i) {
  return i < b.ql ? (a.causal ? min(b.kl, i + b.off + 1) : b.kl) : 0;
}

template <typename T, int HD>
__global__ void __launch_bounds__(NT, HD == 64 ? 5 : 3) attention_small_fwd_kernel(const __grid_constant__ AttnArgs a) {
  extern __shared__ __align__(128) uint8_t small_smem[];
  T* tq = reinterpret_cast<T*>(small_smem);
  T *tk = tq + ROWS * HD, *tv = tk + ROWS * HD;
  const int lane = threadIdx.x & 31, r0 = (threadIdx.x >> 5) * 16, quad = lane >> 2, ql = lane & 3;
  const int seq = blockIdx.x / a.heads, h = blockIdx.x - seq * a.heads, hk = h / a.group;
  const Bounds b = bounds_of(a, seq);
  fetch<T, HD>(tq, static_cast<const T*>(a.q) + head_offset(a.q_s, a, seq, h), a.q_s.row, b.ql, a.hd);
  fetch<T, HD>(tk, static_cast<const T*>(a.k) + head_offset(a.k_s, a, seq, hk), a.k_s.row, b.kl, a.hd);
  cp_commit();
  fetch<T, HD>(tv, static_cast<const T*>(a.v) + head_offset(a.v_s, a, seq, hk), a.v_s.row, b.kl, a.hd);
  cp_commit();
  cp_wait<1>();
  __syncthreads();
  float s[ROWS / 8][4], inv[2];
  rows_dot<T, HD>(s, tq, r0, tk);
  const float c = a.scale * LOG2E;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int i = r0 + quad + 8 * x, limit = key_limit(a, b, i);
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int n = 0; n < ROWS / 8; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float& z = s[n][2 * x + e];
        z = 8 * n + 2 * ql + e < limit ? z * c : -INFINITY;
        top = fmaxf(top, z);
      }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int n = 0; n < ROWS / 8; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float& z = s[n][2 * x + e];
        z = ex2(z - base);
        sum += z;
      }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    inv[x] = sum == 0.f ? 0.f : 1.f / sum;
    if (a.lse && ql == 0 && i < a.lq)
      a.lse[((long long)seq * a.heads + h) * a.lq + i] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * LN2;
  }
  cp_wait<0>();
  __syncthreads();
  float o[HD / 8][4];
  clear(o);
#pragma unroll
  for (int ks = 0; ks < ROWS / 16; ++ks) {
    const uint32_t pf[4] = {pack_pair<T>(s[2 * ks][0], s[2 * ks][1]), pack_pair<T>(s[2 * ks][2], s[2 * ks][3]),
                            pack_pair<T>(s[2 * ks + 1][0], s[2 * ks + 1][1]),
                            pack_pair<T>(s[2 * ks + 1][2], s[2 * ks + 1][3])};
    rows_sum<T, HD>(o, pf, tv, 16 * ks);
  }
  uint32_t packed[HD / 8][2];
  pack_rows<T>(packed, o, inv[0], inv[1]);
  put_rows<T, HD>(tq, packed, static_cast<T*>(a.out) + head_offset(a.out_s, a, seq, h), a.out_s.row, r0, a.lq, a.hd);
}

// GROUPED: a CTA walks the query heads of its key/value head and keeps dK and dV in registers.
template <typename T, int HD, bool GROUPED>
__global__ void __launch_bounds__(NT, HD == 64 ? (GROUPED ? 3 : 4) : 2)
    attention_small_bwd_kernel(const __grid_constant__ AttnArgs a) {
  constexpr float P_SCALE = std::is_same<T, __half>::value ? 4096.f : 1.f;
  extern __shared__ __align__(128) uint8_t small_smem[];
  T* tk = reinterpret_cast<T*>(small_smem);
  T *tv = tk + ROWS * HD, *tq = tv + ROWS * HD, *td = tq + ROWS * HD;
  T *tp = td + ROWS * HD, *ts = tp + ROWS * ROWS;
  T* stage = GROUPED ? ts + ROWS * ROWS : tv;  // of dQ: V is needed again by the next head
  const int lane = threadIdx.x & 31, r0 = (threadIdx.x >> 5) * 16, quad = lane >> 2, ql = lane & 3;
  const int seq = blockIdx.x / a.kv_heads, hk = blockIdx.x - seq * a.kv_heads;
  const Bounds b = bounds_of(a, seq);
  const float c = a.scale * LOG2E;
  float dk[HD / 8][4], dv[HD / 8][4];
  clear(dk);
  clear(dv);
  for (int g = 0; g < (GROUPED ? a.group : 1); ++g) {
    const int h = hk * a.group + g;
    if (g > 0) __syncthreads();  // the last head's tiles have been read
    fetch<T, HD>(tq, static_cast<const T*>(a.q) + head_offset(a.q_s, a, seq, h), a.q_s.row, b.ql, a.hd);
    if (g == 0)
      fetch<T, HD>(tk, static_cast<const T*>(a.k) + head_offset(a.k_s, a, seq, hk), a.k_s.row, b.kl, a.hd);
    cp_commit();
    fetch<T, HD>(td, static_cast<const T*>(a.dout) + head_offset(a.dout_s, a, seq, h), a.dout_s.row, b.ql, a.hd);
    if (g == 0)
      fetch<T, HD>(tv, static_cast<const T*>(a.v) + head_offset(a.v_s, a, seq, hk), a.v_s.row, b.kl, a.hd);
    cp_commit();
    int limit[2];
    float base[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int i = r0 + quad + 8 * x;
      limit[x] = key_limit(a, b, i);
      const float lse = i < b.ql ? a.lse[((long long)seq * a.heads + h) * a.lq + i] : -INFINITY;
      base[x] = lse == -INFINITY ? INFINITY : lse * LOG2E;  // a row that sees nothing: P = 0
    }
    cp_wait<1>();
    __syncthreads();
    float s[ROWS / 8][4], dp[ROWS / 8][4];
    rows_dot<T, HD>(s, tq, r0, tk);
#pragma unroll
    for (int n = 0; n < ROWS / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        s[n][e] = 8 * n + 2 * ql + (e & 1) < limit[e >> 1] ? ex2(fmaf(s[n][e], c, -base[e >> 1])) : 0.f;
    cp_wait<0>();
    __syncthreads();
    rows_dot<T, HD>(dp, td, r0, tv);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float d = 0.f;
#pragma unroll
      for (int n = 0; n < ROWS / 8; ++n)
#pragma unroll
        for (int e = 2 * x; e < 2 * x + 2; ++e) {
          // Keys that the row does not see may hold anything.
          dp[n][e] = 8 * n + 2 * ql + (e & 1) < limit[x] ? dp[n][e] : 0.f;
          d = fmaf(s[n][e], dp[n][e], d);
        }
      d += __shfl_xor_sync(0xffffffffu, d, 1);
      d += __shfl_xor_sync(0xffffffffu, d, 2);
#pragma unroll
      for (int n = 0; n < ROWS / 8; ++n)
#pragma unroll
        for (int e = 2 * x; e < 2 * x + 2; ++e)
          dp[n][e] = 8 * n + 2 * ql + (e & 1) < limit[x] ? s[n][e] * (dp[n][e] - d) : 0.f;
    }
    uint32_t sf[ROWS / 16][4];  // dS as A fragments
#pragma unroll
    for (int n = 0; n < ROWS / 8; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int at = (r0 + quad + 8 * x) * ROWS + ((n ^ quad) * 8) + 2 * ql;
        *reinterpret_cast<uint32_t*>(tp + at) = pack_pair<T>(s[n][2 * x] * P_SCALE, s[n][2 * x + 1] * P_SCALE);
        const uint32_t w = pack_pair<T>(dp[n][2 * x], dp[n][2 * x + 1]);
        *reinterpret_cast<uint32_t*>(ts + at) = w;
        sf[n / 2][2 * (n & 1) + x] = w;
      }
    uint32_t packed[HD / 8][2];
    {
      float dq[HD / 8][4];
      clear(dq);
#pragma unroll
      for (int ks = 0; ks < ROWS / 16; ++ks) rows_sum<T, HD>(dq, sf[ks], tk, 16 * ks);
      pack_rows<T>(packed, dq, a.scale, a.scale);
    }
    __syncthreads();  // P and dS are written, V (and K, after the last head) read
    put_rows<T, HD>(stage, packed, static_cast<T*>(a.dq) + head_offset(a.dq_s, a, seq, h), a.dq_s.row, r0, a.lq, a.hd);
#pragma unroll
    for (int ks = 0; ks < ROWS / 16; ++ks) {
      uint32_t f[4];
      ldmatrix4_trans(f, block<T, ROWS>(tp, 16 * ks, r0 / 8, false));
      rows_sum<T, HD>(dv, f, td, 16 * ks);
    }
#pragma unroll
    for (int ks = 0; ks < ROWS / 16; ++ks) {
      uint32_t f[4];
      ldmatrix4_trans(f, block<T, ROWS>(ts, 16 * ks, r0 / 8, false));
      rows_sum<T, HD>(dk, f, tq, 16 * ks);
    }
  }
  uint32_t packed[HD / 8][2];
  pack_rows<T>(packed, dv, 1.f / P_SCALE, 1.f / P_SCALE);
  put_rows<T, HD>(tv, packed, static_cast<T*>(a.dv) + head_offset(a.dv_s, a, seq, hk), a.dv_s.row, r0, a.lk, a.hd);
  pack_rows<T>(packed, dk, a.scale, a.scale);
  put_rows<T, HD>(tk, packed, static_cast<T*>(a.dk) + head_offset(a.dk_s, a, seq, hk), a.dk_s.row, r0, a.lk, a.hd);
}

template <typename T, int HD>
int launch_fwd(const AttnArgs& a, cudaStream_t st) {
  constexpr int bytes = fwd_smem(HD);
  if (allow_smem<attention_small_fwd_kernel<T, HD>>(bytes) != cudaSuccess) return (int)cudaGetLastError();
  attention_small_fwd_kernel<T, HD><<<(unsigned)(a.seqs * a.heads), NT, bytes, st>>>(a);
  UB_CHECK_LAUNCH();
  return 0;
}

template <typename T, int HD, bool GROUPED>
int launch_bwd(const AttnArgs& a, cudaStream_t st) {
  constexpr int bytes = bwd_smem(HD, GROUPED);
  if (allow_smem<attention_small_bwd_kernel<T, HD, GROUPED>>(bytes) != cudaSuccess) return (int)cudaGetLastError();
  attention_small_bwd_kernel<T, HD, GROUPED><<<(unsigned)(a.seqs * a.kv_heads), NT, bytes, st>>>(a);
  UB_CHECK_LAUNCH();
  return 0;
}

template <typename T>
int backward_types(const AttnArgs& a, cudaStream_t st) {
  if (a.hd > 64) return launch_bwd<T, 128, false>(a, st);
  return a.group > 1 ? launch_bwd<T, 64, true>(a, st) : launch_bwd<T, 64, false>(a, st);
}

}  // namespace

namespace ub {
namespace train {

bool attention_is_small(const UnblendAttnTrainParams& p, bool backward) {
  return p.lq <= ROWS && p.lk <= ROWS && (!backward || p.hd <= 64 || p.heads == p.kv_heads);
}

int attention_small_forward(const AttnArgs& a, const UnblendAttnTrainParams& p, cudaStream_t st) {
  if (p.dtype == UNBLEND_BF16)
    return a.hd <= 64 ? launch_fwd<__nv_bfloat16, 64>(a, st) : launch_fwd<__nv_bfloat16, 128>(a, st);
  return a.hd <= 64 ? launch_fwd<__half, 64>(a, st) : launch_fwd<__half, 128>(a, st);
}

int attention_small_backward(const AttnArgs& a, const UnblendAttnTrainParams& p, cudaStream_t st) {
  return p.dtype == UNBLEND_BF16 ? backward_types<__nv_bfloat16>(a, st) : backward_types<__half>(a, st);
}

}  // namespace train
}  // namespace ub
