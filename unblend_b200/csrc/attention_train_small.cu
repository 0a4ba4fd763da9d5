// Attention with gradients for sequences of one tile (up to 64 queries and 64 keys), bf16 and fp16: a CTA holds a whole
// sequence and head, so each tensor is read once and written once.
//
//   S = scale Q K^T, P = softmax(S), O = P V
//   dP = dO V^T, D = rowsum(dO * O), dS = P * (dP - D)
//   dQ = scale dS K, dK = scale dS^T Q, dV = P^T dO
//
// One kernel makes the three gradients, where the kernels for long rows need one for the statistics, one for dq and one
// for dk and dv, and read the inputs in each. D = rowsum(P * dP) in fp32 is better than from the rounded O (bf16, 6
// queries over 16 keys: gradients off by 0.0024 instead of 0.0029 relative) and needs no O, but holds only when lse
// and O are of these keys alone, which the caller says with all_keys: whoever joins several blocks of keys gives those
// of all.
//
// Bound: HBM. A sequence and head gives 5 products of 64 x 64 x head dim for 8 tensors of 64 rows, far below what the
// tensor cores need per byte, so mma.sync is enough (m16n8k16, fp32 accumulators); tcgen05's 128 rows would be half
// empty, with one round trip through TMEM after the other and nothing to overlap it within a sequence. What hides
// latency here is several independent CTAs per SM.
//
// A warp has 16 query rows for S, dP and dQ; P and dS go through shared memory, and each warp takes 16 keys for
// dK and dV. P and dS are rounded to the inputs' type, as the tensor cores take both operands in one 16-bit type; fp16
// calls keep P times 2^12 there (small probabilities would be subnormal) and dS times the power of two that brings the
// head's largest one below 2^15 (small gradients would be subnormal, large ones infinite). Softmax, D and all sums are
// fp32.
// Results leave through shared memory in 16-byte chunks. 16-byte chunk c of a tile's row lies at c ^ (row & 7).
#include <type_traits>

#include "attention_train.cuh"
#include "warp_mma.cuh"

namespace {

using namespace ub::train;

constexpr int P_COLS = 64;  // pitch of P and dS

// R: rows of a tile, 64, or 32 for shorter sequences; a warp per 16.
constexpr int fwd_smem(int hd, int r) { return 3 * r * hd * 2; }
constexpr int bwd_smem(int hd, int r, bool grouped) { return ((grouped ? 5 : 4) * r * hd + 2 * r * P_COLS) * 2; }

// CTAs per SM, which is what hides latency. 801 x 62 x 62, 8 heads of 64, bf16: forward 39 us (5.2 TB/s) with 7 CTAs of
// 72 registers, 43 us with 5 of 96 and with 8 of 64 (spills); backward 83 us (4.9 TB/s; fp16 87 us) with 4 of 128 (5
// of 96, with dS in V's place, were 1 us slower). Head dim 128: 70 and 171 us. Earlier versions of 48 and 85 us were
// slower with two warps of 32 rows each, which load half the fragments (51 and 101 us), and with the products of
// 16-key blocks behind the sequence left out (56 and 95 us: the branches kept loads and products from overlapping).
constexpr int fwd_ctas(int hd, int r) { return hd == 64 ? 7 * 64 / r : 4; }
constexpr int bwd_ctas(int hd, int r, bool grouped) { return hd == 64 ? (grouped ? 3 : 4) * 64 / r : 2; }

struct SmallArgs {
  AttnArgs a;
  FastDiv by_heads, by_group, by_inner;  // by_heads: of the CTAs
};

__device__ __forceinline__ uint4 lds16(uint32_t p) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(p)
               : "memory");
  return v;
}

__device__ __forceinline__ void sts4(uint32_t p, uint32_t v) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(p), "r"(v) : "memory");
}

template <int N>
__device__ __forceinline__ void clear(float (&d)[N][4]) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) d[n][e] = 0.f;
}

// First byte of a head. Within a head offsets are 32 bits (attention_is_small).
__device__ __forceinline__ char* head_at(const SmallArgs& s, const void* p, const UnblendHeadStrides& t, int seq,
                                         int h) {
  const int o = s.by_inner(seq), i = seq - o * s.a.inner;
  return const_cast<char*>(static_cast<const char*>(p)) +
         2 * ((long long)o * t.outer + (long long)i * t.inner + (long long)h * t.head);
}

// Rows [first, end) of a head by cp.async; the rest of the tile is 0.
template <int HD, int R>
__device__ __forceinline__ void fetch(uint32_t tile, const char* src, const UnblendHeadStrides& t, int first, int end,
                                      int hd) {
  constexpr int CH = HD / 8, STEP = 2 * R / CH;
  static_assert(STEP % 8 == 0, "a thread's chunk keeps its place");
  const int r = threadIdx.x / CH, c = threadIdx.x % CH;
  const uint32_t stride = 2 * (uint32_t)t.row;
  const int mine = 8 * c < hd ? end : 0, last = max(mine - 1, 0);
  tile += r * (2 * HD) + ((c ^ (r & 7)) * 16);
  src += 8 * c < hd ? 16 * c : 0;
#pragma unroll
  for (int x = 0; x < R / STEP; ++x) {
    const int row = r + x * STEP;
    cp_async16_or_zero(tile + x * STEP * 2 * HD, src + min(row, last) * stride, row >= first && row < mine);
  }
}

// Address of a lane's row in ldmatrix: rows r0 .. r0 + 15 (r0 a multiple of 16) and chunks c, c + 1 (c even) of a tile,
// `DOWN` of the four 8 x 8 blocks first.
template <int COLS, bool DOWN>
__device__ __forceinline__ uint32_t block(uint32_t tile, int r0, int c) {
  const uint32_t lane = threadIdx.x & 31, r = lane & 7, m0 = (lane >> 3) & 1, m1 = lane >> 4;
  const uint32_t at = ((DOWN ? m0 : m1) * 8 + r) * (2 * COLS) + (((DOWN ? m1 : m0) ^ r) * 16);
  return tile + r0 * (2 * COLS) + (at ^ (c * 16));
}

// d[16 x R] = A[rows r0 ..][HD] B[R][HD]^T, both tiles as they lie.
template <typename T, int HD, int R>
__device__ __forceinline__ void rows_dot(float (&d)[R / 8][4], uint32_t ta, int r0, uint32_t tb) {
  clear(d);
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks) {
    uint32_t af[4], f[4];
    ldmatrix4(af, block<HD, true>(ta, r0, 2 * ks));
#pragma unroll
    for (int n = 0; n < R / 16; ++n) {
      ldmatrix4(f, block<HD, false>(tb, 16 * n, 2 * ks));
      mma16(d[2 * n], af, f[0], f[1], T());
      mma16(d[2 * n + 1], af, f[2], f[3], T());
    }
  }
}

// d[16 x HD] += A[16][16] B[rows r0 .. r0 + 15][HD].
template <typename T, int HD>
__device__ __forceinline__ void rows_sum(float (&d)[HD / 8][4], const uint32_t (&af)[4], uint32_t tb, int r0) {
#pragma unroll
  for (int n = 0; n < HD / 16; ++n) {
    uint32_t f[4];
    ldmatrix4_trans(f, block<HD, true>(tb, r0, 2 * n));
    mma16(d[2 * n], af, f[0], f[1], T());
    mma16(d[2 * n + 1], af, f[2], f[3], T());
  }
}

// d[16 x HD] += A^T B with A[R][R] (its columns r0 ..) and B[R][HD].
template <typename T, int HD, int R>
__device__ __forceinline__ void columns_sum(float (&d)[HD / 8][4], uint32_t ta, int r0, uint32_t tb) {
#pragma unroll
  for (int ks = 0; ks < R / 16; ++ks) {
    uint32_t f[4];
    ldmatrix4_trans(f, block<P_COLS, false>(ta, 16 * ks, r0 / 8));
    rows_sum<T, HD>(d, f, tb, 16 * ks);
  }
}

// Dot product of row `row` of two tiles, on all four lanes of a quad; every quad takes other banks first.
template <typename T, int HD>
__device__ __forceinline__ float row_product(uint32_t ta, uint32_t tb, int row) {
  const int lane = threadIdx.x & 31;
  const uint32_t at = row * (2 * HD) + (((lane & 3) + 4 * ((lane >> 2) & 1)) ^ (row & 7)) * 16;
  float2 sum = make_float2(0.f, 0.f);
#pragma unroll
  for (int k = 0; k < HD / 32; ++k) {
    const uint4 x = lds16(ta + (at ^ (k * 64))), y = lds16(tb + (at ^ (k * 64)));
    float2 u[4], v[4];
    unpack16(x, u, T());
    unpack16(y, v, T());
#pragma unroll
    for (int e = 0; e < 4; ++e) sum = ub::fma2(u[e], v[e], sum);
  }
  float d = sum.x + sum.y;
  d += __shfl_xor_sync(0xffffffffu, d, 1);
  d += __shfl_xor_sync(0xffffffffu, d, 2);
  return d;
}

// A warp's 16 rows of results, rounded.
template <typename T, int N>
__device__ __forceinline__ void pack_rows(uint32_t (&o)[N][2], const float (&d)[N][4], float f0, float f1) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    o[n][0] = pack_pair<T>(d[n][0] * f0, d[n][1] * f0);
    o[n][1] = pack_pair<T>(d[n][2] * f1, d[n][3] * f1);
  }
}

// Rows r0 .. r0 + 15 through `stage`, where these rows are the warp's own, to the first `rows` of dst; 0 where no key
// or query counts (the products there may hold NaN).
template <int HD, typename F>
__device__ __forceinline__ void put_rows(uint32_t stage, const uint32_t (&o)[HD / 8][2], char* dst,
                                         const UnblendHeadStrides& t, int r0, int rows, int hd, F&& counts) {
  constexpr int CH = HD / 8, STEP = 32 / CH;
  const int lane = threadIdx.x & 31, quad = lane >> 2, ql = lane & 3;
  stage += r0 * (2 * HD);
  const uint32_t at = quad * (2 * HD) + quad * 16 + ql * 4;
  __syncwarp();
#pragma unroll
  for (int n = 0; n < CH; ++n)
#pragma unroll
    for (int x = 0; x < 2; ++x)
      sts4(stage + (at ^ (n * 16)) + x * 8 * (2 * HD), o[n][x]);
  __syncwarp();
  const int r = lane / CH, c = lane % CH;
  const uint32_t from = r * (2 * HD) + ((c ^ r) * 16), stride = 2 * (uint32_t)t.row;
#pragma unroll
  for (int x = 0; x < 16 / STEP; ++x) {
    const int row = r0 + r + x * STEP;
    if (row < rows && 8 * c < hd) {
      const uint4 v = lds16(stage + (from ^ (((x * STEP) & 7) * 16)) + x * STEP * (2 * HD));
      *reinterpret_cast<uint4*>(dst + row * stride + 16 * c) = counts(row) ? v : make_uint4(0, 0, 0, 0);
    }
  }
}

// Queries [first, end) see some key; the others, whatever they hold, count nowhere.
struct Used {
  int first, end;
};
__device__ __forceinline__ Used used_queries(const AttnArgs& a, const Bounds& b) {
  return Used{a.causal ? max(0, -b.off) : 0, b.kl > 0 ? b.ql : 0};
}
// Keys that each of the rows r0 .. r0 + 15 sees: no mask below.
__device__ __forceinline__ int keys_of_all(const AttnArgs& a, const Bounds& b, int r0) {
  return r0 + 16 <= b.ql ? key_limit(a, b, r0) : 0;
}

template <typename T, int HD, int R>
__global__ void __launch_bounds__(2 * R, fwd_ctas(HD, R))
    attention_small_fwd_kernel(const __grid_constant__ SmallArgs args) {
  const AttnArgs& a = args.a;
  constexpr uint32_t TILE = R * HD * 2;
  extern __shared__ __align__(128) uint8_t small_smem[];
  const uint32_t tq = smem_at(small_smem), tk = tq + TILE, tv = tk + TILE;
  const int lane = threadIdx.x & 31, r0 = (threadIdx.x >> 5) * 16, quad = lane >> 2, ql = lane & 3;
  const int seq = args.by_heads(blockIdx.x), h = blockIdx.x - seq * a.heads, hk = args.by_group(h);
  const Bounds b = bounds_of(a, seq);
  const Used rows = used_queries(a, b);
  fetch<HD, R>(tq, head_at(args, a.q, a.q_s, seq, h), a.q_s, rows.first, rows.end, a.hd);
  fetch<HD, R>(tk, head_at(args, a.k, a.k_s, seq, hk), a.k_s, 0, b.kl, a.hd);
  cp_commit();
  fetch<HD, R>(tv, head_at(args, a.v, a.v_s, seq, hk), a.v_s, 0, b.kl, a.hd);
  cp_commit();
  cp_wait<1>();
  __syncthreads();
  float s[R / 8][4], inv[2];
  rows_dot<T, HD, R>(s, tq, r0, tk);
  const float c = a.scale * LOG2E;
  const int all = keys_of_all(a, b, r0);
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int i = r0 + quad + 8 * x, limit = key_limit(a, b, i);
    float top = -INFINITY;
#pragma unroll
    for (int n = 0; n < R / 8; ++n) {
      float &z0 = s[n][2 * x], &z1 = s[n][2 * x + 1];
      if (8 * n + 8 > all) {
        z0 = 8 * n + 2 * ql < limit ? z0 : -INFINITY;
        z1 = 8 * n + 2 * ql + 1 < limit ? z1 : -INFINITY;
      }
      top = fmaxf(top, fmaxf(z0, z1));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)) * c;
    const float base = top == -INFINITY ? 0.f : -top;
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int n = 0; n < R / 8; ++n) {
      float &z0 = s[n][2 * x], &z1 = s[n][2 * x + 1];
      const float2 z = ub::fma2(make_float2(z0, z1), make_float2(c, c), make_float2(base, base));
      z0 = ex2(z.x);
      z1 = ex2(z.y);
      sum = add2(sum, make_float2(z0, z1));
    }
    float total = sum.x + sum.y;
    total += __shfl_xor_sync(0xffffffffu, total, 1);
    total += __shfl_xor_sync(0xffffffffu, total, 2);
    inv[x] = total == 0.f ? 0.f : __frcp_rn(total);
    if (a.lse && ql == 0 && i < a.lq)
      a.lse[(long long)blockIdx.x * a.lq + i] = total == 0.f ? -INFINITY : (top + __log2f(total)) * LN2;
  }
  cp_wait<0>();
  __syncthreads();
  float o[HD / 8][4];
  clear(o);
#pragma unroll
  for (int ks = 0; ks < R / 16; ++ks) {
    uint32_t pf[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float* p = &s[2 * ks + e / 2][2 * (e & 1)];
      pf[e] = pack_pair<T>(p[0], p[1]);
    }
    rows_sum<T, HD>(o, pf, tv, 16 * ks);
  }
  uint32_t packed[HD / 8][2];
  pack_rows<T>(packed, o, inv[0], inv[1]);
  put_rows<HD>(tq, packed, head_at(args, a.out, a.out_s, seq, h), a.out_s, r0, a.lq, a.hd,
               [&](int i) { return key_limit(a, b, i) > 0; });
}

// GROUPED: a CTA walks the query heads of its key/value head and keeps dK and dV in registers.
template <typename T, int HD, int R, bool GROUPED>
__global__ void __launch_bounds__(2 * R, bwd_ctas(HD, R, GROUPED))
    attention_small_bwd_kernel(const __grid_constant__ SmallArgs args) {
  const AttnArgs& a = args.a;
  constexpr uint32_t TILE = R * HD * 2, P_TILE = R * P_COLS * 2;
  constexpr bool FP16 = std::is_same<T, __half>::value;
  constexpr float P_SCALE = FP16 ? 4096.f : 1.f;
  __shared__ unsigned largest[R / 16];  // fp16: bits of the warps' largest |dS|
  extern __shared__ __align__(128) uint8_t small_smem[];
  const uint32_t tk = smem_at(small_smem), tv = tk + TILE, tq = tv + TILE, td = tq + TILE;
  const uint32_t tp = td + TILE, ts = tp + P_TILE;
  const uint32_t to = tp;  // O, before P (head dims over 64: and dS) takes its place
  static_assert(HD == 64 || HD == 128, "O fits P's tile, or P's and dS's");
  const uint32_t stage = GROUPED ? ts + P_TILE : tv;  // of dQ: V is needed again by the next head
  const int lane = threadIdx.x & 31, r0 = (threadIdx.x >> 5) * 16, quad = lane >> 2, ql = lane & 3;
  const int seq = args.by_heads(blockIdx.x), hk = blockIdx.x - seq * a.kv_heads;
  const Bounds b = bounds_of(a, seq);
  const Used rows = used_queries(a, b);
  const float c = a.scale * LOG2E;
  const int all = keys_of_all(a, b, r0);
  int shift = 0;  // dS and dK are times 2^shift (fp16)
  float dk[HD / 8][4], dv[HD / 8][4];
  clear(dk);
  clear(dv);
  for (int g = 0; g < (GROUPED ? a.group : 1); ++g) {
    const int h = GROUPED ? hk * a.group + g : hk;
    if (g > 0) __syncthreads();  // the last head's tiles have been read
    fetch<HD, R>(tq, head_at(args, a.q, a.q_s, seq, h), a.q_s, rows.first, rows.end, a.hd);
    if (g == 0) fetch<HD, R>(tk, head_at(args, a.k, a.k_s, seq, hk), a.k_s, 0, b.kl, a.hd);
    cp_commit();
    fetch<HD, R>(td, head_at(args, a.dout, a.dout_s, seq, h), a.dout_s, rows.first, rows.end, a.hd);
    if (!a.all_keys) fetch<HD, R>(to, head_at(args, a.out_in, a.out_s, seq, h), a.out_s, rows.first, rows.end, a.hd);
    if (g == 0) fetch<HD, R>(tv, head_at(args, a.v, a.v_s, seq, hk), a.v_s, 0, b.kl, a.hd);
    cp_commit();
    float base[2];
    const float* lse = a.lse + ((long long)seq * a.heads + h) * a.lq;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int i = r0 + quad + 8 * x;
      const float l = i < b.ql ? lse[i] : -INFINITY;
      base[x] = l == -INFINITY ? -INFINITY : -l * LOG2E;  // a row that sees nothing: P = 0
    }
    cp_wait<1>();
    __syncthreads();
    float s[R / 8][4], dp[R / 8][4];
    rows_dot<T, HD, R>(s, tq, r0, tk);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int limit = key_limit(a, b, r0 + quad + 8 * x);
#pragma unroll
      for (int n = 0; n < R / 8; ++n) {
        float &z0 = s[n][2 * x], &z1 = s[n][2 * x + 1];
        const float2 z = ub::fma2(make_float2(z0, z1), make_float2(c, c), make_float2(base[x], base[x]));
        z0 = ex2(z.x);
        z1 = ex2(z.y);
        if (8 * n + 8 > all) {
          z0 = 8 * n + 2 * ql < limit ? z0 : 0.f;
          z1 = 8 * n + 2 * ql + 1 < limit ? z1 : 0.f;
        }
      }
    }
    cp_wait<0>();
    __syncthreads();
    rows_dot<T, HD, R>(dp, td, r0, tv);
    float D[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if (a.all_keys) {
        float2 prod = make_float2(0.f, 0.f);
#pragma unroll
        for (int n = 0; n < R / 8; ++n)
          prod = ub::fma2(make_float2(s[n][2 * x], s[n][2 * x + 1]), make_float2(dp[n][2 * x], dp[n][2 * x + 1]), prod);
        D[x] = prod.x + prod.y;
        D[x] += __shfl_xor_sync(0xffffffffu, D[x], 1);
        D[x] += __shfl_xor_sync(0xffffffffu, D[x], 2);
      } else {
        D[x] = row_product<T, HD>(td, to, r0 + quad + 8 * x);
      }
    }
    unsigned most = 0;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int n = 0; n < R / 8; ++n) {
        float2 e = add2(make_float2(dp[n][2 * x], dp[n][2 * x + 1]), make_float2(-D[x], -D[x]));
        e = mul2(make_float2(s[n][2 * x], s[n][2 * x + 1]), e);
        dp[n][2 * x] = e.x;
        dp[n][2 * x + 1] = e.y;
        if constexpr (FP16) most = max(most, max(__float_as_uint(fabsf(e.x)), __float_as_uint(fabsf(e.y))));
      }
    float up = 1.f;
    if constexpr (FP16) {
      most = __reduce_max_sync(0xffffffffu, most);
      if (lane == 0) largest[threadIdx.x >> 5] = most;
      __syncthreads();  // O's rows, too, lie under other warps' rows of P and dS
#pragma unroll
      for (int w = 0; w < R / 16; ++w) most = max(most, largest[w]);
      const int k = fp16_shift(most);
      up = pow2(k);
      if (GROUPED && g > 0) {  // dK of the heads before, to this head's scale
        const float f = pow2(k - shift);
#pragma unroll
        for (int n = 0; n < HD / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) dk[n][e] *= f;
      }
      shift = k;
    } else if (HD > 64) {
      __syncthreads();  // O's rows lie under other warps' rows of P and dS
    } else {
      __syncwarp();
    }
    uint32_t sf[R / 16][4];  // dS as A fragments
    const uint32_t at = (r0 + quad) * (2 * P_COLS) + quad * 16 + ql * 4;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int n = 0; n < R / 8; ++n) {
        const uint32_t w = pack_pair<T>(dp[n][2 * x] * up, dp[n][2 * x + 1] * up);
        const uint32_t put = (at ^ (n * 16)) + x * 8 * (2 * P_COLS);
        sf[n / 2][2 * (n & 1) + x] = w;
        sts4(tp + put, pack_pair<T>(s[n][2 * x] * P_SCALE, s[n][2 * x + 1] * P_SCALE));
        sts4(ts + put, w);
      }
    }
    uint32_t packed[HD / 8][2];
    {
      float dq[HD / 8][4];
      clear(dq);
#pragma unroll
      for (int ks = 0; ks < R / 16; ++ks) rows_sum<T, HD>(dq, sf[ks], tk, 16 * ks);
      pack_rows<T>(packed, dq, a.scale * pow2(-shift), a.scale * pow2(-shift));
    }
    __syncthreads();  // P and dS are written, K and V are read
    put_rows<HD>(stage, packed, head_at(args, a.dq, a.dq_s, seq, h), a.dq_s, r0, a.lq, a.hd,
                 [&](int i) { return key_limit(a, b, i) > 0; });
    columns_sum<T, HD, R>(dv, tp, r0, td);
    columns_sum<T, HD, R>(dk, ts, r0, tq);
  }
  auto counts = [&](int j) { return j < b.kl; };
  uint32_t packed[HD / 8][2];
  pack_rows<T>(packed, dv, 1.f / P_SCALE, 1.f / P_SCALE);
  put_rows<HD>(tv, packed, head_at(args, a.dv, a.dv_s, seq, hk), a.dv_s, r0, a.lk, a.hd, counts);
  pack_rows<T>(packed, dk, a.scale * pow2(-shift), a.scale * pow2(-shift));
  put_rows<HD>(tk, packed, head_at(args, a.dk, a.dk_s, seq, hk), a.dk_s, r0, a.lk, a.hd, counts);
}

SmallArgs small_args(const AttnArgs& a, int heads) {
  return SmallArgs{a, fast_div(heads), fast_div(a.group), fast_div(a.inner)};
}

template <typename T, int HD, int R>
int launch_fwd(const AttnArgs& a, cudaStream_t st) {
  constexpr int bytes = fwd_smem(HD, R);
  if (allow_smem<attention_small_fwd_kernel<T, HD, R>>(bytes) != cudaSuccess) return (int)cudaGetLastError();
  const unsigned grid = (unsigned)(a.seqs * a.heads);
  attention_small_fwd_kernel<T, HD, R><<<grid, 2 * R, bytes, st>>>(small_args(a, a.heads));
  UB_CHECK_LAUNCH();
  return 0;
}

template <typename T, int HD, int R, bool GROUPED>
int launch_bwd(const AttnArgs& a, cudaStream_t st) {
  constexpr int bytes = bwd_smem(HD, R, GROUPED);
  if (allow_smem<attention_small_bwd_kernel<T, HD, R, GROUPED>>(bytes) != cudaSuccess) return (int)cudaGetLastError();
  const unsigned grid = (unsigned)(a.seqs * a.kv_heads);
  attention_small_bwd_kernel<T, HD, R, GROUPED><<<grid, 2 * R, bytes, st>>>(small_args(a, a.kv_heads));
  UB_CHECK_LAUNCH();
  return 0;
}

// Tiles of 32 rows take a quarter of the products: 801 x 32 x 32, 8 heads of 64, bf16 19 us forward (5.6 TB/s) and 38
// us backward (4.9 TB/s); 801 x 17 x 17 17 and 33 us, with tiles of 64 rows 33 and 74 us.
bool half_tiles(const AttnArgs& a) { return a.lq <= 32 && a.lk <= 32; }

template <typename T>
int forward_types(const AttnArgs& a, cudaStream_t st) {
  if (a.hd > 64) return launch_fwd<T, 128, 64>(a, st);
  return half_tiles(a) ? launch_fwd<T, 64, 32>(a, st) : launch_fwd<T, 64, 64>(a, st);
}

template <typename T>
int backward_types(const AttnArgs& a, cudaStream_t st) {
  if (a.hd > 64) return launch_bwd<T, 128, 64, false>(a, st);
  if (a.group > 1) return half_tiles(a) ? launch_bwd<T, 64, 32, true>(a, st) : launch_bwd<T, 64, 64, true>(a, st);
  return half_tiles(a) ? launch_bwd<T, 64, 32, false>(a, st) : launch_bwd<T, 64, 64, false>(a, st);
}

}  // namespace

namespace ub {
namespace train {

bool attention_is_small(const UnblendAttnTrainParams& p, bool backward) {
  if (p.lq > 64 || p.lk > 64 || (backward && p.hd > 64 && p.heads > p.kv_heads)) return false;
  // 32-bit byte offsets within a head (the row stride of a tensor of one row is not used).
  constexpr long long MOST = 1LL << 24;
  for (const UnblendHeadStrides* t : {&p.q, &p.out, &p.dout, &p.dq})
    if (p.lq > 1 && t->row >= MOST && (backward || t == &p.q || t == &p.out)) return false;
  for (const UnblendHeadStrides* t : {&p.k, &p.v, &p.dk, &p.dv})
    if (p.lk > 1 && t->row >= MOST && (backward || t == &p.k || t == &p.v)) return false;
  return true;
}

int attention_small_forward(const AttnArgs& a, const UnblendAttnTrainParams& p, cudaStream_t st) {
  return p.dtype == UNBLEND_BF16 ? forward_types<__nv_bfloat16>(a, st) : forward_types<__half>(a, st);
}

int attention_small_backward(const AttnArgs& a, const UnblendAttnTrainParams& p, cudaStream_t st) {
  return p.dtype == UNBLEND_BF16 ? backward_types<__nv_bfloat16>(a, st) : backward_types<__half>(a, st);
}

}  // namespace train
}  // namespace ub
