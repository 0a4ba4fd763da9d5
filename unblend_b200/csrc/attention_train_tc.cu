// Attention with gradients on the tcgen05 tensor cores: bf16 and fp16, head dims that are multiples of 8.
//
// All products take the form D[128 rows x N] += A[128 x K] B[N x K]^T with fp32 accumulators in TMEM. Operand tiles
// are rows of 64 elements (128 bytes, 128-byte swizzle) written by TMA, two such column blocks for head dims over 64;
// columns past the head dim and rows past the tensor read as 0. The same tile serves as a K-major operand (summed
// over the head dim: S, dP) and as an MN-major one (summed over its rows: O, dQ, dK, dV): nothing is transposed in
// shared memory. P and dS go from registers to TMEM as 16-bit A operands, over the scores that they came from.
//
//   forward   rows = queries: S = Q K^T (Q resident, K streamed), O += P V
//   dq        rows = queries: S = Q K^T, dP = dO V^T, dQ += dS K
//   dk / dv   rows = keys:    S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q
//
// P and dS are rounded to the inputs' type, as the tensor cores take both operands in one 16-bit type; softmax, its
// statistics and all sums are fp32. 2^x is the hardware approximation (2 ulp). Backward, fp16 keeps P times 2^12 and dS
// times a power of two that its bound |dS| <= |dO_i| |V_j| + |D_i| (norms of the rows) gives: for dQ one per query, for
// dK, which is summed over queries, one per sequence and key/value head. Both cost nothing in the loops: dQ's is added
// to the exponent of P, dK's to the factor that takes P's 2^12 back.
//
// A thread owns a row (or half a row), so row maxima and sums need no shuffles. One warp issues TMA, one the MMAs;
// every barrier wait gives up after two seconds and sets the error flag. A warp gives up as a whole (its lanes vote),
// as the instructions behind a wait need all of them, and a CTA leaves only when what it started is done: the TMA warp
// waits until its last copies have been used, or, after a wait that ran out, until they have landed; a MMA warp that
// gives up waits for the products that it issued.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cudaTypedefs.h>

#include <type_traits>

#include "attention_train.cuh"
#include "tc_common.cuh"

namespace {

using namespace ub::tc;
using namespace ub::train;

constexpr int ROWS = 128;                  // rows of a tile: TMEM lanes
constexpr float RESCALE_THRESHOLD = 8.f;   // log2 units by which the maximum may grow before O is rescaled

// 2^x of a pair on the FMA pipe, for a share of the exponentials (the special function unit takes 16 per cycle and SM,
// the tightest limit at head dim 64). x = n + f with n the nearest integer, read off the low bits of x + 1.5 2^23; 2^f
// by a polynomial of degree 5 on [-1/2, 1/2] fitted for the least relative error (2.1e-7 in fp32, half the hardware
// approximation's two ulp); n goes into the exponent. x below -127 counts as -127, where the exponent field comes out
// as 0 and 2^f as 1 + 2^-23: 2^-149, which the 16-bit types round to 0 (a masked key must not keep even 2^-126, which
// a value near bf16's largest would carry into the sum). Between -127 and -126 the result is off by up to 2^-126. f *
// 0 carries NaN into the result.
__device__ __forceinline__ float2 ex2_fma(float2 x) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.x) : "f"(-127.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.y) : "f"(-127.f));
  constexpr float MAGIC = 12582912.f;
  auto both = [](float v) { return make_float2(v, v); };
  const float2 t = add2(x, both(MAGIC));
  const float2 f = add2(x, ub::fma2(t, both(-1.f), both(MAGIC)));
  float2 p = ub::fma2(both(0.0013276470126584172f), f, both(0.009675540961325169f));
  p = ub::fma2(p, f, both(0.05550713092088699f));
  p = ub::fma2(p, f, both(0.24022120237350464f));
  p = ub::fma2(p, f, both(0.6931469440460205f));
  p = ub::fma2(p, f, both(1.0000001192092896f));
  p.x = __uint_as_float(__float_as_uint(p.x) + (__float_as_uint(t.x) << 23));
  p.y = __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(t.y) << 23));
  return ub::fma2(f, both(0.f), p);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// 32 lanes x 32 columns without waiting for the data (tmem_wait_ld does).
__device__ __forceinline__ void tmem_ld32_async(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16_async(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_ld_async(uint32_t addr, uint32_t (&r)[N]) {
  if constexpr (N == 32)
    tmem_ld32_async(addr, r);
  else
    tmem_ld16_async(addr, r);
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// The same, with the registers as operands: nothing that reads them can move in front of it.
template <int N>
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 16)
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]),
                   "+r"(r[i + 6]), "+r"(r[i + 7]), "+r"(r[i + 8]), "+r"(r[i + 9]), "+r"(r[i + 10]), "+r"(r[i + 11]),
                   "+r"(r[i + 12]), "+r"(r[i + 13]), "+r"(r[i + 14]), "+r"(r[i + 15])::"memory");
}

// One lane of a converged warp. The MMA warps run their loops and waits with all lanes and issue under this predicate:
// operands that the compiler knows to be uniform go straight to the tensor core's uniform registers, where issuing
// from a divergent `lane == 0` branch took 200 cycles per MMA, three times its execution.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// A wait of a whole warp: true for all lanes or for none.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}

// The end of a TMA warp's work (one lane): `n` tiles went through a ring of STAGES, `nr` through the resident tiles.
// All of them have been used, `ok`, or at least nothing is in flight any more.
template <int STAGES>
__device__ __forceinline__ bool drain_tma(bool ok, uint64_t* full, uint64_t* empty, int n, uint64_t* res_full,
                                          uint64_t* res_free, int nr) {
  const int first = n > STAGES ? n - STAGES : 0;
  for (int i = first; ok && i < n; ++i) ok = mbar_wait(&empty[i % STAGES], (i / STAGES) & 1);
  if (ok && nr > 0) ok = mbar_wait(res_free, (nr - 1) & 1);
  if (ok) return true;
  for (int i = first; i < n; ++i) mbar_wait(&full[i % STAGES], (i / STAGES) & 1);
  if (nr > 0) mbar_wait(res_full, (nr - 1) & 1);
  return false;
}

// A MMA warp that gives up (all lanes): the products that it issued are complete.
__device__ __forceinline__ void drain_mma(uint64_t* idle) {
  if (elect_one()) umma_commit(idle);
  __syncwarp();
  warp_wait(idle, 0);
}

// Moves a warpgroup's registers per thread; the warpgroups' shares of a CTA add up to what it was launched with.
template <int N>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Instruction descriptor of kind::f16, M = 128, fp32 accumulate. fmt: 0 fp16, 1 bf16; b_mn: B is MN-major.
__device__ __forceinline__ uint32_t idesc_of(uint32_t fmt, uint32_t n, uint32_t b_mn) {
  return instr_desc(fmt, n) | (b_mn << 16);
}

// Descriptor of an MN-major operand at `addr`: rows (K) of 64 elements (MN), 8-row swizzle atoms back to back; the next
// 64 elements of MN lie `block_bytes` on. 16 rows further: + 2048 bytes.
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t addr, int block_bytes) {
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3FFF);
  d |= (uint64_t)((block_bytes >> 4) & 0x3FFF) << 16;  // leading byte offset: next 64 elements of MN
  d |= (uint64_t)(1024 >> 4) << 32;                    // stride byte offset: next 8 rows
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;  // 128-byte swizzle
  return d;
}

// D = A B^T over the head dim: A [128 x hd] and B [n x hd] as K-major tiles of a_rows / b_rows rows per column block.
template <int HD>
__device__ __forceinline__ void mma_heads(uint32_t d, uint32_t a, uint32_t b, int a_rows, int b_rows, int ksteps,
                                          uint32_t idesc) {
  const uint64_t da = smem_desc(a, 128), db = smem_desc(b, 128);
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks)
    if (ks < ksteps)
      umma_bf16(d, da + (ks >> 2) * a_rows * 8 + (ks & 3) * 2, db + (ks >> 2) * b_rows * 8 + (ks & 3) * 2, idesc,
                ks > 0 ? 1u : 0u);
}

// D (+)= A B over the rows of B's tile: A in TMEM, 16 rows (8 columns) per step; step ks of A is at col(ks).
template <int STEPS, typename Col>
__device__ __forceinline__ void mma_rows(uint32_t d, Col col, uint32_t b, int block_bytes, uint32_t idesc,
                                         uint32_t accum) {
  const uint64_t db = smem_desc_mn(b, block_bytes);
#pragma unroll
  for (int ks = 0; ks < STEPS; ++ks) umma_bf16_ts(d, col(ks), db + ks * 128, idesc, ks > 0 ? 1u : accum);
}

// Rows r with r0 + r outside [lo, hi) of a tile become 0 (thread = row; the tile's products over the head dim are
// complete). 0 * NaN in a masked row would otherwise reach the sums over rows.
__device__ __forceinline__ void clear_row(uint8_t* tile, int rows, int blocks, int r) {
  for (int b = 0; b < blocks; ++b) {
    uint4* p = reinterpret_cast<uint4*>(tile + b * rows * 128 + r * 128);
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = make_uint4(0, 0, 0, 0);
  }
}

struct TcArgs {
  AttnArgs a;
  const float2* stats;   // backward: (-lse log2 e, -D) of each query row, (-inf, 0) for rows that see nothing
  FastDiv by_splits, by_tiles, by_heads, by_inner, by_seq_heads, by_group;
  int row_tiles, units;  // units of the kernel's rows
  int ksteps, n_hd;      // head dim / 16 rounded up, and * 16
  uint32_t fmt;
};

struct TcUnit {
  int seq, so, si;  // sequence, and its outer and inner index
  int h, tile, split;
};

// Unit number -> work. Causal units are ordered by row tile across all heads, the longest first (`last_is_long`: the
// last row tile is the longest); others by head, so that CTAs at work together share the streamed operand in L2.
__device__ __forceinline__ TcUnit tc_unit(const TcArgs& t, int heads, int u, bool last_is_long) {
  TcUnit r;
  int q = t.by_splits(u);
  r.split = u - q * t.a.splits;
  u = q;
  int sh;
  if (t.a.causal) {
    const int rank = t.by_seq_heads(u);
    sh = u - rank * (int)t.by_seq_heads.d;
    r.tile = last_is_long ? t.row_tiles - 1 - rank : rank;
  } else {
    sh = t.by_tiles(u);
    r.tile = u - sh * t.row_tiles;
  }
  r.seq = t.by_heads(sh);
  r.h = sh - r.seq * heads;
  r.so = t.by_inner(r.seq);
  r.si = r.seq - r.so * t.a.inner;
  return r;
}

__device__ __forceinline__ long long unit_offset(const UnblendHeadStrides& s, const TcUnit& u, int h) {
  return (long long)u.so * s.outer + (long long)u.si * s.inner + (long long)h * s.head;
}

// The part `split` of n tiles: [t0, t1).
__device__ __forceinline__ void split_range(const TcArgs& t, int n, int split, int& t0, int& t1) {
  if (t.a.splits == 1) {
    t0 = 0;
    t1 = n;
  } else {
    t0 = t.by_splits(n * split);
    t1 = t.by_splits(n * (split + 1));
  }
}

// The k-th unit of this CTA: alternate rounds walk the CTAs in opposite directions, which evens out causal work.
__device__ __forceinline__ int unit_index(int k) {
  const int g = gridDim.x, c = blockIdx.x;
  return k * g + ((k & 1) ? g - 1 - c : c);
}

__device__ __forceinline__ void tma_head(void* dst, const CUtensorMap* map, uint64_t* bar, int col, int row, int head,
                                         const TcUnit& u) {
  tma_load_5d(dst, map, bar, col, row, head, u.si, u.so);
}

// Up to 32 consecutive values of a row (n left, a multiple of 8), times mul, to T or fp32. Handing 16-byte chunks round
// a quad of lanes, to write 64 bytes of a row at a time, was no faster.
template <typename T>
__device__ __forceinline__ void store_cols(T* out, const uint32_t* v, float mul, int n) {
#pragma unroll
  for (int d = 0; d < 32; d += 8) {
    if (d < n) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = pack2<T>(__uint_as_float(v[d + 2 * e]) * mul, __uint_as_float(v[d + 2 * e + 1]) * mul);
      *reinterpret_cast<uint4*>(out + d) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}
__device__ __forceinline__ void store_cols_f32(float* out, const uint32_t* v, float mul, int n) {
#pragma unroll
  for (int d = 0; d < 32; d += 4)
    if (d < n)
      *reinterpret_cast<float4*>(out + d) =
          make_float4(__uint_as_float(v[d]) * mul, __uint_as_float(v[d + 1]) * mul, __uint_as_float(v[d + 2]) * mul,
                      __uint_as_float(v[d + 3]) * mul);
}

// SHORT kernels (head dims to 64, at most 64 streamed rows): an axis of one tile gives nothing to overlap within a
// unit, so a tile is 64 rows and nothing is double buffered; the forward kernel's CTAs then fit an SM three times.
// Without them and with, 801 sequences, 8 heads: 200 queries and 62 keys 158 and 118 us forward, 498 and 469 us
// backward; 62 queries and 200 keys 505 and 439 us backward. (Two CTAs per SM of the backward kernels, with half the
// registers and spills, were slower than one.)
constexpr int SHORT_ROWS = 64;

// ---------------------------------------------------------------------------------------------- forward
//
// A CTA holds NQ tiles of 128 queries of one head (NQ = 2 shares each K / V tile between 256 queries), each with its
// own softmax warpgroup; while one warpgroup takes exponentials, the tensor cores work for the other. With NQ = 1 that
// is another CTA's. Bound by the chain from one product to the next, through TMEM, the exponentials (49 % of the
// special function rate) and TMEM again; tensor cores 28 % busy, issue slots 43 %: 62 x 801 x 801, 8 heads of 64 173
// us (471 TFLOP/s of visible pairs), causal 8192, 16 over 4 heads of 128 249 us (1104 TFLOP/s). Making the next scores
// ahead, with P beside S in TMEM, gained 1 to 2 % at head dim 64 and is left out.

template <int HD, int NQ, bool SHORT>
struct FwdCfg {
  static constexpr int BN = SHORT ? SHORT_ROWS : 128;  // keys per tile
  static constexpr int NB = HD / 64;                   // 64-column blocks
  static constexpr int Q_BYTES = 128 * 128 * NB;       // a Q tile
  static constexpr int TILE_BYTES = BN * 128 * NB;     // a K or V tile
  static constexpr int STAGES = NQ == 1 && HD == 128 ? 2 : 4;  // ring of K and V tiles
  static constexpr int SMEM = NQ * Q_BYTES + STAGES * TILE_BYTES + 1024 + 512;
  static constexpr int THREADS = NQ * 128 + 128;       // softmax warpgroups, then one for TMA and MMA issue
  static constexpr int PER_SM = SHORT ? 3 : NQ == 2 ? 1 : 2;
  // Registers: 3 x 168 = 2 x 208 + 88 (NQ = 2), 2 x 128 = 200 + 56 (NQ = 1), 2 x 80 = 112 + 48 (SHORT).
  static constexpr int REGS_MORE = SHORT ? 112 : NQ == 2 ? 208 : 200, REGS_LESS = SHORT ? 48 : NQ == 2 ? 88 : 56;
  static constexpr int TMEM = SHORT ? 128 : NQ * 256;
  static constexpr int S_COL = 0, O_COL = BN;  // per query tile, 256 columns apart; P over its scores
  // One pair in eight of the exponentials goes to the FMA pipe: 62 x 801 x 801, 8 heads of 64 174 us; one in four 188
  // us, one in sixteen 182 us.
  static constexpr int FMA_EVERY = 8;
};

template <typename T, int HD, int NQ, bool SHORT>
__global__ void __launch_bounds__(FwdCfg<HD, NQ, SHORT>::THREADS, FwdCfg<HD, NQ, SHORT>::PER_SM)
    attention_fwd_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                            const __grid_constant__ CUtensorMap mv, const __grid_constant__ TcArgs ta) {
  using C = FwdCfg<HD, NQ, SHORT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* ring = smem + NQ * C::Q_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + C::STAGES * C::TILE_BYTES);
  uint64_t* full = bars;                   // [STAGES]
  uint64_t* empty = full + C::STAGES;      // [STAGES]
  uint64_t* q_full = empty + C::STAGES;
  uint64_t* q_free = q_full + 1;
  uint64_t* s_full = q_free + 1;           // [NQ]
  uint64_t* p_ready = s_full + NQ;         // [NQ]
  uint64_t* pv_done = p_ready + NQ;        // [NQ]
  uint64_t* o_free = pv_done + NQ;         // [NQ]
  uint64_t* idle = o_free + NQ;
  uint32_t* slot = reinterpret_cast<uint32_t*>(idle + 1);

  const AttnArgs& a = ta.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    mbar_init(q_full, 1);
    mbar_init(q_free, 1);
    for (int h = 0; h < NQ; ++h) {
      mbar_init(&s_full[h], 1);
      mbar_init(&p_ready[h], 4);
      mbar_init(&pv_done[h], 1);
      mbar_init(&o_free[h], 4);
    }
    mbar_init(idle, 1);
    fence_mbar_init();
  }
  if (warp == NQ * 4 + 1) tmem_alloc(slot, C::TMEM);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *slot;

  // Key tiles of unit u: [t0, t1).
  auto range = [&](const TcUnit& u, const Bounds& b, int& t0, int& t1) {
    const int n = (key_end(a, b, u.tile * NQ * ROWS, NQ * ROWS) + C::BN - 1) / C::BN;
    split_range(ta, n, u.split, t0, t1);
  };

  if (warp >= NQ * 4) {
    regs_down<C::REGS_LESS>();
    if (warp == NQ * 4) {
      if (lane == 0) {
        bool ok = true;
        int it = 0, nq = 0;  // ring tiles and Q loads so far
        auto load = [&](const CUtensorMap* m, int row, int head, const TcUnit& u) {
          const int s = it % C::STAGES, r = it / C::STAGES;
          if (r > 0 && !mbar_wait(&empty[s], (r - 1) & 1)) return false;
          mbar_expect_tx(&full[s], C::TILE_BYTES);
#pragma unroll
          for (int b = 0; b < C::NB; ++b)
            tma_head(ring + s * C::TILE_BYTES + b * C::BN * 128, m, &full[s], 64 * b, row, head, u);
          ++it;
          return true;
        };
        for (int k = 0; ok; ++k) {
          const int ui = unit_index(k);
          if (ui >= ta.units && k * (int)gridDim.x >= ta.units) break;
          if (ui >= ta.units) continue;
          const TcUnit u = tc_unit(ta, a.heads, ui, true);
          const Bounds b = bounds_of(a, u.seq);
          int t0, t1;
          range(u, b, t0, t1);
          if (t0 >= t1) continue;
          if (nq > 0 && !mbar_wait(q_free, (nq - 1) & 1)) {
            ok = false;
            break;
          }
          ++nq;
          mbar_expect_tx(q_full, NQ * C::Q_BYTES);
#pragma unroll
          for (int h = 0; h < NQ; ++h)
#pragma unroll
            for (int c = 0; c < C::NB; ++c)
              tma_head(sQ + h * C::Q_BYTES + c * 128 * 128, &mq, q_full, 64 * c, (u.tile * NQ + h) * ROWS, u.h,
                       u);
          const int hk = u.h / a.group;
          for (int t = t0; t < t1 && ok; ++t) ok = load(&mk, t * C::BN, hk, u) && load(&mv, t * C::BN, hk, u);
        }
        ok = drain_tma<C::STAGES>(ok, full, empty, it, q_full, q_free, nq);
        if (!ok) atomicExch(&g_error_flag, 11);
      }
    } else if (warp == NQ * 4 + 1) {
      {
        const uint32_t id_s = idesc_of(ta.fmt, C::BN, 0), id_o = idesc_of(ta.fmt, ta.n_hd, 1);
        const uint32_t q0 = smem_u32(sQ), r0 = smem_u32(ring);
        bool ok = true;
        int it = 0, nq = 0, g = 0;  // ring tiles, Q loads, key tiles done
        int units = 0;
        auto stage = [&](int i) { return r0 + (i % C::STAGES) * C::TILE_BYTES; };
        for (int k = 0; ok; ++k) {
          const int ui = unit_index(k);
          if (ui >= ta.units && k * (int)gridDim.x >= ta.units) break;
          if (ui >= ta.units) continue;
          const TcUnit u = tc_unit(ta, a.heads, ui, true);
          const Bounds b = bounds_of(a, u.seq);
          int t0, t1;
          range(u, b, t0, t1);
          if (t0 >= t1) continue;
          const int n = t1 - t0;
          // K of tile t is ring tile it + 2 t, V is it + 2 t + 1.
          if (!warp_wait(q_full, nq & 1) || !warp_wait(&full[it % C::STAGES], (it / C::STAGES) & 1)) {
            ok = false;
            break;
          }
          ++nq;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int h = 0; h < NQ; ++h) {
              mma_heads<HD>(tmem + h * 256 + C::S_COL, q0 + h * C::Q_BYTES, stage(it), 128, C::BN, ta.ksteps, id_s);
              umma_commit(&s_full[h]);
            }
            umma_commit(&empty[it % C::STAGES]);
            if (n == 1) umma_commit(q_free);
          }
          __syncwarp();
          for (int t = 0; t < n && ok; ++t) {
            const int vi = it + 2 * t + 1, ki = vi + 1;
            const bool more = t + 1 < n;
            if (!warp_wait(&full[vi % C::STAGES], (vi / C::STAGES) & 1) ||
                (more && !warp_wait(&full[ki % C::STAGES], (ki / C::STAGES) & 1))) {
              ok = false;
              break;
            }
#pragma unroll
            for (int h = 0; h < NQ; ++h) {
              if (ok && t == 0 && units > 0 && !warp_wait(&o_free[h], (units - 1) & 1)) ok = false;
              if (ok && !warp_wait(&p_ready[h], g & 1)) ok = false;
              if (!ok) break;
              tc_fence_after();
              const uint32_t d = tmem + h * 256;
              if (elect_one()) {
                auto p = [&](int ks) { return d + C::S_COL + 8 * ks; };
                mma_rows<C::BN / 16>(d + C::O_COL, p, stage(vi), C::BN * 128, id_o, t > 0 ? 1u : 0u);
                umma_commit(&pv_done[h]);
                if (more) {
                  mma_heads<HD>(d + C::S_COL, q0 + h * C::Q_BYTES, stage(ki), 128, C::BN, ta.ksteps, id_s);
                  umma_commit(&s_full[h]);
                }
                if (h == NQ - 1) {
                  umma_commit(&empty[vi % C::STAGES]);
                  if (more) {
                    umma_commit(&empty[ki % C::STAGES]);
                    if (t + 2 == n) umma_commit(q_free);
                  }
                }
              }
              __syncwarp();
            }
            if (!ok) break;
            ++g;
          }
          it += 2 * n;
          ++units;
        }
        if (!ok) {
          drain_mma(idle);
          if (lane == 0) atomicExch(&g_error_flag, 12);
        }
      }
    }
  } else {
    regs_up<C::REGS_MORE>();
    const int h = warp >> 2, row = threadIdx.x & 127;
    const uint32_t lanes = tmem + h * 256 + ((uint32_t)((warp & 3) * 32) << 16);
    const float c = a.scale * LOG2E;
    const long long rows = (long long)a.seqs * a.heads * a.lq;
    bool ok = true;
    int g = 0, it = 0;
    // The next unit is worked out before the wait for this one's last product, not after its stores.
    TcUnit u_next = tc_unit(ta, a.heads, blockIdx.x, true);
    Bounds b_next = bounds_of(a, u_next.seq);
    for (int k = 0; ok; ++k) {
      const int ui = unit_index(k);
      if (ui >= ta.units && k * (int)gridDim.x >= ta.units) break;
      if (ui >= ta.units) continue;
      const TcUnit u = u_next;
      const Bounds b = b_next;
      int t0, t1;
      range(u, b, t0, t1);
      const int i0 = (u.tile * NQ + h) * ROWS, i = i0 + row;
      const int limit = a.causal ? min(b.kl, i + b.off + 1) : b.kl;  // this row sees keys [0, limit)
      float m = -INFINITY;
      float2 sum2 = make_float2(0.f, 0.f);
      for (int t = t0; t < t1; ++t, ++g) {
        const int j0 = t * C::BN;
        if (!warp_wait(&s_full[h], g & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t s[C::BN];
#pragma unroll
        for (int q = 0; q < C::BN / 32; ++q) tmem_ld32_async(lanes + C::S_COL + 32 * q, s + 32 * q);
        tmem_wait_ld();
        if (j0 + C::BN > b.kl || (a.causal && j0 + C::BN - 1 > i0 + b.off)) {
#pragma unroll
          for (int e = 0; e < C::BN; ++e)
            if (e >= limit - j0) s[e] = __float_as_uint(-INFINITY);
          // V rows behind the length (NaN included) must be 0 before P V. Query tile 0 goes first.
          if (h == 0 && a.k_lens && j0 + C::BN > b.kl) {
            const int vi = it + 2 * (t - t0) + 1;
            if (!warp_wait(&full[vi % C::STAGES], (vi / C::STAGES) & 1)) {
              ok = false;
              break;
            }
            if (row < C::BN && j0 + row >= b.kl)
              clear_row(ring + (vi % C::STAGES) * C::TILE_BYTES, C::BN, C::NB, row);
            fence_proxy_async_smem();
          }
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < C::BN; ++e) mx[e & 3] = fmaxf(mx[e & 3], __uint_as_float(s[e]));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;
        bool rescale = false;
        float corr = 1.f;
        if (top > m + RESCALE_THRESHOLD || (m == -INFINITY && top > -INFINITY)) {
          corr = ex2(m - top);  // 0 on the first tile
          rescale = t > t0;
          m = top;
          sum2.x *= corr, sum2.y *= corr;
        }
        const float base = m == -INFINITY ? 0.f : m;
        const float2 c2 = make_float2(c, c), mb = make_float2(-base, -base);
#pragma unroll
        for (int e = 0; e < C::BN / 2; ++e) {
          const float2 x = ub::fma2(make_float2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), c2, mb);
          const float2 p = e % C::FMA_EVERY == 1 ? ex2_fma(x) : make_float2(ex2(x.x), ex2(x.y));
          sum2 = add2(sum2, p);
          s[e] = pack2<T>(p.x, p.y);
        }
        if (__any_sync(0xffffffffu, rescale)) {
          // O holds the sums up to tile t - 1: they are complete once their product has signalled.
          if (!warp_wait(&pv_done[h], (g - 1) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll 1
          for (int q = 0; q < HD / 32; ++q) {
            uint32_t o[32];
            tmem_ld32(lanes + C::O_COL + 32 * q, o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
            tmem_st32(lanes + C::O_COL + 32 * q, o);
          }
        }
        tmem_st32(lanes + C::S_COL, *reinterpret_cast<uint32_t(*)[32]>(s));
        if constexpr (C::BN > 64) tmem_st32(lanes + C::S_COL + 32, *reinterpret_cast<uint32_t(*)[32]>(s + 32));
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[h]);
      }
      if (!ok) break;
      it += 2 * (t1 - t0);
      if (const int un = unit_index(k + 1); un < ta.units) {
        u_next = tc_unit(ta, a.heads, un, true);
        b_next = bounds_of(a, u_next.seq);
      }
      const float sum = sum2.x + sum2.y;
      const bool live = i < b.ql && (m > -INFINITY || sum != sum);  // all scores NaN: no maximum, but a NaN sum
      const float inv = live ? 1.f / sum : 0.f;
      const long long orow = ((long long)u.seq * a.heads + u.h) * a.lq + i;
      if (t0 < t1) {
        if (!warp_wait(&pv_done[h], (g - 1) & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
      }
      T* out = static_cast<T*>(a.out) + unit_offset(a.out_s, u, u.h) + (long long)i * a.out_s.row;
      float* part = a.splits > 1 ? a.part + (u.split * rows + orow) * a.hd : nullptr;
#pragma unroll 1
      for (int q = 0; q < HD / 32; ++q) {
        uint32_t o[32];
        if (t0 < t1) tmem_ld32(lanes + C::O_COL + 32 * q, o);
        if (!live) {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0;
        }
        const int n = a.hd - 32 * q;
        if (i < a.lq && n > 0) {
          if (part)
            store_cols_f32(part + 32 * q, o, inv, n);
          else
            store_cols<T>(out + 32 * q, o, inv, n);
        }
      }
      if (t0 < t1) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[h]);
      }
      if (i < a.lq) {
        const float lse = live ? (m + log2f(sum)) * LN2 : -INFINITY;
        if (a.splits > 1)
          a.part_lse[u.split * rows + orow] = lse;
        else if (a.lse)
          a.lse[orow] = lse;
      }
    }
    if (!ok) {
      tmem_wait_ld();
      tmem_st_wait();
      atomicExch(&g_error_flag, 13);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == NQ * 4 + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM);
  }
}

// ---------------------------------------------------------------------------------------- row statistics
//
// (-lse log2 e, -D) of each query row, D = rowsum(dO * O) (from O as the caller keeps it, in the inputs' type: half a
// step of its values, next to the like rounding of dS); (-inf, 0) for rows that see nothing. LANES lanes per row, 8
// values each; rows in memory order (heads fastest) for whole lines; all loads of a thread's STATS_ROWS rows are issued
// before the first is used. A kernel of its own: inside the dq kernel the loads stood in front of every unit's first
// tile (5000 of 24000 cycles for 11 tiles). Bound: HBM, one read of dO and O; 62 x 801, 8 heads of 64 22 us (4.6 TB/s;
// one row per thread and hardware divisions 31 us).
constexpr int STATS_ROWS = 4;

template <typename T, int LANES>
__global__ void __launch_bounds__(256)
    attention_stats_kernel(const __grid_constant__ AttnArgs a, float2* stats, FastDiv by_heads, FastDiv by_lq,
                           FastDiv by_inner) {
  constexpr int STEP = 256 / LANES;
  const int lane = threadIdx.x & (LANES - 1);
  const long long n = (long long)a.seqs * a.lq * a.heads;
  const long long first = (long long)blockIdx.x * (STEP * STATS_ROWS) + threadIdx.x / LANES;
  const bool small = n < (1LL << 31);
  long long row[STATS_ROWS];
  float lse[STATS_ROWS];
  uint4 dv[STATS_ROWS], ov[STATS_ROWS];
#pragma unroll
  for (int u = 0; u < STATS_ROWS; ++u) {
    const long long id = min(first + u * STEP, n - 1);  // the last row again: the same values
    int h, seq, i, o;
    if (small) {
      const int token = by_heads((int)id);
      h = (int)id - token * a.heads;
      seq = by_lq(token);
      i = token - seq * a.lq;
      o = by_inner(seq);
    } else {
      const long long token = id / a.heads;
      h = (int)(id - token * a.heads);
      seq = (int)(token / a.lq);
      i = (int)(token - (long long)seq * a.lq);
      o = seq / a.inner;
    }
    const Bounds b = bounds_of(a, seq);
    row[u] = ((long long)seq * a.heads + h) * a.lq + i;
    const bool in = i < b.ql;
    auto at = [&](const void* p, const UnblendHeadStrides& t) {
      return static_cast<const T*>(p) + (long long)o * t.outer + (long long)(seq - o * a.inner) * t.inner +
             (long long)h * t.head + (long long)i * t.row + 8 * lane;
    };
    lse[u] = in ? a.lse[row[u]] : -INFINITY;
    dv[u] = ov[u] = make_uint4(0, 0, 0, 0);
    if (in && 8 * lane < a.hd) {
      dv[u] = *reinterpret_cast<const uint4*>(at(a.dout, a.dout_s));
      ov[u] = *reinterpret_cast<const uint4*>(at(a.out_in, a.out_s));
    }
  }
#pragma unroll
  for (int u = 0; u < STATS_ROWS; ++u) {
    const T* x = reinterpret_cast<const T*>(&dv[u]);
    const T* y = reinterpret_cast<const T*>(&ov[u]);
    float D = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) D = fmaf(to_f(x[e]), to_f(y[e]), D);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) D += __shfl_xor_sync(0xffffffffu, D, o);
    if (lane == 0) stats[row[u]] = lse[u] == -INFINITY ? make_float2(-INFINITY, 0.f) : make_float2(-lse[u] * LOG2E, -D);
  }
}

// The same for fp16, with the norms of dO's rows and, per sequence and key/value head, the largest norm of a row of dO
// and V and the largest |D|: by integer maxima of the bits, whose order does not matter. Queries that see nothing and
// keys behind the length stay out. A warp walks rows of one head, so many that the GPU is full once (its maxima go to
// memory once); units below q_units are rows of dO, the rest rows of V. 62 x 801, 8 heads of 64: 44 us (3.5 TB/s; 96
// warps per SM 40 us, but 2 x 2000, 16 over 4 heads of 128 17 instead of 13 us, for the maxima of few heads).
struct RangeArgs {
  unsigned q_units, units;
  int q_chunks, v_chunks;  // units of a head
  int q_steps, v_steps;    // of a unit, STATS_ROWS * 32 / LANES rows each
  FastDiv by_heads, by_kv_heads, by_q_chunks, by_v_chunks, by_group, by_inner;
};

template <typename T, int LANES>
__global__ void __launch_bounds__(256) attention_stats_range_kernel(const __grid_constant__ AttnArgs a, float2* stats,
                                                                    const __grid_constant__ RangeArgs ra) {
  constexpr int APART = 32 / LANES, STEP = APART * STATS_ROWS;
  const unsigned unit = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (unit >= ra.units) return;
  const bool is_v = unit >= ra.q_units;
  const int id = (int)(is_v ? unit - ra.q_units : unit);
  int h, hk, seq, chunk;  // heads fastest, then the rows
  if (is_v) {
    const int rest = ra.by_kv_heads(id);
    h = hk = id - rest * a.kv_heads;
    seq = ra.by_v_chunks(rest);
    chunk = rest - seq * ra.v_chunks;
  } else {
    const int rest = ra.by_heads(id);
    h = id - rest * a.heads;
    hk = ra.by_group(h);
    seq = ra.by_q_chunks(rest);
    chunk = rest - seq * ra.q_chunks;
  }
  const int o = ra.by_inner(seq), lane = threadIdx.x & (LANES - 1);
  const Bounds b = bounds_of(a, seq);
  const int valid = is_v ? b.kl : b.ql, rows = is_v ? b.kl : a.lq;
  const long long row0 = ((long long)seq * a.heads + h) * a.lq;
  auto head = [&](const void* p, const UnblendHeadStrides& t) {
    return static_cast<const T*>(p) + (long long)o * t.outer + (long long)(seq - o * a.inner) * t.inner +
           (long long)h * t.head + 8 * lane;
  };
  const T* x_at = is_v ? head(a.v, a.v_s) : head(a.dout, a.dout_s);
  const T* o_at = is_v ? nullptr : head(a.out_in, a.out_s);
  const long long x_row = is_v ? a.v_s.row : a.dout_s.row, o_row = a.out_s.row;
  unsigned top_norm = 0, top_D = 0;
  const int span = (is_v ? ra.v_steps : ra.q_steps) * STEP, begin = chunk * span, end = min(rows, begin + span);
  for (int i0 = begin; i0 < end; i0 += STEP) {
    const int first = i0 + (threadIdx.x & 31) / LANES;
    uint4 xv[STATS_ROWS], ov[STATS_ROWS];
    float lse[STATS_ROWS];
#pragma unroll
    for (int u = 0; u < STATS_ROWS; ++u) {
      const int i = first + u * APART;
      xv[u] = ov[u] = make_uint4(0, 0, 0, 0);
      lse[u] = i < valid ? (is_v ? 0.f : a.lse[row0 + i]) : -INFINITY;
      if (i < valid && 8 * lane < a.hd) {
        xv[u] = *reinterpret_cast<const uint4*>(x_at + i * x_row);
        if (!is_v) ov[u] = *reinterpret_cast<const uint4*>(o_at + i * o_row);
      }
    }
#pragma unroll
    for (int u = 0; u < STATS_ROWS; ++u) {
      const int i = first + u * APART;
      const T* x = reinterpret_cast<const T*>(&xv[u]);
      const T* y = reinterpret_cast<const T*>(&ov[u]);
      float D = 0.f, square = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) square = fmaf(to_f(x[e]), to_f(x[e]), square);
#pragma unroll
      for (int s = LANES / 2; s > 0; s >>= 1) square += __shfl_xor_sync(0xffffffffu, square, s);
      if (!is_v) {
#pragma unroll
        for (int e = 0; e < 8; ++e) D = fmaf(to_f(x[e]), to_f(y[e]), D);
#pragma unroll
        for (int s = LANES / 2; s > 0; s >>= 1) D += __shfl_xor_sync(0xffffffffu, D, s);
      }
      const bool counts = lse[u] != -INFINITY;
      const float norm = counts ? sqrtf(square) : 0.f;
      if (!counts) D = 0.f;
      top_norm = max(top_norm, __float_as_uint(norm));
      top_D = max(top_D, __float_as_uint(fabsf(D)));
      if (!is_v && lane == 0 && i < end) {
        stats[row0 + i] = counts ? make_float2(-lse[u] * LOG2E, -D) : make_float2(-INFINITY, 0.f);
        a.dnorm[row0 + i] = norm;
      }
    }
  }
  top_norm = __reduce_max_sync(0xffffffffu, top_norm);
  top_D = __reduce_max_sync(0xffffffffu, top_D);
  if ((threadIdx.x & 31) == 0) {
    unsigned* to = a.range + 4 * ((long long)seq * a.kv_heads + hk);
    atomicMax(to + (is_v ? 0 : 1), top_norm);
    if (!is_v) atomicMax(to + 2, top_D);
  }
}

// --------------------------------------------------------------------------------------------------- dq
//
// 128 queries of one head per unit, keys streamed 128 at a time; two threads per row, 64 keys each. S is double
// buffered and dP is read into registers first, so the tensor cores make S and dP of the next tile while this one's
// exponentials are taken. dS of 32 keys takes 16 of the 32 columns that their scores came from. Bound as the forward
// pass, with one more product to read and one CTA per SM: 62 x 801 x 801, 8 heads of 64 222 us (550 TFLOP/s of visible
// pairs), causal 8192, 16 over 4 heads of 128 410 us (1005 TFLOP/s).

template <int HD, bool SHORT>
struct DqCfg {
  static constexpr int BN = SHORT ? SHORT_ROWS : 128;
  static constexpr int NB = HD / 64;
  static constexpr int Q_BYTES = 128 * 128 * NB;
  static constexpr int TILE_BYTES = BN * 128 * NB;
  static constexpr int STAGES = HD == 64 && !SHORT ? 8 : 4;
  static constexpr int SMEM = 2 * Q_BYTES + STAGES * TILE_BYTES + 1024 + 512;
  static constexpr int THREADS = 384;  // two warpgroups of rows, one for TMA and MMA issue
  static constexpr int REGS_MORE = 208, REGS_LESS = 88;  // 2 x 208 + 88 = 3 x 168
  static constexpr int HALF = BN / 2, CH = HALF / 2;  // keys of a tile per thread, and taken at once
  static constexpr int SB = SHORT ? 1 : 2;  // S buffers
  static constexpr int S_COL = 0, DP_COL = SB * BN, DQ_COL = (SB + 1) * BN, TMEM = SHORT ? 256 : 512;
  // Head dims over 64 are bound by the products: dP is read at once, so that the next one starts at once.
  static constexpr bool EARLY = HD > 64 || SHORT;
};

template <typename T, int HD, bool SHORT>
__global__ void __launch_bounds__(DqCfg<HD, SHORT>::THREADS, 1)
    attention_dq_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mdo,
                           const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                           const __grid_constant__ TcArgs ta) {
  using C = DqCfg<HD, SHORT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                      // Q, then dO
  uint8_t* sO = smem + C::Q_BYTES;
  uint8_t* ring = smem + 2 * C::Q_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + C::STAGES * C::TILE_BYTES);
  uint64_t* full = bars;
  uint64_t* empty = full + C::STAGES;
  uint64_t* q_full = empty + C::STAGES;
  uint64_t* q_free = q_full + 1;
  uint64_t* dp_full = q_free + 1;  // S of the tile too: its product is issued before
  uint64_t* dp_free = dp_full + 1;
  // [2], by tile: a warp can be done with tile g + 1 while another still works on g, but not with g + 2, whose dP is
  // issued after all of g has been waited for.
  uint64_t* ds_ready = dp_free + 1;
  uint64_t* dq_done = ds_ready + 2;
  uint64_t* dq_free = dq_done + 1;
  uint64_t* idle = dq_free + 1;
  uint32_t* slot = reinterpret_cast<uint32_t*>(idle + 1);

  const AttnArgs& a = ta.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    mbar_init(q_full, 1);
    mbar_init(q_free, 1);
    mbar_init(dp_full, 1);
    mbar_init(dp_free, 8);
    mbar_init(&ds_ready[0], 8);
    mbar_init(&ds_ready[1], 8);
    mbar_init(dq_done, 1);
    mbar_init(dq_free, 8);
    mbar_init(idle, 1);
    fence_mbar_init();
  }
  if (warp == 9) tmem_alloc(slot, C::TMEM);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *slot;

  auto range = [&](const TcUnit& u, const Bounds& b, int& t0, int& t1) {
    const int n = (key_end(a, b, u.tile * ROWS, ROWS) + C::BN - 1) / C::BN;
    split_range(ta, n, u.split, t0, t1);
  };

  if (warp >= 8) {
    regs_down<C::REGS_LESS>();
    if (warp == 8) {
      if (lane == 0) {
        bool ok = true;
        int it = 0, nq = 0;
        auto load = [&](const CUtensorMap* m, int row, int head, const TcUnit& u) {
          const int s = it % C::STAGES, r = it / C::STAGES;
          if (r > 0 && !mbar_wait(&empty[s], (r - 1) & 1)) return false;
          mbar_expect_tx(&full[s], C::TILE_BYTES);
#pragma unroll
          for (int b = 0; b < C::NB; ++b)
            tma_head(ring + s * C::TILE_BYTES + b * C::BN * 128, m, &full[s], 64 * b, row, head, u);
          ++it;
          return true;
        };
        for (int k = 0; ok; ++k) {
          const int ui = unit_index(k);
          if (ui >= ta.units && k * (int)gridDim.x >= ta.units) break;
          if (ui >= ta.units) continue;
          const TcUnit u = tc_unit(ta, a.heads, ui, true);
          const Bounds b = bounds_of(a, u.seq);
          int t0, t1;
          range(u, b, t0, t1);
          if (t0 >= t1) continue;
          if (nq > 0 && !mbar_wait(q_free, (nq - 1) & 1)) {
            ok = false;
            break;
          }
          ++nq;
          mbar_expect_tx(q_full, 2 * C::Q_BYTES);
#pragma unroll
          for (int c = 0; c < C::NB; ++c) {
            tma_head(sQ + c * 128 * 128, &mq, q_full, 64 * c, u.tile * ROWS, u.h, u);
            tma_head(sO + c * 128 * 128, &mdo, q_full, 64 * c, u.tile * ROWS, u.h, u);
          }
          const int hk = u.h / a.group;
          for (int t = t0; t < t1 && ok; ++t) ok = load(&mk, t * C::BN, hk, u) && load(&mv, t * C::BN, hk, u);
        }
        ok = drain_tma<C::STAGES>(ok, full, empty, it, q_full, q_free, nq);
        if (!ok) atomicExch(&g_error_flag, 21);
      }
    } else if (warp == 9) {
      {
        const uint32_t id_s = idesc_of(ta.fmt, C::BN, 0), id_o = idesc_of(ta.fmt, ta.n_hd, 1);
        const uint32_t q0 = smem_u32(sQ), o0 = smem_u32(sO), r0 = smem_u32(ring);
        bool ok = true;
        int it = 0, nq = 0, g = 0, units = 0;
        auto stage = [&](int i) { return r0 + (i % C::STAGES) * C::TILE_BYTES; };
        auto wait_full = [&](int i) { return warp_wait(&full[i % C::STAGES], (i / C::STAGES) & 1); };
        for (int k = 0; ok; ++k) {
          const int ui = unit_index(k);
          if (ui >= ta.units && k * (int)gridDim.x >= ta.units) break;
          if (ui >= ta.units) continue;
          const TcUnit u = tc_unit(ta, a.heads, ui, true);
          const Bounds b = bounds_of(a, u.seq);
          int t0, t1;
          range(u, b, t0, t1);
          if (t0 >= t1) continue;
          const int n = t1 - t0;
          // Tile g (counted over all units): its K is ring tile it + 2 t, its V it + 2 t + 1; S in buffer g & 1.
          auto issue_s = [&](int t) {
            if (!wait_full(it + 2 * t)) return false;
            tc_fence_after();
            if (elect_one())
              mma_heads<HD>(tmem + C::S_COL + ((g + t) % C::SB) * C::BN, q0, stage(it + 2 * t), 128, C::BN, ta.ksteps,
                            id_s);
            __syncwarp();
            return true;
          };
          auto issue_dp = [&](int t) {
            if (!wait_full(it + 2 * t + 1)) return false;
            // dP of the tile before has been read (every tile signals once).
            if (g + t > 0 && !warp_wait(dp_free, (g + t - 1) & 1)) return false;
            tc_fence_after();
            if (elect_one()) {
              mma_heads<HD>(tmem + C::DP_COL, o0, stage(it + 2 * t + 1), 128, C::BN, ta.ksteps, id_s);
              umma_commit(dp_full);
              umma_commit(&empty[(it + 2 * t + 1) % C::STAGES]);
              if (t + 1 == n) umma_commit(q_free);
            }
            __syncwarp();
            return true;
          };
          if (!warp_wait(q_full, nq & 1) || !issue_s(0) || !issue_dp(0)) {
            ok = false;
            break;
          }
          ++nq;
          for (int t = 0; t < n; ++t) {
            // S of the next tile overwrites dS of tile t - 1 (of tile t with one buffer), whose product is issued
            // first.
            if (C::SB == 2 && t + 1 < n && (!issue_s(t + 1) || !issue_dp(t + 1))) {
              ok = false;
              break;
            }
            if (t == 0 && units > 0 && !warp_wait(dq_free, (units - 1) & 1)) {
              ok = false;
              break;
            }
            if (!warp_wait(&ds_ready[(g + t) & 1], ((g + t) >> 1) & 1)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t ds = tmem + C::S_COL + ((g + t) % C::SB) * C::BN;
            if (elect_one()) {
              auto a_col = [&](int ks) { return ds + ks / (C::CH / 16) * C::CH + ks % (C::CH / 16) * 8; };
              mma_rows<C::BN / 16>(tmem + C::DQ_COL, a_col, stage(it + 2 * t), C::BN * 128, id_o, t > 0 ? 1u : 0u);
              umma_commit(&empty[(it + 2 * t) % C::STAGES]);
              if (t + 1 == n) umma_commit(dq_done);
            }
            __syncwarp();
            if (C::SB == 1 && t + 1 < n && (!issue_s(t + 1) || !issue_dp(t + 1))) {
              ok = false;
              break;
            }
          }
          if (!ok) break;
          g += n;
          it += 2 * n;
          ++units;
        }
        if (!ok) {
          drain_mma(idle);
          if (lane == 0) atomicExch(&g_error_flag, 22);
        }
      }
    }
  } else {
    regs_up<C::REGS_MORE>();
    const int half = warp >> 2, row = threadIdx.x & 127;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const float c = a.scale * LOG2E;
    const long long rows = (long long)a.seqs * a.heads * a.lq;
    bool ok = true;
    int g = 0, it = 0, units = 0;
    // Statistics of this thread's row in the k-th unit; fp16: the norm of its dO too.
    struct Row {
      float2 st;
      float dnorm;
    };
    auto load_stats = [&](int k) {
      Row r{make_float2(-INFINITY, 0.f), 0.f};
      const int ui = unit_index(k);
      if (ui >= ta.units) return r;
      const TcUnit u = tc_unit(ta, a.heads, ui, true);
      const int i = u.tile * ROWS + row;
      if (i >= a.lq) return r;
      const long long at = ((long long)u.seq * a.heads + u.h) * a.lq + i;
      r.st = ta.stats[at];
      if constexpr (std::is_same<T, __half>::value) r.dnorm = a.dnorm[at];
      return r;
    };
    Row next = load_stats(0);
    for (int k = 0; ok; ++k) {
      const int ui = unit_index(k);
      if (ui >= ta.units && k * (int)gridDim.x >= ta.units) break;
      const Row own = next;
      next = load_stats(k + 1);
      if (ui >= ta.units) continue;
      float2 st = own.st;
      float unscale = a.scale;
      const TcUnit u = tc_unit(ta, a.heads, ui, true);
      const Bounds b = bounds_of(a, u.seq);
      int t0, t1;
      range(u, b, t0, t1);
      const int i0 = u.tile * ROWS, i = i0 + row;
      const int limit = a.causal ? min(b.kl, i + b.off + 1) : b.kl;
      const long long orow = ((long long)u.seq * a.heads + u.h) * a.lq + i;
      const bool live = st.x != -INFINITY;  // dead rows: P = 0
      if constexpr (std::is_same<T, __half>::value) {
        const float vnorm = __uint_as_float(a.range[4 * ((long long)u.seq * a.kv_heads + ta.by_group(u.h))]);
        const int shift = fp16_shift(__float_as_uint(fmaf(own.dnorm, vnorm, fabsf(st.y))));
        st.x += (float)shift;
        unscale *= pow2(-shift);
      }
      const float2 c2 = make_float2(c, c), l2 = make_float2(st.x, st.x), d2 = make_float2(st.y, st.y);
      // A thread's 64 keys go in two chunks; the loads of the next one are in flight during this one's exponentials.
      uint32_t s0[C::CH], d0[C::CH], s1[C::CH], d1[C::CH];
      auto load = [&](int tile, int chunk, uint32_t (&s)[C::CH], uint32_t (&d)[C::CH]) {
        tmem_ld_async(lanes + C::DP_COL + half * C::HALF + C::CH * chunk, d);
        tmem_ld_async(lanes + C::S_COL + (tile % C::SB) * C::BN + half * C::HALF + C::CH * chunk, s);
      };
      // dS of one chunk from its scores and dP, stored over the scores.
      auto chunk_ds = [&](int t, int chunk, bool edge, uint32_t (&s)[C::CH], uint32_t (&d)[C::CH]) {
        if (edge) {
          // Masked keys: P = exp(-inf) = 0, so dS = 0; behind a length, where V may hold NaN, dP is set aside too.
          const int left = limit - (t * C::BN + half * C::HALF + C::CH * chunk);
#pragma unroll
          for (int e = 0; e < C::CH; ++e)
            if (e >= left) s[e] = __float_as_uint(-INFINITY);
          if (a.k_lens) {
#pragma unroll
            for (int e = 0; e < C::CH; ++e)
              if (e >= left) d[e] = 0;
          }
        }
        uint32_t w[C::CH / 2];
#pragma unroll
        for (int e = 0; e < C::CH / 2; ++e) {
          const float2 x = ub::fma2(make_float2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), c2, l2);
          const float2 p = make_float2(ex2(x.x), ex2(x.y));
          const float2 ds = mul2(p, add2(make_float2(__uint_as_float(d[2 * e]), __uint_as_float(d[2 * e + 1])), d2));
          w[e] = pack2<T>(ds.x, ds.y);
        }
        const uint32_t to = lanes + C::S_COL + (g % C::SB) * C::BN + half * C::HALF + C::CH * chunk;
        if constexpr (C::CH == 32)
          tmem_st16(to, w);
        else
          tmem_st8(to, w);
      };
      if (!C::EARLY && t0 < t1) {
        if (!warp_wait(dp_full, g & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        load(g, 0, s0, d0);
      }
      for (int t = t0; t < t1; ++t, ++g) {
        const bool edge = t * C::BN + C::BN > b.kl || (a.causal && t * C::BN + C::BN - 1 > i0 + b.off);
        if (C::EARLY) {
          if (!warp_wait(dp_full, g & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          load(g, 0, s0, d0);
        }
        if (!C::EARLY) {
          tmem_wait_ld(s0);
          tmem_wait_ld(d0);
        }
        load(g, 1, s1, d1);
        if (C::EARLY) {
          tmem_wait_ld(s0);
          tmem_wait_ld(d0);
        } else {
          chunk_ds(t, 0, edge, s0, d0);
        }
        tmem_wait_ld(s1);
        tmem_wait_ld(d1);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(dp_free);
        if (C::EARLY) chunk_ds(t, 0, edge, s0, d0);
        // Keys behind the length (NaN included) must be 0 before dS K; S, which also reads them, is complete.
        if (edge && a.k_lens && t * C::BN + C::BN > b.kl && half == 0) {
          if (row < C::BN && t * C::BN + row >= b.kl)
            clear_row(ring + ((it + 2 * (t - t0)) % C::STAGES) * C::TILE_BYTES, C::BN, C::NB, row);
          fence_proxy_async_smem();
        }
        chunk_ds(t, 1, edge, s1, d1);
        if (!C::EARLY && t + 1 < t1) {
          if (!warp_wait(dp_full, (g + 1) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          load(g + 1, 0, s0, d0);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ds_ready[g & 1]);
      }
      if (!ok) break;
      it += 2 * (t1 - t0);
      if (t0 < t1) {
        if (!warp_wait(dq_done, units & 1)) {
          ok = false;
          break;
        }
        ++units;
        tc_fence_after();
      }
      T* dq = static_cast<T*>(a.dq) + unit_offset(a.dq_s, u, u.h) + (long long)i * a.dq_s.row;
      float* part = a.splits > 1 ? a.part + (u.split * rows + orow) * a.hd : nullptr;
#pragma unroll 1
      for (int q = half * (HD / 64); q < (half + 1) * (HD / 64); ++q) {
        uint32_t v[32];
        if (t0 < t1) tmem_ld32(lanes + C::DQ_COL + 32 * q, v);
        if (!live || t0 >= t1) {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0;
        }
        const int n = a.hd - 32 * q;
        if (i < a.lq && n > 0) {
          if (part)
            store_cols_f32(part + 32 * q, v, unscale, n);
          else
            store_cols<T>(dq + 32 * q, v, unscale, n);
        }
      }
      if (t0 < t1) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(dq_free);
      }
    }
    if (!ok) {
      tmem_wait_ld();
      tmem_st_wait();
      atomicExch(&g_error_flag, 23);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM);
  }
}

// ---------------------------------------------------------------------------------------------- dk, dv
//
// 128 keys of one key/value head per unit; the queries of all heads of its group are streamed (128 at a time, 64 for
// head dims over 64, where the two accumulators take half of TMEM). Two threads per key, half of the tile's queries
// each. lse and D go by column here: a warp brings them to shared memory, and rows that must not count come with
// -lse = -inf, P = 0. P^T and dS^T of a thread share the columns of its scores. 62 x 801 x 801, 8 heads of 64:
// 273 us (597 TFLOP/s of visible pairs), causal 8192, 16 over 4 heads of 128 551 us (998 TFLOP/s).

template <int HD, bool SHORT>
struct DkvCfg {
  static constexpr int BN = HD == 64 && !SHORT ? 128 : 64;
  static constexpr int NB = HD / 64;
  static constexpr int KV_BYTES = 128 * 128 * NB;
  static constexpr int TILE_BYTES = BN * 128 * NB;  // Q or dO: 16 KB
  static constexpr int STAGES = SHORT ? 2 : 4;                  // (Q, dO) pairs
  static constexpr int STATS = 4;                   // (lse, D) rows
  static constexpr int SMEM = 2 * KV_BYTES + 2 * STAGES * TILE_BYTES + STATS * BN * 8 + 1024 + 512;
  static constexpr int THREADS = 384;  // two warpgroups of keys, one for TMA, MMA issue and lse / D
  static constexpr int REGS_MORE = 208, REGS_LESS = 88;  // 2 x 208 + 88 = 3 x 168
  static constexpr int HALF = BN / 2;  // queries of a tile per thread
  static constexpr int CH = HALF / 2;  // taken at once
  static constexpr int SB = SHORT ? 1 : 2;  // S buffers
  static constexpr int S_COL = 0, DP_COL = SB * BN, DV_COL = (SB + 1) * BN, DK_COL = DV_COL + HD;
  static constexpr int TMEM = SHORT ? 256 : 512;
  static_assert(DK_COL + HD <= TMEM, "TMEM columns");
  static constexpr bool EARLY = HD > 64 || SHORT;  // as in the dq kernel
};

// P of fp16 calls is kept times 2^12: probabilities of long rows would sink into fp16's subnormals.
template <typename T>
__device__ __forceinline__ constexpr float p_shift() {
  return 0.f;
}
template <>
__device__ __forceinline__ constexpr float p_shift<__half>() {
  return 12.f;
}

template <typename T, int HD, bool SHORT>
__global__ void __launch_bounds__(DkvCfg<HD, SHORT>::THREADS, 1)
    attention_dkv_tc_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                            const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mdo,
                            const __grid_constant__ TcArgs ta) {
  using C = DkvCfg<HD, SHORT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = smem;
  uint8_t* sV = smem + C::KV_BYTES;
  uint8_t* ring = smem + 2 * C::KV_BYTES;  // [STAGES][Q, dO]
  float* stats = reinterpret_cast<float*>(ring + 2 * C::STAGES * C::TILE_BYTES);  // [STATS][-lse2 BN, -D BN]
  uint64_t* bars = reinterpret_cast<uint64_t*>(stats + C::STATS * 2 * C::BN);
  uint64_t* full = bars;                  // [STAGES] Q and dO
  uint64_t* empty = full + C::STAGES;
  uint64_t* kv_full = empty + C::STAGES;
  uint64_t* kv_free = kv_full + 1;
  uint64_t* dp_full = kv_free + 1;        // S of the tile too: its product is issued before
  uint64_t* dp_free = dp_full + 1;
  uint64_t* ps_ready = dp_free + 1;       // [2], by tile, as ds_ready of the dq kernel
  uint64_t* st_full = ps_ready + 2;       // [STATS]
  uint64_t* st_free = st_full + C::STATS; // [STATS]
  uint64_t* acc_done = st_free + C::STATS;
  uint64_t* acc_free = acc_done + 1;
  uint64_t* idle = acc_free + 1;
  uint32_t* slot = reinterpret_cast<uint32_t*>(idle + 1);

  const AttnArgs& a = ta.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    for (int i = 0; i < C::STATS; ++i) mbar_init(&st_full[i], 32), mbar_init(&st_free[i], 8);
    mbar_init(kv_full, 1);
    mbar_init(kv_free, 1);
    mbar_init(dp_full, 1);
    mbar_init(dp_free, 8);
    mbar_init(&ps_ready[0], 8);
    mbar_init(&ps_ready[1], 8);
    mbar_init(acc_done, 1);
    mbar_init(acc_free, 8);
    mbar_init(idle, 1);
    fence_mbar_init();
  }
  if (warp == 9) tmem_alloc(slot, C::TMEM);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *slot;

  // Tiles of a unit: for each head of the group, query tiles [begin, begin + per); t in [t0, t1) of all of them.
  struct Walk {
    int head, tile, per;  // within the group, within the head
    __device__ __forceinline__ Walk(int t0, int per_) : head(t0 ? t0 / per_ : 0), tile(t0 - head * per_), per(per_) {}
    __device__ __forceinline__ void next() {
      if (++tile == per) tile = 0, ++head;
    }
  };
  auto range = [&](const TcUnit& u, const Bounds& b, int& begin, int& per, int& t0, int& t1) {
    const int j0 = u.tile * ROWS;
    begin = query_begin(a, b, j0) / C::BN;
    per = j0 < b.kl ? max(0, (b.ql + C::BN - 1) / C::BN - begin) : 0;
    split_range(ta, per * a.group, u.split, t0, t1);
  };

  if (warp >= 8) {
    regs_down<C::REGS_LESS>();
    if (warp == 8) {
      if (lane == 0) {
        bool ok = true;
        int it = 0, nkv = 0;
        for (int k = 0; ok; ++k) {
          const int ui = unit_index(k);
          if (ui >= ta.units && k * (int)gridDim.x >= ta.units) break;
          if (ui >= ta.units) continue;
          const TcUnit u = tc_unit(ta, a.kv_heads, ui, false);
          const Bounds b = bounds_of(a, u.seq);
          int begin, per, t0, t1;
          range(u, b, begin, per, t0, t1);
          if (t0 >= t1) continue;
          if (nkv > 0 && !mbar_wait(kv_free, (nkv - 1) & 1)) {
            ok = false;
            break;
          }
          ++nkv;
          mbar_expect_tx(kv_full, 2 * C::KV_BYTES);
#pragma unroll
          for (int c = 0; c < C::NB; ++c) {
            tma_head(sK + c * 128 * 128, &mk, kv_full, 64 * c, u.tile * ROWS, u.h, u);
            tma_head(sV + c * 128 * 128, &mv, kv_full, 64 * c, u.tile * ROWS, u.h, u);
          }
          Walk w(t0, per);
          for (int t = t0; t < t1; ++t, ++it, w.next()) {
            const int h = u.h * a.group + w.head, i0 = (begin + w.tile) * C::BN;
            const int s = it % C::STAGES, r = it / C::STAGES;
            if (r > 0 && !mbar_wait(&empty[s], (r - 1) & 1)) {
              ok = false;
              break;
            }
            mbar_expect_tx(&full[s], 2 * C::TILE_BYTES);
            uint8_t* d = ring + 2 * s * C::TILE_BYTES;
#pragma unroll
            for (int c = 0; c < C::NB; ++c) {
              tma_head(d + c * C::BN * 128, &mq, &full[s], 64 * c, i0, h, u);
              tma_head(d + C::TILE_BYTES + c * C::BN * 128, &mdo, &full[s], 64 * c, i0, h, u);
            }
          }
        }
        ok = drain_tma<C::STAGES>(ok, full, empty, it, kv_full, kv_free, nkv);
        if (!ok) atomicExch(&g_error_flag, 31);
      }
    } else if (warp == 9) {
      {
        const uint32_t id_s = idesc_of(ta.fmt, C::BN, 0), id_o = idesc_of(ta.fmt, ta.n_hd, 1);
        const uint32_t k0 = smem_u32(sK), v0 = smem_u32(sV), r0 = smem_u32(ring);
        bool ok = true;
        int g = 0, units = 0;  // tiles of all units: ring, S buffers and barriers go by g
        auto q_tile = [&](int i) { return r0 + 2 * (i % C::STAGES) * C::TILE_BYTES; };
        auto issue_s = [&](int i) {
          if (!warp_wait(&full[i % C::STAGES], (i / C::STAGES) & 1)) return false;
          tc_fence_after();
          if (elect_one())
            mma_heads<HD>(tmem + C::S_COL + (i % C::SB) * C::BN, k0, q_tile(i), 128, C::BN, ta.ksteps, id_s);
          __syncwarp();
          return true;
        };
        auto issue_dp = [&](int i, bool last) {
          if (i > 0 && !warp_wait(dp_free, (i - 1) & 1)) return false;
          tc_fence_after();
          if (elect_one()) {
            mma_heads<HD>(tmem + C::DP_COL, v0, q_tile(i) + C::TILE_BYTES, 128, C::BN, ta.ksteps, id_s);
            umma_commit(dp_full);
            if (last) umma_commit(kv_free);
          }
          __syncwarp();
          return true;
        };
        for (int k = 0; ok; ++k) {
          const int ui = unit_index(k);
          if (ui >= ta.units && k * (int)gridDim.x >= ta.units) break;
          if (ui >= ta.units) continue;
          const TcUnit u = tc_unit(ta, a.kv_heads, ui, false);
          const Bounds b = bounds_of(a, u.seq);
          int begin, per, t0, t1;
          range(u, b, begin, per, t0, t1);
          if (t0 >= t1) continue;
          const int n = t1 - t0;
          if (!warp_wait(kv_full, units & 1) || !issue_s(g) || !issue_dp(g, n == 1)) {
            ok = false;
            break;
          }
          for (int t = 0; t < n; ++t) {
            if (C::SB == 2 && t + 1 < n && (!issue_s(g + t + 1) || !issue_dp(g + t + 1, t + 2 == n))) {
              ok = false;
              break;
            }
            if ((t == 0 && units > 0 && !warp_wait(acc_free, (units - 1) & 1)) ||
                !warp_wait(&ps_ready[(g + t) & 1], ((g + t) >> 1) & 1)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t p = tmem + C::S_COL + ((g + t) % C::SB) * C::BN, q = q_tile(g + t);
            // The chunk of K step ks (16 queries, 8 columns): P in its first half, dS in its second.
            constexpr int KC = C::CH / 16;
            auto p_col = [&](int ks) { return p + (ks / KC) * C::CH + (ks % KC) * 8; };
            auto ds_col = [&](int ks) { return p_col(ks) + C::CH / 2; };
            if (elect_one()) {
              mma_rows<C::BN / 16>(tmem + C::DV_COL, p_col, q + C::TILE_BYTES, C::BN * 128, id_o, t > 0 ? 1u : 0u);
              mma_rows<C::BN / 16>(tmem + C::DK_COL, ds_col, q, C::BN * 128, id_o, t > 0 ? 1u : 0u);
              umma_commit(&empty[(g + t) % C::STAGES]);
              if (t + 1 == n) umma_commit(acc_done);
            }
            __syncwarp();
            if (C::SB == 1 && t + 1 < n && (!issue_s(g + t + 1) || !issue_dp(g + t + 1, t + 2 == n))) {
              ok = false;
              break;
            }
          }
          if (!ok) break;
          g += n;
          ++units;
        }
        if (!ok) {
          drain_mma(idle);
          if (lane == 0) atomicExch(&g_error_flag, 32);
        }
      }
    } else if (warp == 10) {
      // (-lse in log2 units, -D) of each streamed tile; -inf and 0 for rows outside the queries.
      bool ok = true;
      int g = 0;
      for (int k = 0; ok; ++k) {
        const int ui = unit_index(k);
        if (ui >= ta.units && k * (int)gridDim.x >= ta.units) break;
        if (ui >= ta.units) continue;
        const TcUnit u = tc_unit(ta, a.kv_heads, ui, false);
        const Bounds b = bounds_of(a, u.seq);
        int begin, per, t0, t1;
        range(u, b, begin, per, t0, t1);
        if (t0 >= t1) continue;
        Walk wk(t0, per);
        for (int t = t0; t < t1; ++t, ++g, wk.next()) {
          const int h = u.h * a.group + wk.head, i0 = (begin + wk.tile) * C::BN;
          const long long row0 = ((long long)u.seq * a.heads + h) * a.lq + i0;
          const int sb = g % C::STATS, r = g / C::STATS;
          float l[C::BN / 32], d[C::BN / 32];
#pragma unroll
          for (int e = 0; e < C::BN / 32; ++e) {
            const int i = 32 * e + lane;
            const float2 x = i0 + i < b.ql ? ta.stats[row0 + i] : make_float2(-INFINITY, 0.f);
            l[e] = x.x + p_shift<T>();
            d[e] = x.y;
          }
          if (r > 0 && !warp_wait(&st_free[sb], (r - 1) & 1)) {
            ok = false;
            break;
          }
          float* s = stats + sb * 2 * C::BN;
#pragma unroll
          for (int e = 0; e < C::BN / 32; ++e) {
            s[32 * e + lane] = l[e];
            s[C::BN + 32 * e + lane] = d[e];
          }
          mbar_arrive(&st_full[sb]);
        }
      }
      if (!ok && lane == 0) atomicExch(&g_error_flag, 34);
    }
  } else {
    regs_up<C::REGS_MORE>();
    const int half = warp >> 2, row = threadIdx.x & 127;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const float c = a.scale * LOG2E;
    const float unshift = exp2f(-p_shift<T>());
    const float2 c2 = make_float2(c, c);
    const long long rows = (long long)a.seqs * a.kv_heads * a.lk;
    bool ok = true;
    int g = 0, units = 0;
    for (int k = 0; ok; ++k) {
      const int ui = unit_index(k);
      if (ui >= ta.units && k * (int)gridDim.x >= ta.units) break;
      if (ui >= ta.units) continue;
      const TcUnit u = tc_unit(ta, a.kv_heads, ui, false);
      const Bounds b = bounds_of(a, u.seq);
      int begin, per, t0, t1;
      range(u, b, begin, per, t0, t1);
      const int j0 = u.tile * ROWS, j = j0 + row;
      float ds_scale = unshift, dk_scale = a.scale;  // of dS next to P, and back
      if constexpr (std::is_same<T, __half>::value) {
        const uint4 r = *reinterpret_cast<const uint4*>(a.range + 4 * ((long long)u.seq * a.kv_heads + u.h));
        const int shift = fp16_shift(
            __float_as_uint(fmaf(__uint_as_float(r.x), __uint_as_float(r.y), __uint_as_float(r.z))));
        ds_scale *= pow2(shift);
        dk_scale *= pow2(-shift);
      }
      const float2 un2 = make_float2(ds_scale, ds_scale);
      const int first = a.causal ? max(0, -b.off) : 0;       // queries before it see no key
      const int from = a.causal ? max(first, j - b.off) : 0; // this key is seen by queries [from, b.ql)
      // A thread's queries of a tile go in two chunks; the loads of the next one are in flight during this one's
      // exponentials.
      uint32_t s0[C::CH], d0[C::CH], s1[C::CH], d1[C::CH];
      auto load = [&](int tile, int chunk, uint32_t (&s)[C::CH], uint32_t (&d)[C::CH]) {
        tmem_ld_async(lanes + C::DP_COL + half * C::HALF + C::CH * chunk, d);
        tmem_ld_async(lanes + C::S_COL + (tile % C::SB) * C::BN + half * C::HALF + C::CH * chunk, s);
      };
      auto arrived = [&](int tile) {  // S, dP and the row statistics of a tile
        return warp_wait(&st_full[tile % C::STATS], (tile / C::STATS) & 1) && warp_wait(dp_full, tile & 1);
      };
      // P^T and dS^T of one chunk, stored over its scores.
      auto chunk_pds = [&](int i0, int chunk, bool edge, uint32_t (&s)[C::CH], uint32_t (&d)[C::CH]) {
        const int col = half * C::HALF + C::CH * chunk;
        const float* row_stats = stats + (g % C::STATS) * 2 * C::BN + col;
        const float4* l4 = reinterpret_cast<const float4*>(row_stats);
        const float4* d4 = reinterpret_cast<const float4*>(row_stats + C::BN);
        if (edge) {
          const int lo = from - i0 - col, hi = b.ql - i0 - col;
#pragma unroll
          for (int e = 0; e < C::CH; ++e)
            if (e < lo || e >= hi) s[e] = __float_as_uint(-INFINITY), d[e] = 0;
        }
        uint32_t w[C::CH];  // P, then dS
#pragma unroll
        for (int e = 0; e < C::CH / 4; ++e) {
          const float4 l = l4[e], dd = d4[e];
          const float2 xa = ub::fma2(make_float2(__uint_as_float(s[4 * e]), __uint_as_float(s[4 * e + 1])), c2,
                                     make_float2(l.x, l.y));
          const float2 xb = ub::fma2(make_float2(__uint_as_float(s[4 * e + 2]), __uint_as_float(s[4 * e + 3])), c2,
                                     make_float2(l.z, l.w));
          const float2 pa = make_float2(ex2(xa.x), ex2(xa.y)), pb = make_float2(ex2(xb.x), ex2(xb.y));
          float2 ga = add2(make_float2(__uint_as_float(d[4 * e]), __uint_as_float(d[4 * e + 1])),
                           make_float2(dd.x, dd.y));
          float2 gb = add2(make_float2(__uint_as_float(d[4 * e + 2]), __uint_as_float(d[4 * e + 3])),
                           make_float2(dd.z, dd.w));
          if (p_shift<T>() != 0.f) ga = mul2(ga, un2), gb = mul2(gb, un2);
          ga = mul2(pa, ga);
          gb = mul2(pb, gb);
          w[2 * e] = pack2<T>(pa.x, pa.y);
          w[2 * e + 1] = pack2<T>(pb.x, pb.y);
          w[C::CH / 2 + 2 * e] = pack2<T>(ga.x, ga.y);
          w[C::CH / 2 + 2 * e + 1] = pack2<T>(gb.x, gb.y);
        }
        const uint32_t to = lanes + C::S_COL + (g % C::SB) * C::BN + col;
        if constexpr (C::CH == 32)
          tmem_st32(to, w);
        else
          tmem_st16(to, w);
      };
      Walk w(t0 < t1 ? t0 : 0, per);
      if (!C::EARLY && t0 < t1) {
        if (!arrived(g)) {
          ok = false;
          break;
        }
        tc_fence_after();
        load(g, 0, s0, d0);
      }
      for (int t = t0; t < t1; ++t, ++g, w.next()) {
        const int i0 = (begin + w.tile) * C::BN;
        // Queries past the tensor need no mask: their rows were read as 0 and come with -lse = -inf.
        const bool edge = (a.q_lens && i0 + C::BN > b.ql) || i0 < first || (a.causal && j0 + ROWS - 1 > i0 + b.off);
        if (C::EARLY) {
          if (!arrived(g)) {
            ok = false;
            break;
          }
          tc_fence_after();
          load(g, 0, s0, d0);
        }
        if (!C::EARLY) {
          tmem_wait_ld(s0);
          tmem_wait_ld(d0);
        }
        load(g, 1, s1, d1);
        if (C::EARLY) {
          tmem_wait_ld(s0);
          tmem_wait_ld(d0);
        } else {
          chunk_pds(i0, 0, edge, s0, d0);
        }
        tmem_wait_ld(s1);
        tmem_wait_ld(d1);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(dp_free);
        if (C::EARLY) chunk_pds(i0, 0, edge, s0, d0);
        // Rows of Q and dO that must not count (NaN included) become 0 before they are summed over.
        if (edge && ((a.q_lens && i0 + C::BN > b.ql) || i0 < first)) {
          if (row < C::BN && (i0 + row >= b.ql || i0 + row < first))
            clear_row(ring + (2 * (g % C::STAGES) + half) * C::TILE_BYTES, C::BN, C::NB, row);
          fence_proxy_async_smem();
        }
        chunk_pds(i0, 1, edge, s1, d1);
        if (!C::EARLY && t + 1 < t1) {
          if (!arrived(g + 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          load(g + 1, 0, s0, d0);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&ps_ready[g & 1]);
          mbar_arrive(&st_free[g % C::STATS]);
        }
      }
      if (!ok) break;
      if (t0 < t1) {
        if (!warp_wait(acc_done, units & 1)) {
          ok = false;
          break;
        }
        ++units;
        tc_fence_after();
      }
      const bool live = j < b.kl && t0 < t1;
      const long long orow = ((long long)u.seq * a.kv_heads + u.h) * a.lk + j;
      // Threads of half 0 write dV, of half 1 dK.
      T* out = static_cast<T*>(half ? a.dk : a.dv) + unit_offset(half ? a.dk_s : a.dv_s, u, u.h) +
               (long long)j * (half ? a.dk_s.row : a.dv_s.row);
      float* part = a.splits > 1 ? a.part + ((half ? 0 : a.splits) + u.split) * rows * a.hd + orow * a.hd : nullptr;
      const float mul = half ? dk_scale : unshift;
#pragma unroll 1
      for (int q = 0; q < HD / 32; ++q) {
        uint32_t v[32];
        if (t0 < t1) tmem_ld32(lanes + (half ? C::DK_COL : C::DV_COL) + 32 * q, v);
        if (!live) {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0;
        }
        const int n = a.hd - 32 * q;
        if (j < a.lk && n > 0) {
          if (part)
            store_cols_f32(part + 32 * q, v, mul, n);
          else
            store_cols<T>(out + 32 * q, v, mul, n);
        }
      }
      if (t0 < t1) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_free);
      }
    }
    if (!ok) {
      tmem_wait_ld();
      tmem_st_wait();
      atomicExch(&g_error_flag, 33);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM);
  }
}

// ------------------------------------------------------------------------------------------------- host

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

// (dim, row, head, inner, outer) map of a tensor: boxes of 64 dims x `box_rows` rows of one head.
bool head_map(CUtensorMap* m, const void* base, const UnblendHeadStrides& s, const UnblendAttnTrainParams& p, int heads,
              int rows, int box_rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  auto legal = [](long long st, int n) { return (cuuint64_t)(n == 1 ? 16 : st * 2); };
  cuuint64_t dims[5] = {(cuuint64_t)p.hd, (cuuint64_t)rows, (cuuint64_t)heads, (cuuint64_t)p.inner,
                        (cuuint64_t)p.outer};
  cuuint64_t strides[4] = {legal(s.row, rows), legal(s.head, heads), legal(s.inner, p.inner),
                           legal(s.outer, p.outer)};
  cuuint32_t box[5] = {64, (cuuint32_t)box_rows, 1, 1, 1};
  cuuint32_t es[5] = {1, 1, 1, 1, 1};
  return fn(m, p.dtype == UNBLEND_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
            const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

TcArgs tc_args(const AttnArgs& a, const UnblendAttnTrainParams& p, int heads, int len, int rows_per_unit, int splits,
               float* part) {
  TcArgs t{};
  t.a = a;
  t.a.splits = splits;
  t.a.part = splits > 1 ? part : nullptr;
  t.row_tiles = (len + rows_per_unit - 1) / rows_per_unit;
  t.units = (int)((long long)a.seqs * heads * t.row_tiles * splits);
  t.ksteps = (p.hd + 15) / 16;
  t.n_hd = 16 * t.ksteps;
  t.fmt = p.dtype == UNBLEND_BF16 ? 1u : 0u;
  t.by_splits = fast_div(splits);
  t.by_tiles = fast_div(t.row_tiles);
  t.by_heads = fast_div(heads);
  t.by_inner = fast_div(a.inner);
  t.by_group = fast_div(a.group);
  t.by_seq_heads = fast_div((long long)a.seqs * heads);
  t.stats = reinterpret_cast<const float2*>(a.dsum);
  return t;
}

int grid_of(int units, int per_sm) { return units < per_sm * ub::kNumSMs ? units : per_sm * ub::kNumSMs; }

template <typename T, int HD, int NQ, bool SHORT>
int launch_fwd(const AttnArgs& a, const UnblendAttnTrainParams& p, int splits, cudaStream_t st) {
  using C = FwdCfg<HD, NQ, SHORT>;
  CUtensorMap mq, mk, mv;
  if (!head_map(&mq, a.q, p.q, p, p.heads, p.lq, 128) || !head_map(&mk, a.k, p.k, p, p.kv_heads, p.lk, C::BN) ||
      !head_map(&mv, a.v, p.v, p, p.kv_heads, p.lk, C::BN))
    return UNBLEND_ERR_INVALID;
  const TcArgs t = tc_args(a, p, p.heads, p.lq, NQ * ROWS, splits, a.part);
  constexpr auto kern = attention_fwd_tc_kernel<T, HD, NQ, SHORT>;
  if (allow_smem<kern>(C::SMEM) != cudaSuccess) return (int)cudaGetLastError();
  kern<<<grid_of(t.units, C::PER_SM), C::THREADS, C::SMEM, st>>>(mq, mk, mv, t);
  UB_CHECK_LAUNCH();
  return 0;
}

template <typename T, int LANES>
int launch_stats_lanes(const AttnArgs& a, cudaStream_t st) {
  float2* stats = reinterpret_cast<float2*>(a.dsum);
  if constexpr (std::is_same<T, __half>::value) {
    constexpr int STEP = STATS_ROWS * 32 / LANES;
    RangeArgs ra{};
    // About 32 warps per SM, what runs at once; a unit's rows are of one head, whose units are alike.
    const long long rows = (long long)a.seqs * ((long long)a.heads * a.lq + (long long)a.kv_heads * a.lk);
    const long long most = rows / (32LL * ub::kNumSMs * STEP);  // steps of a unit
    auto share = [&](int len, int* chunks, int* each) {
      const int steps = (len + STEP - 1) / STEP;
      *each = (int)(most < 1 ? 1 : most < steps ? most : steps);
      *chunks = (steps + *each - 1) / *each;
      *each = (steps + *chunks - 1) / *chunks;
    };
    share(a.lq, &ra.q_chunks, &ra.q_steps);
    share(a.lk, &ra.v_chunks, &ra.v_steps);
    ra.q_units = (unsigned)((long long)a.seqs * a.heads * ra.q_chunks);
    ra.units = ra.q_units + (unsigned)((long long)a.seqs * a.kv_heads * ra.v_chunks);
    ra.by_heads = fast_div(a.heads);
    ra.by_kv_heads = fast_div(a.kv_heads);
    ra.by_q_chunks = fast_div(ra.q_chunks);
    ra.by_v_chunks = fast_div(ra.v_chunks);
    ra.by_group = fast_div(a.group);
    ra.by_inner = fast_div(a.inner);
    if (cudaMemsetAsync(a.range, 0, sizeof(unsigned) * 4 * a.seqs * a.kv_heads, st) != cudaSuccess)
      return (int)cudaGetLastError();
    attention_stats_range_kernel<T, LANES><<<ra.units / 8 + (ra.units % 8 != 0), 256, 0, st>>>(a, stats, ra);
  } else {
    constexpr int PER_CTA = STATS_ROWS * 256 / LANES;
    const long long rows = (long long)a.seqs * a.lq * a.heads;
    attention_stats_kernel<T, LANES><<<(unsigned)((rows + PER_CTA - 1) / PER_CTA), 256, 0, st>>>(
        a, stats, fast_div(a.heads), fast_div(a.lq), fast_div(a.inner));
  }
  UB_CHECK_LAUNCH();
  return 0;
}

template <typename T>
int launch_stats(const AttnArgs& a, cudaStream_t st) {
  if (a.hd <= 32) return launch_stats_lanes<T, 4>(a, st);
  return a.hd <= 64 ? launch_stats_lanes<T, 8>(a, st) : launch_stats_lanes<T, 16>(a, st);
}

template <typename T, int HD, bool SHORT>
int launch_dq(const AttnArgs& a, const UnblendAttnTrainParams& p, int splits, float* part, cudaStream_t st) {
  using C = DqCfg<HD, SHORT>;
  CUtensorMap mq, mdo, mk, mv;
  if (!head_map(&mq, a.q, p.q, p, p.heads, p.lq, 128) || !head_map(&mdo, a.dout, p.dout, p, p.heads, p.lq, 128) ||
      !head_map(&mk, a.k, p.k, p, p.kv_heads, p.lk, C::BN) || !head_map(&mv, a.v, p.v, p, p.kv_heads, p.lk, C::BN))
    return UNBLEND_ERR_INVALID;
  const TcArgs t = tc_args(a, p, p.heads, p.lq, ROWS, splits, part);
  constexpr auto kern = attention_dq_tc_kernel<T, HD, SHORT>;
  if (allow_smem<kern>(C::SMEM) != cudaSuccess) return (int)cudaGetLastError();
  kern<<<grid_of(t.units, 1), C::THREADS, C::SMEM, st>>>(mq, mdo, mk, mv, t);
  UB_CHECK_LAUNCH();
  return 0;
}

template <typename T, int HD, bool SHORT>
int launch_dkv(const AttnArgs& a, const UnblendAttnTrainParams& p, int splits, float* part, cudaStream_t st) {
  using C = DkvCfg<HD, SHORT>;
  CUtensorMap mq, mdo, mk, mv;
  if (!head_map(&mq, a.q, p.q, p, p.heads, p.lq, C::BN) || !head_map(&mdo, a.dout, p.dout, p, p.heads, p.lq, C::BN) ||
      !head_map(&mk, a.k, p.k, p, p.kv_heads, p.lk, 128) || !head_map(&mv, a.v, p.v, p, p.kv_heads, p.lk, 128))
    return UNBLEND_ERR_INVALID;
  const TcArgs t = tc_args(a, p, p.kv_heads, p.lk, ROWS, splits, part);
  constexpr auto kern = attention_dkv_tc_kernel<T, HD, SHORT>;
  if (allow_smem<kern>(C::SMEM) != cudaSuccess) return (int)cudaGetLastError();
  kern<<<grid_of(t.units, 1), C::THREADS, C::SMEM, st>>>(mk, mv, mq, mdo, t);
  UB_CHECK_LAUNCH();
  return 0;
}

}  // namespace

namespace ub {
namespace train {

template <typename F>
int by_type(const UnblendAttnTrainParams& p, F go) {
  return p.dtype == UNBLEND_BF16 ? go(__nv_bfloat16()) : go(__half());
}

int attention_stats_tc(const AttnArgs& a, const UnblendAttnTrainParams& p, cudaStream_t st) {
  return by_type(p, [&](auto x) { return launch_stats<decltype(x)>(a, st); });
}

int attention_fwd_tc(const AttnArgs& a, const UnblendAttnTrainParams& p, int rows_per_cta, cudaStream_t st) {
  return by_type(p, [&](auto x) {
    using T = decltype(x);
    if (p.hd <= 64 && p.lk <= SHORT_ROWS) return launch_fwd<T, 64, 1, true>(a, p, a.splits, st);
    if (rows_per_cta == 256) return launch_fwd<T, 128, 2, false>(a, p, a.splits, st);  // head dims over 64 only
    return p.hd <= 64 ? launch_fwd<T, 64, 1, false>(a, p, a.splits, st)
                      : launch_fwd<T, 128, 1, false>(a, p, a.splits, st);
  });
}

int attention_dq_tc(const AttnArgs& a, const UnblendAttnTrainParams& p, int splits, float* part, cudaStream_t st) {
  return by_type(p, [&](auto x) {
    using T = decltype(x);
    if (p.hd > 64) return launch_dq<T, 128, false>(a, p, splits, part, st);
    return p.lk <= SHORT_ROWS ? launch_dq<T, 64, true>(a, p, splits, part, st)
                              : launch_dq<T, 64, false>(a, p, splits, part, st);
  });
}

int attention_dkv_tc(const AttnArgs& a, const UnblendAttnTrainParams& p, int splits, float* part, cudaStream_t st) {
  return by_type(p, [&](auto x) {
    using T = decltype(x);
    if (p.hd > 64) return launch_dkv<T, 128, false>(a, p, splits, part, st);
    return p.lq <= SHORT_ROWS ? launch_dkv<T, 64, true>(a, p, splits, part, st)
                              : launch_dkv<T, 64, false>(a, p, splits, part, st);
  });
}

// Rows of whole 16-byte chunks, and a positive scale (the row maximum is taken before the scale).
bool attention_tc_sizes(const UnblendAttnTrainParams& p) {
  return p.dtype != UNBLEND_F32 && p.hd % 8 == 0 && p.scale > 0.f;
}

// What the tensor-core kernels can address: bases and strides of whole 16-byte chunks (TMA, vector stores).
bool attention_tc_fits(const UnblendAttnTrainParams& p, const void* const* ptrs, const UnblendHeadStrides* strides,
                       const int* heads, const int* rows, int n) {
  if (!attention_tc_sizes(p)) return false;
  for (int i = 0; i < n; ++i) {
    if (reinterpret_cast<uintptr_t>(ptrs[i]) % 16 != 0) return false;
    const UnblendHeadStrides& s = strides[i];
    const long long st[4] = {s.row, s.head, s.inner, s.outer};
    const int ext[4] = {rows[i], heads[i], p.inner, p.outer};
    for (int k = 0; k < 4; ++k)
      if (ext[k] > 1 && (st[k] <= 0 || st[k] % 8 != 0 || st[k] >= (1LL << 38))) return false;
  }
  return true;
}

}  // namespace train
}  // namespace ub

extern "C" int unblend_attention_train_error_flag(int* out_host, int clear) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_error_flag, sizeof(int));
  if (e != cudaSuccess) return (int)e;
  if (out_host) *out_host = v;
  if (clear) {
    int z = 0;
    e = cudaMemcpyToSymbol(g_error_flag, &z, sizeof(int));
    if (e != cudaSuccess) return (int)e;
  }
  return 0;
}
