// Dropout of a residual branch with its LayerScale and residual add, and the gradients:
//
//   y  = residual + scale[c] * keep * x / (1 - p)
//   dx = scale[c] * keep * dy / (1 - p),   dscale[c] = sum_rows keep * x * dy / (1 - p)
//
// keep is never stored: element e = row * cols + c is kept when word e % 4 of Philox-4x32-10 (Salmon, Moraes, Dror,
// Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011) with key = seed and counter = (e / 4, offset) is at
// least round(p 2^32). Both directions draw the same words from (seed, offset), which lie in device memory so that a
// captured graph can be replayed with new ones. A dropped element is selected away, not multiplied by 0: infinities
// and NaN in it leave no trace.
//
// Bound: HBM for fp32. With 16-bit tensors the generator (a block of four words is 10 rounds of two 32 x 32 -> 64 bit
// products) shares the time with 4 to 10 bytes per element and nothing is full: all bf16 forward, issue slots are 56 %
// busy, DRAM 33 %, and warps wait for loads. Measured, 86016 x 512 with
// all gradients: fp32 72 us forward (7.3 TB/s), 94 us backward (5.6); bf16 on an fp32 stream 84 us (5.2 TB/s) and 78 us
// (4.5); all bf16 74 us (3.6) and 79 us (3.3).
//
// Three kernels. Contiguous tensors on 16-byte boundaries, whatever their width, are one run of 16-byte chunks (flat).
// Strided rows that are whole 16-byte chunks keep those (vector), and all others are read element by element with the
// words shared by ballots (any). Both sides at 50000 x 1001, bf16 on an fp32 stream: flat 98 us forward and 89 us
// backward, any 183 and 286 us; at 86016 x 512 backward: flat 78 us, vector 122 us.
#include <cmath>
#include <type_traits>

#include "train_common.cuh"

namespace {

using namespace ub::train;

struct DropArgs {
  const void* x;
  const void* r;  // residual (forward, may be null) or dy (backward)
  const void* scale;
  void* out;      // y (the stream's type) or dx (x's type)
  float* part;    // backward: [gridDim.y][cols], null without dscale
  const unsigned long long* rng;
  RowMap xm, rm;
  unsigned rows;
  int cols;
  uint32_t threshold;  // words below it are dropped; p that rounds to 2^32 drops all of them
  int drop_all;
  float inv_keep;
};

struct Words {
  uint32_t w[4];
};

__device__ __forceinline__ Words philox(unsigned long long seed, unsigned long long offset, unsigned long long block) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Words{{c0, c1, c2, c3}};
}

// Strided rows, columns in runs of VEC (a multiple of 4, so a run is whole word blocks): thread (tx, ty) keeps its
// columns and walks the rows blockIdx.y * TY + ty + k * gridDim.y * TY.
template <typename T, typename TR, typename TW, int VEC, bool BWD, bool SUMS>
__global__ void __launch_bounds__(256) dropout_add_vec_kernel(const __grid_constant__ DropArgs a) {
  extern __shared__ float red[];  // [TY][TX * VEC] of the backward sums
  const int tx = threadIdx.x, ty = threadIdx.y;
  const int c = (blockIdx.x * blockDim.x + tx) * VEC;
  const bool active = c < a.cols;
  const unsigned long long seed = a.rng[0], offset = a.rng[1];
  const bool any = !a.drop_all;
  float s[VEC], ds[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) s[i] = 1.f, ds[i] = 0.f;
  if (a.scale && active) load_vec<TW, VEC>(static_cast<const TW*>(a.scale) + c, s);
  if (active) {
    for (long long row = (long long)blockIdx.y * blockDim.y + ty; row < a.rows;
         row += (long long)gridDim.y * blockDim.y) {
      const long long e = row * a.cols + c;
      float x[VEC], r[VEC], o[VEC];
      if (!BWD || SUMS) load_vec<T, VEC>(static_cast<const T*>(a.x) + row_offset(a.xm, (unsigned)row) + c, x);
      if (BWD || a.r) load_vec<TR, VEC>(static_cast<const TR*>(a.r) + row_offset(a.rm, (unsigned)row) + c, r);
#pragma unroll
      for (int b = 0; b < VEC / 4; ++b) {
        const Words w = philox(seed, offset, (unsigned long long)(e >> 2) + b);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = b * 4 + j;
          const bool keep = any && w.w[j] >= a.threshold;
          if constexpr (BWD) {
            const float d = keep ? r[i] * a.inv_keep : 0.f;
            o[i] = s[i] * d;
            if (SUMS) ds[i] += keep ? d * x[i] : 0.f;
          } else {
            const float v = keep ? s[i] * (x[i] * a.inv_keep) : 0.f;
            o[i] = a.r ? r[i] + v : v;
          }
        }
      }
      if constexpr (BWD)
        store_vec<T, VEC>(static_cast<T*>(a.out) + e, o);
      else
        store_vec<TR, VEC>(static_cast<TR*>(a.out) + e, o);
    }
  }
  if constexpr (SUMS) {
    const int width = blockDim.x * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) red[ty * width + tx * VEC + i] = ds[i];
    __syncthreads();
    if (ty == 0 && active) {
      for (int y = 1; y < (int)blockDim.y; ++y)
#pragma unroll
        for (int i = 0; i < VEC; ++i) ds[i] += red[y * width + tx * VEC + i];
#pragma unroll
      for (int i = 0; i < VEC; ++i) a.part[(long long)blockIdx.y * a.cols + c + i] = ds[i];
    }
  }
}

// Any width and alignment: a warp takes 124 consecutive columns of a row. Wherever the run starts within a block of
// four words, it lies in 32 consecutive blocks: lane l draws block l, four ballots carry the keep bits, and lane l
// handles columns l, l + 32, l + 64, l + 96 of the run, so that accesses stay coalesced.
constexpr int RUN = 124;

template <typename T, typename TR, typename TW, bool BWD>
__global__ void __launch_bounds__(256) dropout_add_any_kernel(const __grid_constant__ DropArgs a) {
  __shared__ float red[8][RUN + 4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c0 = blockIdx.x * RUN;
  const int n = min(RUN, a.cols - c0);
  const unsigned long long seed = a.rng[0], offset = a.rng[1];
  const bool any = !a.drop_all;
  float s[4], ds[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int k = 32 * i + lane;
    s[i] = a.scale && k < n ? to_f(static_cast<const TW*>(a.scale)[c0 + k]) : 1.f;
    ds[i] = 0.f;
  }
  for (long long row = (long long)blockIdx.y * 8 + warp; row < a.rows; row += (long long)gridDim.y * 8) {
    const long long e0 = row * a.cols + c0;
    const int shift = (int)(e0 & 3);
    const Words w = philox(seed, offset, (unsigned long long)(e0 >> 2) + lane);
    uint32_t bits[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) bits[j] = __ballot_sync(0xffffffffu, any && w.w[j] >= a.threshold);
    const T* x = static_cast<const T*>(a.x) + (!BWD || a.part ? row_offset(a.xm, (unsigned)row) + c0 : 0);
    const TR* r = static_cast<const TR*>(a.r) + (a.r ? row_offset(a.rm, (unsigned)row) + c0 : 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = 32 * i + lane;
      if (k < n) {
        const int q = shift + k, j = q & 3;
        const uint32_t b = j == 0 ? bits[0] : j == 1 ? bits[1] : j == 2 ? bits[2] : bits[3];
        const bool keep = (b >> (q >> 2)) & 1u;
        if constexpr (BWD) {
          const float d = keep ? to_f(r[k]) * a.inv_keep : 0.f;
          if (a.part) ds[i] += keep ? d * to_f(x[k]) : 0.f;
          static_cast<T*>(a.out)[e0 + k] = from_f<T>(s[i] * d);
        } else {
          const float v = keep ? s[i] * (to_f(x[k]) * a.inv_keep) : 0.f;
          static_cast<TR*>(a.out)[e0 + k] = from_f<TR>(a.r ? to_f(r[k]) + v : v);
        }
      }
    }
  }
  if constexpr (BWD) {
    if (a.part == nullptr) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) red[warp][32 * i + lane] = ds[i];
    __syncthreads();
    for (int k = threadIdx.x; k < n; k += blockDim.x) {
      float t = red[0][k];
#pragma unroll
      for (int y = 1; y < 8; ++y) t += red[y][k];
      a.part[(long long)blockIdx.y * a.cols + c0 + k] = t;
    }
  }
}

// Contiguous tensors of any width, as one run of 16-byte chunks: T = cols * m threads take chunk t, t + T, ..., and as
// T chunks are whole rows, a thread's columns stay the same. Its sums are then entries t * VEC ... of a [VEC * m][cols]
// array of partial sums as they are; where a CTA's entries cover each column twice or more it adds those and leaves one
// row.
constexpr bool flat_joins(int cols, int vec) { return 2 * cols <= 256 * vec; }

template <typename T, typename TR, typename TW, bool BWD, bool SUMS>
__global__ void __launch_bounds__(256) dropout_add_flat_kernel(const __grid_constant__ DropArgs a, int threads) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (!SUMS && t >= threads) return;
  const unsigned long long seed = a.rng[0], offset = a.rng[1];
  const bool any = !a.drop_all;
  const long long n = (long long)a.rows * a.cols, step = (long long)threads * VEC;
  float s[VEC], ds[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    s[i] = a.scale ? to_f(static_cast<const TW*>(a.scale)[((long long)t * VEC + i) % a.cols]) : 1.f;
    ds[i] = 0.f;
  }
  for (long long e = t < threads ? (long long)t * VEC : n; e < n; e += step) {
    float x[VEC], r[VEC], o[VEC];
    const bool whole = e + VEC <= n;
    if (whole) {
      if (!BWD || SUMS) load_vec<T, VEC>(static_cast<const T*>(a.x) + e, x);
      if (BWD || a.r) load_vec<TR, VEC>(static_cast<const TR*>(a.r) + e, r);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        x[i] = (!BWD || SUMS) && e + i < n ? to_f(static_cast<const T*>(a.x)[e + i]) : 0.f;
        r[i] = (BWD || a.r) && e + i < n ? to_f(static_cast<const TR*>(a.r)[e + i]) : 0.f;
      }
    }
#pragma unroll
    for (int b = 0; b < VEC / 4; ++b) {
      const Words w = philox(seed, offset, (unsigned long long)(e >> 2) + b);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = b * 4 + j;
        const bool keep = any && w.w[j] >= a.threshold;
        if constexpr (BWD) {
          const float d = keep ? r[i] * a.inv_keep : 0.f;
          o[i] = s[i] * d;
          if (SUMS) ds[i] += keep ? d * x[i] : 0.f;
        } else {
          const float v = keep ? s[i] * (x[i] * a.inv_keep) : 0.f;
          o[i] = a.r ? r[i] + v : v;
        }
      }
    }
    using TO = typename std::conditional<BWD, T, TR>::type;
    TO* out = static_cast<TO*>(a.out) + e;
    if (whole) {
      store_vec<TO, VEC>(out, o);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (e + i < n) out[i] = from_f<TO>(o[i]);
    }
  }
  if constexpr (SUMS) {
    if (!flat_joins(a.cols, VEC)) {
      if (t < threads) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) a.part[(long long)t * VEC + i] = ds[i];
      }
      return;
    }
    __shared__ float sums[256 * VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) sums[threadIdx.x * VEC + i] = ds[i];
    __syncthreads();
    const int first = (int)((long long)blockIdx.x * 256 * VEC % a.cols);  // column of entry 0
    for (int c = threadIdx.x; c < a.cols; c += 256) {
      float v = 0.f;
      for (int e = c >= first ? c - first : c - first + a.cols; e < 256 * VEC; e += a.cols) v += sums[e];
      a.part[(long long)blockIdx.x * a.cols + c] = v;
    }
  }
}

enum Path { ANY, VECTOR, FLAT };

struct Shape {
  dim3 grid, block;
};

// m of the flat kernel, no more than the rows need. Without sums about eight CTAs per SM (fp32 86016 x 512 backward:
// 67 us, with four 81 us; bf16 74 and 76 us); with sums four, as each CTA leaves partial sums.
constexpr int FLAT_CTAS = 8, FLAT_SUM_CTAS = 4;

long long flat_runs(long long rows, int cols, int vec, int ctas_per_sm) {
  const long long fill = ctas_per_sm * 256LL * ub::kNumSMs / cols, need = (rows + vec - 1) / vec;
  const long long m = fill < need ? fill : need;
  return m < 1 ? 1 : m;
}

// Row CTAs: enough to fill the GPU, at most one per `rows_per_cta` rows; the backward partial sums have one row each.
unsigned row_ctas(long long rows, int rows_per_cta, unsigned col_ctas, int per_sm) {
  const long long most = (rows + rows_per_cta - 1) / rows_per_cta;
  long long n = (long long)per_sm * ub::kNumSMs / col_ctas;
  if (n < 1) n = 1;
  return (unsigned)(n < most ? n : most);
}

Shape vec_shape(long long rows, int cols, int vec) {
  const int cv = cols / vec;
  Shape s;
  s.block = dim3(cv < 256 ? cv : 256, cv < 256 ? 256 / cv : 1);
  const unsigned gx = (cv + s.block.x - 1) / s.block.x;
  s.grid = dim3(gx, row_ctas(rows, s.block.y, gx, 8));
  return s;
}

Shape any_shape(long long rows, int cols) {
  Shape s;
  s.block = dim3(256);
  const unsigned gx = (cols + RUN - 1) / RUN;
  s.grid = dim3(gx, row_ctas(rows, 8, gx, 8));
  return s;
}

template <typename T, typename TR, typename TW, bool BWD>
int launch_types(const DropArgs& a, Path path, int* parts, cudaStream_t st) {
  constexpr int VEC = sizeof(T) == 2 ? 8 : 4;
  if (path == FLAT) {
    const long long m = flat_runs(a.rows, a.cols, VEC, BWD && a.part ? FLAT_SUM_CTAS : FLAT_CTAS);
    const int threads = (int)(m * a.cols);
    const unsigned grid = (threads + 255) / 256;
    if (BWD && a.part)
      dropout_add_flat_kernel<T, TR, TW, BWD, BWD><<<grid, 256, 0, st>>>(a, threads);
    else
      dropout_add_flat_kernel<T, TR, TW, BWD, false><<<grid, 256, 0, st>>>(a, threads);
    *parts = flat_joins(a.cols, VEC) ? (int)grid : (int)(m * VEC);
  } else if (path == VECTOR) {
    const Shape s = vec_shape(a.rows, a.cols, VEC);
    if (BWD && a.part)
      dropout_add_vec_kernel<T, TR, TW, VEC, BWD, BWD>
          <<<s.grid, s.block, sizeof(float) * s.block.x * s.block.y * VEC, st>>>(a);
    else
      dropout_add_vec_kernel<T, TR, TW, VEC, BWD, false><<<s.grid, s.block, 0, st>>>(a);
    *parts = s.grid.y;
  } else {
    const Shape s = any_shape(a.rows, a.cols);
    dropout_add_any_kernel<T, TR, TW, BWD><<<s.grid, s.block, 0, st>>>(a);
    *parts = s.grid.y;
  }
  UB_CHECK_LAUNCH();
  return 0;
}

template <typename T, bool BWD>
int launch_streams(const DropArgs& a, int r_dtype, int w_dtype, Path path, int* parts, cudaStream_t st) {
  if (r_dtype == UNBLEND_F32) {
    if (w_dtype == UNBLEND_F32) return launch_types<T, float, float, BWD>(a, path, parts, st);
    return launch_types<T, float, T, BWD>(a, path, parts, st);
  }
  if (w_dtype == UNBLEND_F32) return launch_types<T, T, float, BWD>(a, path, parts, st);
  return launch_types<T, T, T, BWD>(a, path, parts, st);
}

template <bool BWD>
int launch(const DropArgs& a, int dtype, int r_dtype, int w_dtype, Path path, int* parts, cudaStream_t st) {
  if (dtype == UNBLEND_F32) return launch_types<float, float, float, BWD>(a, path, parts, st);
  if (dtype == UNBLEND_BF16) return launch_streams<__nv_bfloat16, BWD>(a, r_dtype, w_dtype, path, parts, st);
  return launch_streams<__half, BWD>(a, r_dtype, w_dtype, path, parts, st);
}

constexpr int FLAT_COLS = 1 << 22;

// One run of values. Very wide rows are left to the other kernels: each of the VEC rows of partial sums is as wide.
bool contiguous(const RowMap& m, long long outer, int cols) {
  return (m.inner <= 1 || m.si == cols) && (outer <= 1 || m.so == (long long)m.inner * cols) && cols <= FLAT_COLS;
}

void set_p(DropArgs* a, double p) {
  const double t = std::nearbyint(p * 4294967296.0);
  a->drop_all = t >= 4294967296.0;
  a->threshold = a->drop_all ? 0xFFFFFFFFu : (uint32_t)t;
  a->inv_keep = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f;
}

}  // namespace

extern "C" int unblend_dropout_add_grad_workspace(long long rows, int cols, long long* bytes) {
  UB_REQUIRE(bytes && rows_ok(1, rows, cols));
  // The largest of the layouts (which of them runs depends on the pointers' alignment).
  unsigned parts = any_shape(rows, cols).grid.y;
  for (int vec = 4; vec <= 8; vec += 4)
    if (cols % vec == 0) {
      const unsigned v = vec_shape(rows, cols, vec).grid.y;
      parts = v > parts ? v : parts;
    }
  for (int vec = 4; vec <= 8 && cols <= FLAT_COLS; vec += 4) {
    const long long m = flat_runs(rows, cols, vec, FLAT_SUM_CTAS);
    const long long v = flat_joins(cols, vec) ? (m * cols + 255) / 256 : m * vec;
    parts = v > parts ? (unsigned)v : parts;
  }
  *bytes = (long long)parts * cols * (long long)sizeof(float);
  return 0;
}

extern "C" int unblend_dropout_add_forward(const void* x, long long x_so, long long x_si, const void* residual,
                                           long long r_so, long long r_si, const void* scale, void* y, double p,
                                           const void* rng, long long outer, long long inner, int cols, int dtype,
                                           int r_dtype, int w_dtype, void* stream) {
  UB_REQUIRE(x && y && rng && rows_ok(outer, inner, cols) && p >= 0.0 && p <= 1.0);
  UB_REQUIRE(known_type(dtype) && (r_dtype == UNBLEND_F32 || r_dtype == dtype) &&
             (w_dtype == UNBLEND_F32 || w_dtype == dtype));
  UB_REQUIRE(reinterpret_cast<uintptr_t>(rng) % 8 == 0);
  DropArgs a{};
  a.x = x;
  a.r = residual;
  a.scale = scale;
  a.out = y;
  a.rng = static_cast<const unsigned long long*>(rng);
  a.xm = row_map(x_so, x_si, inner);
  a.rm = row_map(r_so, r_si, inner);
  a.rows = (unsigned)(outer * inner);
  a.cols = cols;
  set_p(&a, p);
  const int vec_n = dtype == UNBLEND_F32 ? 4 : 8;
  const bool vec = cols % vec_n == 0 && rows_aligned(x, a.xm, outer, elem_size(dtype), 16) && aligned16(y) &&
                   aligned16(scale) && (!residual || rows_aligned(residual, a.rm, outer, elem_size(r_dtype), 16));
  const bool flat = aligned16(x) && aligned16(y) && contiguous(a.xm, outer, cols) &&
                    (!residual || (aligned16(residual) && contiguous(a.rm, outer, cols)));
  const Path path = flat ? FLAT : vec ? VECTOR : ANY;
  int parts = 0;
  return launch<false>(a, dtype, r_dtype, w_dtype, path, &parts, ub::as_stream(stream));
}

extern "C" int unblend_dropout_add_backward(const void* dy, long long dy_so, long long dy_si, const void* x,
                                            long long x_so, long long x_si, const void* scale, void* dx, void* dscale,
                                            float* work, double p, const void* rng, long long outer, long long inner,
                                            int cols, int dtype, int dy_dtype, int w_dtype, void* stream) {
  UB_REQUIRE(dy && dx && rng && rows_ok(outer, inner, cols) && p >= 0.0 && p <= 1.0);
  UB_REQUIRE(known_type(dtype) && (dy_dtype == UNBLEND_F32 || dy_dtype == dtype) &&
             (w_dtype == UNBLEND_F32 || w_dtype == dtype));
  UB_REQUIRE(reinterpret_cast<uintptr_t>(rng) % 8 == 0);
  UB_REQUIRE(dscale == nullptr || (scale && x && work));
  DropArgs a{};
  a.x = x;
  a.r = dy;
  a.scale = scale;
  a.out = dx;
  a.part = dscale ? work : nullptr;
  a.rng = static_cast<const unsigned long long*>(rng);
  a.xm = row_map(x_so, x_si, inner);
  a.rm = row_map(dy_so, dy_si, inner);
  a.rows = (unsigned)(outer * inner);
  a.cols = cols;
  set_p(&a, p);
  const int vec_n = dtype == UNBLEND_F32 ? 4 : 8;
  const bool vec = cols % vec_n == 0 && (!dscale || rows_aligned(x, a.xm, outer, elem_size(dtype), 16)) &&
                   aligned16(dx) && aligned16(scale) && rows_aligned(dy, a.rm, outer, elem_size(dy_dtype), 16);
  const bool flat = aligned16(dy) && aligned16(dx) && contiguous(a.rm, outer, cols) &&
                    (!dscale || (aligned16(x) && contiguous(a.xm, outer, cols)));
  const Path path = flat ? FLAT : vec ? VECTOR : ANY;
  cudaStream_t st = ub::as_stream(stream);
  int parts = 0;
  const int rc = launch<true>(a, dtype, dy_dtype, w_dtype, path, &parts, st);
  if (rc || !dscale) return rc;
  if (w_dtype == UNBLEND_F32) return launch_column_sums<float>(work, parts, cols, 1, dscale, nullptr, st);
  if (w_dtype == UNBLEND_BF16) return launch_column_sums<__nv_bfloat16>(work, parts, cols, 1, dscale, nullptr, st);
  return launch_column_sums<__half>(work, parts, cols, 1, dscale, nullptr, st);
}
