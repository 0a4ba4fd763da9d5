// LayerNorm with gradients: forward that leaves each row's (mean, rstd), backward for the input and the weights.
//
//   y = xhat * gamma + beta,  xhat = (x - mean) * rstd,  rstd = 1 / sqrt(var + eps)
//   gy = dy * gamma
//   dx = rstd * (gy - mean(gy) - xhat * mean(gy * xhat))
//   dgamma = sum_rows dy * xhat,  dbeta = sum_rows dy
//
// Statistics, sums and all arithmetic are fp32; x, y, dy and dx are fp32, bf16 or fp16.
// Both directions are bound by HBM: one read of each input and one write of each output, a row held in registers
// between its reductions.
//
// Rows of up to 1024 columns are handled by one warp each (no barrier), wider ones up to 8192 by one CTA; wider rows
// are read again for every reduction. The weights' gradients are summed in registers over the rows that a warp (or
// CTA) walks, joined across the CTA in shared memory, and the CTAs' partial rows added in a fixed order by a second
// kernel: the result is the same on every run.
#include "train_common.cuh"

namespace {

using namespace ub::train;

constexpr int WARP_COLS = 1024;   // widest row of the warp-per-row kernels
constexpr int CTA_COLS = 8192;    // widest row held in a CTA's registers
constexpr int MAX_PARTS = 2 * ub::kNumSMs;

struct NormArgs {
  const void* x;
  const void* dy;
  const void* gamma;
  const void* beta;
  void* y;       // forward output, or dx
  float* stats;  // [rows][2]
  float* part;   // [gridDim.x][2][cols]
  RowMap xm, dym;
  unsigned rows;
  int cols;
  float eps;
};

// Sum of N values over the threads of one row. CTA rows alternate between two shared arrays: an array is written
// again only after the barrier of the reduction in between, which every reader of it has passed.
template <bool WARP, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*red)[32 * 2], int& phase) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = ub::warp_sum(v[i]);
  if constexpr (!WARP) {
    float* r = red[phase];
    phase ^= 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) r[warp * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = ub::warp_sum(lane < warps ? r[lane * N + i] : 0.f);
  }
}

template <typename T, typename TW, int VEC, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 512)
    layer_norm_fwd_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[2][64];
  int phase = 0;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int tpr = WARP ? 32 : blockDim.x;
  const int groups = WARP ? blockDim.x >> 5 : 1, group = WARP ? threadIdx.x >> 5 : 0;
  const float inv_c = 1.f / (float)a.cols;
  for (long long row = (long long)blockIdx.x * groups + group; row < a.rows; row += (long long)gridDim.x * groups) {
    const T* x = static_cast<const T*>(a.x) + row_offset(a.xm, (unsigned)row);
    float v[NV][VEC];
    float s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * tpr + t) * VEC;
      if (c < a.cols) {
        load_vec<T, VEC>(x + c, v[k]);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[k][i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) s[0] += v[k][i];
    }
    row_sum<WARP, 1>(s, red, phase);
    const float mean = s[0] * inv_c;
    float q[1] = {0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * tpr + t) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float d = c < a.cols ? v[k][i] - mean : 0.f;
        q[0] = fmaf(d, d, q[0]);
      }
    }
    row_sum<WARP, 1>(q, red, phase);
    const float rstd = 1.f / sqrtf(q[0] * inv_c + a.eps);
    T* y = static_cast<T*>(a.y) + row * a.cols;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * tpr + t) * VEC;
      if (c < a.cols) {
        float g[VEC], b[VEC], o[VEC];
        if (a.gamma) load_vec<TW, VEC>(static_cast<const TW*>(a.gamma) + c, g);
        if (a.beta) load_vec<TW, VEC>(static_cast<const TW*>(a.beta) + c, b);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float xhat = (v[k][i] - mean) * rstd;
          o[i] = fmaf(xhat, a.gamma ? g[i] : 1.f, a.beta ? b[i] : 0.f);
        }
        store_vec<T, VEC>(y + c, o);
      }
    }
    if (t == 0) reinterpret_cast<float2*>(a.stats)[row] = make_float2(mean, rstd);
  }
}

// Rows wider than the registers of a CTA: three passes over the row (the second and third hit L2).
template <typename T, typename TW>
__global__ void __launch_bounds__(1024) layer_norm_fwd_wide_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[2][64];
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

template <typename T, typename TW, int VEC, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 512)
    layer_norm_bwd_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[2][64];
  extern __shared__ float cols_sum[];  // [2][cols], warp-per-row kernels
  int phase = 0;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int tpr = WARP ? 32 : blockDim.x;
  const int groups = WARP ? blockDim.x >> 5 : 1, group = WARP ? threadIdx.x >> 5 : 0;
  const float inv_c = 1.f / (float)a.cols;
  float dg[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i) dg[k][i] = db[k][i] = 0.f;
  for (long long row = (long long)blockIdx.x * groups + group; row < a.rows; row += (long long)gridDim.x * groups) {
    const T* x = static_cast<const T*>(a.x) + row_offset(a.xm, (unsigned)row);
    const T* dy = static_cast<const T*>(a.dy) + row_offset(a.dym, (unsigned)row);
    const float2 st = reinterpret_cast<const float2*>(a.stats)[row];
    float xh[NV][VEC], gy[NV][VEC];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * tpr + t) * VEC;
      if (c < a.cols) {
        load_vec<T, VEC>(x + c, xh[k]);
        load_vec<T, VEC>(dy + c, gy[k]);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) xh[k][i] = st.x, gy[k][i] = 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * tpr + t) * VEC;
      float g[VEC];
      if (a.gamma && c < a.cols) load_vec<TW, VEC>(static_cast<const TW*>(a.gamma) + c, g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        xh[k][i] = (xh[k][i] - st.x) * st.y;
        dg[k][i] = fmaf(gy[k][i], xh[k][i], dg[k][i]);
        db[k][i] += gy[k][i];
        if (a.gamma && c < a.cols) gy[k][i] *= g[i];
        s[0] += gy[k][i];
        s[1] = fmaf(gy[k][i], xh[k][i], s[1]);
      }
    }
    row_sum<WARP, 2>(s, red, phase);
    const float m0 = s[0] * inv_c, m1 = s[1] * inv_c;
    T* dx = static_cast<T*>(a.y) + row * a.cols;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * tpr + t) * VEC;
      if (c < a.cols) {
        float o[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = st.y * (gy[k][i] - m0 - xh[k][i] * m1);
        store_vec<T, VEC>(dx + c, o);
      }
    }
  }
  if (a.part == nullptr) return;
  float* part = a.part + (long long)blockIdx.x * 2 * a.cols;
  if constexpr (WARP) {
    for (int w = 0; w < groups; ++w) {
      if (w == group) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int c = (k * 32 + t) * VEC;
          if (c < a.cols) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              cols_sum[c + i] = (w ? cols_sum[c + i] : 0.f) + dg[k][i];
              cols_sum[a.cols + c + i] = (w ? cols_sum[a.cols + c + i] : 0.f) + db[k][i];
            }
          }
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < 2 * a.cols; c += blockDim.x) part[c] = cols_sum[c];
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * tpr + t) * VEC;
      if (c < a.cols) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          part[c + i] = dg[k][i];
          part[a.cols + c + i] = db[k][i];
        }
      }
    }
  }
}

// Input gradient of rows wider than the registers of a CTA: two passes over the row.
template <typename T, typename TW>
__global__ void __launch_bounds__(1024) layer_norm_dx_wide_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[2][64];
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

// CTAs of the backward kernel, each of which leaves one partial row of the weights' gradients.
int bwd_parts(long long rows, int cols) {
  const long long units = cols <= WARP_COLS ? (rows + 7) / 8 : rows;
  return (int)(units < MAX_PARTS ? units : MAX_PARTS);
}

template <typename T, typename TW, int VEC, int NV, bool WARP>
int launch_one(const NormArgs& a, bool backward, cudaStream_t st) {
  const int threads = WARP ? 256 : ((a.cols + VEC * NV - 1) / (VEC * NV) + 31) / 32 * 32;
  if (backward) {
    const int grid = bwd_parts(a.rows, a.cols);
    const size_t smem = WARP ? 2 * sizeof(float) * a.cols : 0;
    layer_norm_bwd_kernel<T, TW, VEC, NV, WARP><<<grid, threads, smem, st>>>(a);
  } else {
    const unsigned grid = WARP ? ub::grid_1d(a.rows, 8) : ub::grid_1d(a.rows, 1);
    layer_norm_fwd_kernel<T, TW, VEC, NV, WARP><<<grid, threads, 0, st>>>(a);
  }
  UB_CHECK_LAUNCH();
  return 0;
}

template <typename T, typename TW, int VEC>
int launch_vec(const NormArgs& a, bool backward, cudaStream_t st) {
  if (a.cols <= 256) return launch_one<T, TW, VEC, 8 / VEC, true>(a, backward, st);
  if (a.cols <= 512) return launch_one<T, TW, VEC, 16 / VEC, true>(a, backward, st);
  if (a.cols <= WARP_COLS) return launch_one<T, TW, VEC, 32 / VEC, true>(a, backward, st);
  return launch_one<T, TW, VEC, 16 / VEC, false>(a, backward, st);
}

template <typename T, typename TW>
int launch_types(const NormArgs& a, bool vec, bool backward, cudaStream_t st) {
  if (a.cols > CTA_COLS) {
    const unsigned grid = ub::grid_1d(a.rows, 1, 4LL * ub::kNumSMs);
    if (!backward) {
      layer_norm_fwd_wide_kernel<T, TW><<<grid, 1024, 0, st>>>(a);
      UB_CHECK_LAUNCH();
      return 0;
    }
    layer_norm_dx_wide_kernel<T, TW><<<grid, 1024, 0, st>>>(a);
    UB_CHECK_LAUNCH();
    if (a.part) {
      const dim3 g((a.cols + 255) / 256, bwd_parts(a.rows, a.cols));
      layer_norm_dw_wide_kernel<T><<<g, 256, 0, st>>>(a);
      UB_CHECK_LAUNCH();
    }
    return 0;
  }
  if (vec) return launch_vec<T, TW, 16 / (int)sizeof(T)>(a, backward, st);
  return launch_vec<T, TW, 1>(a, backward, st);
}

int launch(const NormArgs& a, int dtype, int w_dtype, bool vec, bool backward, cudaStream_t st) {
  if (dtype == UNBLEND_F32) return launch_types<float, float>(a, vec, backward, st);
  if (dtype == UNBLEND_BF16)
    return w_dtype == UNBLEND_F32 ? launch_types<__nv_bfloat16, float>(a, vec, backward, st)
                                  : launch_types<__nv_bfloat16, __nv_bfloat16>(a, vec, backward, st);
  return w_dtype == UNBLEND_F32 ? launch_types<__half, float>(a, vec, backward, st)
                                : launch_types<__half, __half>(a, vec, backward, st);
}

bool types_ok(int dtype, int w_dtype) {
  return known_type(dtype) && (w_dtype == UNBLEND_F32 || w_dtype == dtype);
}

}  // namespace

extern "C" int unblend_layer_norm_grad_workspace(long long rows, int cols, long long* bytes) {
  UB_REQUIRE(bytes && rows_ok(1, rows, cols));
  *bytes = (long long)bwd_parts(rows, cols) * 2 * cols * (long long)sizeof(float);
  return 0;
}

extern "C" int unblend_layer_norm_forward(const void* x, long long x_so, long long x_si, void* y, float* stats,
                                          const void* gamma, const void* beta, float eps, long long outer,
                                          long long inner, int cols, int dtype, int w_dtype, void* stream) {
  UB_REQUIRE(x && y && stats && rows_ok(outer, inner, cols) && types_ok(dtype, w_dtype) && eps >= 0.f);
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
  const bool vec = cols % (16 / es) == 0 && rows_aligned(x, a.xm, outer, es, 16) &&
                   aligned16(y) && aligned16(gamma) &&
                   aligned16(beta);
  return launch(a, dtype, w_dtype, vec, false, ub::as_stream(stream));
}

extern "C" int unblend_layer_norm_backward(const void* dy, long long dy_so, long long dy_si, const void* x,
                                           long long x_so, long long x_si, const float* stats, const void* gamma,
                                           void* dx, void* dgamma, void* dbeta, float* work, long long outer,
                                           long long inner, int cols, int dtype, int w_dtype, void* stream) {
  UB_REQUIRE(dy && x && stats && dx && rows_ok(outer, inner, cols) && types_ok(dtype, w_dtype));
  UB_REQUIRE((dgamma != nullptr) == (dbeta != nullptr) && (dgamma == nullptr || work != nullptr));
  NormArgs a{};
  a.x = x;
  a.dy = dy;
  a.y = dx;
  a.stats = const_cast<float*>(stats);
  a.gamma = gamma;
  a.part = dgamma ? work : nullptr;
  a.xm = row_map(x_so, x_si, inner);
  a.dym = row_map(dy_so, dy_si, inner);
  a.rows = (unsigned)(outer * inner);
  a.cols = cols;
  const int es = elem_size(dtype);
  const bool vec = cols % (16 / es) == 0 && rows_aligned(x, a.xm, outer, es, 16) &&
                   rows_aligned(dy, a.dym, outer, es, 16) && aligned16(dx) &&
                   aligned16(gamma);
  cudaStream_t st = ub::as_stream(stream);
  const int rc = launch(a, dtype, w_dtype, vec, true, st);
  if (rc || !dgamma) return rc;
  const int parts = bwd_parts(a.rows, cols);
  if (w_dtype == UNBLEND_F32) return launch_column_sums<float>(work, parts, cols, 2, dgamma, dbeta, st);
  if (w_dtype == UNBLEND_BF16) return launch_column_sums<__nv_bfloat16>(work, parts, cols, 2, dgamma, dbeta, st);
  return launch_column_sums<__half>(work, parts, cols, 2, dgamma, dbeta, st);
}
