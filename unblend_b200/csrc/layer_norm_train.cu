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
// are read again for every reduction. Rows come through shared memory, several in flight per warp (cp.async). The weights' gradients are summed in registers over the rows that a warp (or
// CTA) walks, joined across the CTA in shared memory, and the CTAs' partial rows added in a fixed order by a second
// kernel: the result is the same on every run.
#include "train_common.cuh"

namespace {

using namespace ub::train;

constexpr int WARP_COLS = 1024;   // widest row of the warp-per-row kernels
constexpr int CTA_COLS = 8192;    // widest row held in a CTA's registers
constexpr int MAX_PARTS = 2 * ub::kNumSMs;
constexpr int ONE_CTA_ROWS = 64;  // backward calls of up to so many rows run in one CTA, without partial sums

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
  int stages;      // rows in flight per warp (or CTA)
  int slot_bytes;  // one row in shared memory, padded
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

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_wait(int pending) {  // all but the newest `pending` (1 to 3) groups are there
  if (pending >= 3)
    asm volatile("cp.async.wait_group 3;" ::: "memory");
  else if (pending == 2)
    asm volatile("cp.async.wait_group 2;" ::: "memory");
  else
    asm volatile("cp.async.wait_group 1;" ::: "memory");
}

// The rows of one warp or CTA on their way from global to shared memory, `stages` deep. VEC > 1: every row starts on a
// 16-byte boundary, and a thread copies exactly the 16-byte chunks that it reads back, so no barrier is needed. VEC
// == 1: rows start anywhere. The whole 16-byte chunks inside a row are copied as such, the elements before and behind
// them one by one, and the row keeps its offset to the boundary in shared memory; a barrier lets the others read it.
template <typename T, int VEC, int NV, bool WARP>
struct RowRing {
  uint8_t* base;
  int t, tpr;

  __device__ __forceinline__ uint8_t* slot(const NormArgs& a, int i) const { return base + i * a.slot_bytes; }

  __device__ __forceinline__ void fetch(const NormArgs& a, int i, const T* row) const {
    uint8_t* s = slot(a, i);
    if constexpr (VEC > 1) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * tpr + t) * VEC;
        if (c < a.cols) cp_async16(s + c * sizeof(T), row + c);
      }
    } else {
      constexpr int E = 16 / (int)sizeof(T);
      const int mis = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));  // elements past the boundary
      const int head = min(a.cols, mis ? E - mis : 0);
      const int chunks = (a.cols - head) / E;
      const int tail = head + chunks * E;
      T* d = reinterpret_cast<T*>(s) + mis;
      for (int k = t; k < chunks; k += tpr) cp_async16(d + head + k * E, row + head + k * E);
      if (t < head) d[t] = row[t];
      if (t < a.cols - tail) d[tail + t] = row[tail + t];
    }
  }

  // Column values k of this thread: columns (k * tpr + t) * VEC ...
  __device__ __forceinline__ void read(const NormArgs& a, int i, int mis, int k, float (&v)[VEC]) const {
    load_vec<T, VEC>(reinterpret_cast<const T*>(slot(a, i)) + (VEC > 1 ? 0 : mis) + (k * tpr + t) * VEC, v);
  }
};

template <bool WARP>
__device__ __forceinline__ void row_sync() {
  if constexpr (WARP)
    __syncwarp();
  else
    __syncthreads();
}

template <typename T>
__device__ __forceinline__ int misalign(const T* p) {
  return (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
}

// A row from shared memory (at its own offset to the 16-byte boundary) to global memory, by whole chunks.
template <typename T>
__device__ __forceinline__ void store_row(T* row, const T* s, int cols, int t, int tpr) {
  constexpr int E = 16 / (int)sizeof(T);
  const int mis = misalign(row);
  const int head = min(cols, mis ? E - mis : 0);
  const int chunks = (cols - head) / E, tail = head + chunks * E;
  for (int k = t; k < chunks; k += tpr)
    *reinterpret_cast<uint4*>(row + head + k * E) = *reinterpret_cast<const uint4*>(s + mis + head + k * E);
  if (t < head) row[t] = s[mis + t];
  if (t < cols - tail) row[tail + t] = s[mis + tail + t];
}

template <typename T, typename TW, int VEC, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 512)
    layer_norm_fwd_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[2][64];
  extern __shared__ __align__(16) uint8_t rows_smem[];
  int phase = 0;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int tpr = WARP ? 32 : blockDim.x;
  const int groups = WARP ? blockDim.x >> 5 : 1, group = WARP ? threadIdx.x >> 5 : 0;
  const float inv_c = 1.f / (float)a.cols;
  const long long step = (long long)gridDim.x * groups, row0 = (long long)blockIdx.x * groups + group;
  const int slots = a.stages + (VEC > 1 ? 0 : 1);  // one more to gather an unaligned output row
  const RowRing<T, VEC, NV, WARP> ring{rows_smem + (size_t)group * slots * a.slot_bytes, t, tpr};
  const T* xb = static_cast<const T*>(a.x);
  for (int s = 0; s < a.stages - 1; ++s) {
    const long long row = row0 + s * step;
    if (row < a.rows) ring.fetch(a, s, xb + row_offset(a.xm, (unsigned)row));
    cp_commit();
  }
  int cur = 0, next = a.stages - 1;
  for (long long row = row0; row < a.rows; row += step) {
    const long long ahead = row + (a.stages - 1) * step;
    if (ahead < a.rows) ring.fetch(a, next, xb + row_offset(a.xm, (unsigned)ahead));
    cp_commit();
    cp_wait(a.stages - 1);
    const int mis = misalign(xb + row_offset(a.xm, (unsigned)row));
    if constexpr (VEC == 1) row_sync<WARP>();
    float v[NV][VEC];
    float s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * tpr + t) * VEC;
      if (c < a.cols) {
        ring.read(a, cur, mis, k, v[k]);
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
    T* out = VEC > 1 ? y : reinterpret_cast<T*>(ring.slot(a, a.stages)) + misalign(y);
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
        store_vec<T, VEC>(out + c, o);
      }
    }
    if constexpr (VEC == 1) {
      row_sync<WARP>();
      store_row(y, reinterpret_cast<const T*>(ring.slot(a, a.stages)), a.cols, t, tpr);
    }
    if (t == 0) reinterpret_cast<float2*>(a.stats)[row] = make_float2(mean, rstd);
    cur = cur + 1 == a.stages ? 0 : cur + 1;
    next = next + 1 == a.stages ? 0 : next + 1;
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

// A row's x and dy stay in shared memory between its two passes (sums, then dx), so that registers hold the sums of
// the weights' gradients and two CTAs fit an SM.
template <typename T, typename TW, int VEC, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 512, WARP ? 2 : 1)
    layer_norm_bwd_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[2][64];
  extern __shared__ __align__(16) uint8_t rows_smem[];
  int phase = 0;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int tpr = WARP ? 32 : blockDim.x;
  const int groups = WARP ? blockDim.x >> 5 : 1, group = WARP ? threadIdx.x >> 5 : 0;
  const float inv_c = 1.f / (float)a.cols;
  const long long step = (long long)gridDim.x * groups, row0 = (long long)blockIdx.x * groups + group;
  const int slots = 2 * a.stages + (VEC > 1 ? 0 : 1);
  const RowRing<T, VEC, NV, WARP> ring{rows_smem + (size_t)group * slots * a.slot_bytes, t, tpr};
  const T *xb = static_cast<const T*>(a.x), *db_ = static_cast<const T*>(a.dy);
  float dg[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i) dg[k][i] = db[k][i] = 0.f;
  for (int s = 0; s < a.stages - 1; ++s) {
    const long long row = row0 + s * step;
    if (row < a.rows) {
      ring.fetch(a, 2 * s, xb + row_offset(a.xm, (unsigned)row));
      ring.fetch(a, 2 * s + 1, db_ + row_offset(a.dym, (unsigned)row));
    }
    cp_commit();
  }
  int cur = 0, next = a.stages - 1;
  float2 st_next = row0 < a.rows ? reinterpret_cast<const float2*>(a.stats)[row0] : make_float2(0.f, 0.f);
  for (long long row = row0; row < a.rows; row += step) {
    const long long ahead = row + (a.stages - 1) * step;
    const float2 st = st_next;
    if (row + step < a.rows) st_next = reinterpret_cast<const float2*>(a.stats)[row + step];
    if (ahead < a.rows) {
      ring.fetch(a, 2 * next, xb + row_offset(a.xm, (unsigned)ahead));
      ring.fetch(a, 2 * next + 1, db_ + row_offset(a.dym, (unsigned)ahead));
    }
    cp_commit();
    cp_wait(a.stages - 1);
    int mx = 0, md = 0;
    if constexpr (VEC == 1) {
      mx = misalign(xb + row_offset(a.xm, (unsigned)row));
      md = misalign(db_ + row_offset(a.dym, (unsigned)row));
      row_sync<WARP>();
    }
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * tpr + t) * VEC;
      if (c < a.cols) {
        float g[VEC], x[VEC], d[VEC];
        ring.read(a, 2 * cur, mx, k, x);
        ring.read(a, 2 * cur + 1, md, k, d);
        if (a.gamma) load_vec<TW, VEC>(static_cast<const TW*>(a.gamma) + c, g);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float xh = (x[i] - st.x) * st.y;
          dg[k][i] = fmaf(d[i], xh, dg[k][i]);
          db[k][i] += d[i];
          const float gy = a.gamma ? d[i] * g[i] : d[i];
          s[0] += gy;
          s[1] = fmaf(gy, xh, s[1]);
        }
      }
    }
    row_sum<WARP, 2>(s, red, phase);
    const float m0 = s[0] * inv_c, m1 = s[1] * inv_c;
    T* dx = static_cast<T*>(a.y) + row * a.cols;
    T* out = VEC > 1 ? dx : reinterpret_cast<T*>(ring.slot(a, 2 * a.stages)) + misalign(dx);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * tpr + t) * VEC;
      if (c < a.cols) {
        float g[VEC], x[VEC], d[VEC], o[VEC];
        ring.read(a, 2 * cur, mx, k, x);
        ring.read(a, 2 * cur + 1, md, k, d);
        if (a.gamma) load_vec<TW, VEC>(static_cast<const TW*>(a.gamma) + c, g);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float gy = a.gamma ? d[i] * g[i] : d[i];
          o[i] = st.y * (gy - m0 - (x[i] - st.x) * st.y * m1);
        }
        store_vec<T, VEC>(out + c, o);
      }
    }
    if constexpr (VEC == 1) {
      row_sync<WARP>();
      store_row(dx, reinterpret_cast<const T*>(ring.slot(a, 2 * a.stages)), a.cols, t, tpr);
    }
    cur = cur + 1 == a.stages ? 0 : cur + 1;
    next = next + 1 == a.stages ? 0 : next + 1;
  }
  if (a.dgamma == nullptr) return;
  auto put = [&](int c, float g, float b) {
    if (a.part) {
      float* part = a.part + (long long)blockIdx.x * 2 * a.cols;
      part[c] = g;
      part[a.cols + c] = b;
    } else {
      static_cast<TW*>(a.dgamma)[c] = from_f<TW>(g);
      static_cast<TW*>(a.dbeta)[c] = from_f<TW>(b);
    }
  };
  if constexpr (WARP) {
    // Warps leave their sums behind one another in shared memory; the threads add them by column, in warp order.
    asm volatile("cp.async.wait_all;" ::: "memory");
    float* sums = reinterpret_cast<float*>(rows_smem);  // [groups][cols]
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * 32 + t) * VEC;
        if (c < a.cols) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) sums[group * a.cols + c + i] = which ? db[k][i] : dg[k][i];
        }
      }
      __syncthreads();
      for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
        float v = 0.f;
        for (int w = 0; w < groups; ++w) v += sums[w * a.cols + c];
        if (a.part)
          a.part[((long long)blockIdx.x * 2 + which) * a.cols + c] = v;
        else
          static_cast<TW*>(which ? a.dbeta : a.dgamma)[c] = from_f<TW>(v);
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * tpr + t) * VEC;
      if (c < a.cols) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) put(c + i, dg[k][i], db[k][i]);
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

// CTAs of the backward kernel, each of which leaves one partial row of the weights' gradients; 1: none are needed.
int bwd_parts(long long rows, int cols) {
  if (cols <= WARP_COLS && rows <= ONE_CTA_ROWS) return 1;
  const long long units = cols <= WARP_COLS ? (rows + 7) / 8 : rows;
  return (int)(units < MAX_PARTS ? units : MAX_PARTS);
}

template <typename T, typename TW, int VEC, int NV, bool WARP>
int launch_one(NormArgs a, bool backward, cudaStream_t st) {
  const int threads = WARP ? 256 : ((a.cols + VEC * NV - 1) / (VEC * NV) + 31) / 32 * 32;
  const int groups = WARP ? 8 : 1;
  // Rows in flight: 4, fewer where two CTAs (three of the smaller wide-row ones) would not fit the shared memory.
  a.slot_bytes = (a.cols * (int)sizeof(T) + 15) / 16 * 16 + (VEC > 1 ? 0 : 16);
  const int per_stage = (backward ? 2 : 1) * groups * a.slot_bytes;
  const int extra = VEC > 1 ? 0 : groups * a.slot_bytes;
  a.stages = 4;
  while (a.stages > 2 && a.stages * per_stage + extra > 100 * 1024) --a.stages;
  int smem = a.stages * per_stage + extra;
  if (backward) {
    if (WARP && smem < (int)sizeof(float) * groups * a.cols) smem = sizeof(float) * groups * a.cols;
    auto kern = layer_norm_bwd_kernel<T, TW, VEC, NV, WARP>;
    if (smem > 40 * 1024) cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    kern<<<bwd_parts(a.rows, a.cols), threads, smem, st>>>(a);
  } else {
    auto kern = layer_norm_fwd_kernel<T, TW, VEC, NV, WARP>;
    if (smem > 40 * 1024) cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    const long long cap = ub::kNumSMs * (smem > 56 * 1024 ? 2LL : 4LL);
    kern<<<WARP ? ub::grid_1d(a.rows, 8, cap) : ub::grid_1d(a.rows, 1, cap), threads, smem, st>>>(a);
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
    if (a.dgamma) {
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

// A wide row's sums always take the second kernel.
bool joins(long long rows, int cols) { return cols > CTA_COLS || bwd_parts(rows, cols) > 1; }

bool types_ok(int dtype, int w_dtype) {
  return known_type(dtype) && (w_dtype == UNBLEND_F32 || w_dtype == dtype);
}

}  // namespace

extern "C" int unblend_layer_norm_grad_workspace(long long rows, int cols, long long* bytes) {
  UB_REQUIRE(bytes && rows_ok(1, rows, cols));
  *bytes = joins(rows, cols) ? (long long)bwd_parts(rows, cols) * 2 * cols * (long long)sizeof(float) : 0;
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
                   rows_aligned(dy, a.dym, outer, es, 16) && aligned16(dx) &&
                   aligned16(gamma);
  cudaStream_t st = ub::as_stream(stream);
  const int rc = launch(a, dtype, w_dtype, vec, true, st);
  if (rc || !a.part) return rc;
  const int parts = bwd_parts(a.rows, cols);
  if (w_dtype == UNBLEND_F32) return launch_column_sums<float>(work, parts, cols, 2, dgamma, dbeta, st);
  if (w_dtype == UNBLEND_BF16) return launch_column_sums<__nv_bfloat16>(work, parts, cols, 2, dgamma, dbeta, st);
  return launch_column_sums<__half>(work, parts, cols, 2, dgamma, dbeta, st);
}
