// Shared helpers of the training operators (layer norm, dropout-add, attention with gradients): element types,
// vector loads into fp32 registers, two-level row addressing and the fixed-order join of column sums.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "common.cuh"

namespace ub {
namespace train {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f<__half>(float v) {
  return __float2half_rn(v);
}

// Two fp32 sums or products in one instruction, each rounded once.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(r)
      : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
  return *reinterpret_cast<float2*>(&r);
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(r)
      : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
  return *reinterpret_cast<float2*>(&r);
}

// The elements of a 16-byte chunk as fp32 pairs, and back.
__device__ __forceinline__ void unpack16(const uint4& w, float2 (&v)[2], float) {
  v[0] = make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
  v[1] = make_float2(__uint_as_float(w.z), __uint_as_float(w.w));
}
__device__ __forceinline__ void unpack16(const uint4& w, float2 (&v)[4], __nv_bfloat16) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xFFFF0000u));
}
__device__ __forceinline__ void unpack16(const uint4& w, float2 (&v)[4], __half) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
}
__device__ __forceinline__ uint4 pack16(const float2 (&v)[2], float) {
  return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x),
                    __float_as_uint(v[1].y));
}
__device__ __forceinline__ uint4 pack16(const float2 (&v)[4], __nv_bfloat16) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(v[i].x, v[i].y);
    u[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ uint4 pack16(const float2 (&v)[4], __half) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 b = __floats2half2_rn(v[i].x, v[i].y);
    u[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// VEC consecutive elements as fp32. VEC * sizeof(T) is the access width (2, 4, 8, 16 or 32 bytes; p is aligned to
// it, 32 bytes as two 16-byte halves).
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[VEC]) {
  constexpr int BYTES = VEC * (int)sizeof(T);
  if constexpr (VEC == 1) {
    v[0] = to_f(*p);
  } else {
    alignas(16) T raw[VEC];
    if constexpr (BYTES == 8)
      *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(p);
    else {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i)
        reinterpret_cast<uint4*>(raw)[i] = reinterpret_cast<const uint4*>(p)[i];
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_f(raw[i]);
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
  constexpr int BYTES = VEC * (int)sizeof(T);
  if constexpr (VEC == 1) {
    *p = from_f<T>(v[0]);
  } else {
    alignas(16) T raw[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) raw[i] = from_f<T>(v[i]);
    if constexpr (BYTES == 8)
      *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(raw);
    else {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i)
        reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(raw)[i];
    }
  }
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {  // all but the newest N groups are there
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Lets a kernel use `bytes` of dynamic shared memory: a driver call, made once per kernel and device.
template <auto KERNEL>
inline cudaError_t allow_smem(int bytes) {
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// Rows of a tensor whose leading axes are (outer, inner): row r starts at (r / inner) * so + (r % inner) * si.
struct RowMap {
  long long so, si;
  unsigned inner;
};

__device__ __forceinline__ long long row_offset(const RowMap& m, unsigned r) {
  if (r < m.inner) return (long long)r * m.si;  // one level, or its first run: no division
  const unsigned o = r / m.inner;
  return (long long)o * m.so + (long long)(r - o * m.inner) * m.si;
}

inline RowMap row_map(long long so, long long si, long long inner) { return RowMap{so, si, (unsigned)inner}; }

inline bool known_type(int t) { return t == UNBLEND_F32 || t == UNBLEND_BF16 || t == UNBLEND_F16; }
inline int elem_size(int t) { return t == UNBLEND_F32 ? 4 : 2; }
inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

inline bool rows_ok(long long outer, long long inner, int cols) {
  return outer > 0 && inner > 0 && cols > 0 && outer < (1LL << 31) && inner < (1LL << 31) &&
         outer * inner < (1LL << 31);
}

// True when every row of `m` starts on a `bytes` boundary.
inline bool rows_aligned(const void* p, const RowMap& m, long long outer, int elem, int bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && (m.inner <= 1 || m.si * elem % bytes == 0) &&
         (outer <= 1 || m.so * elem % bytes == 0);
}

// Column sums out[c] = sum_p part[p][c] of n_part partial rows, always added in the same order (each of 64 threads
// takes every 64th row, then the 64 sums in sequence), so the result does not depend on scheduling. The columns are
// `sums` runs of `cols` values, run i going to out_i. Eight columns (one 32-byte sector) per CTA, so that a few hundred
// columns already occupy many SMs.
constexpr int COLSUM_X = 8, COLSUM_Y = 64;

template <typename TO>
__global__ void __launch_bounds__(COLSUM_X* COLSUM_Y)
    column_sums_kernel(const float* __restrict__ part, int n_part, int cols, int sums, TO* out0, TO* out1) {
  __shared__ float red[COLSUM_Y][COLSUM_X];
  const int tx = threadIdx.x % COLSUM_X, ty = threadIdx.x / COLSUM_X;
  const long long width = (long long)cols * sums;
  const long long c = blockIdx.x * (long long)COLSUM_X + tx;
  float s = 0.f;
  if (c < width) {
#pragma unroll 4
    for (int p = ty; p < n_part; p += COLSUM_Y) s += part[p * width + c];
  }
  red[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < width) {
    const int n = n_part < COLSUM_Y ? n_part : COLSUM_Y;
    for (int y = 1; y < n; ++y) s += red[y][tx];
    if (c < cols)
      out0[c] = from_f<TO>(s);
    else
      out1[c - cols] = from_f<TO>(s);
  }
}

template <typename TO>
inline int launch_column_sums(const float* part, int n_part, int cols, int sums, void* out0, void* out1,
                              cudaStream_t st) {
  const long long width = (long long)cols * sums;
  column_sums_kernel<TO><<<(unsigned)((width + COLSUM_X - 1) / COLSUM_X), COLSUM_X * COLSUM_Y, 0, st>>>(
      part, n_part, cols, sums, static_cast<TO*>(out0), static_cast<TO*>(out1));
  UB_CHECK_LAUNCH();
  return 0;
}

}  // namespace train
}  // namespace ub
