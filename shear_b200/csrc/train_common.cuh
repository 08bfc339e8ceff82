// Element types, aligned vectors and dispatch shared by the kernels that train
// a table of vectors (embedding.cu, fp8_quantize.cu, fp8_matmul.cu, distill.cu).
#pragma once
#include <atomic>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"

namespace tessa {
namespace train {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
// The one rounding of a result: nearest, ties to even.
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}

template <class T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

// Marks a bad input; the word is mapped host memory that only ever receives
// this store or a wait's bit, and any of them names a failure.
__device__ __forceinline__ void report(uint32_t* err, uint32_t bit) { *reinterpret_cast<volatile uint32_t*>(err) = bit; }

// Calls f with a value of the C++ type of `dtype`.
template <class F>
cudaError_t with_type(uint32_t dtype, F f) {
  switch (dtype) {
    case TESSA_F32: return f(float());
    case TESSA_BF16: return f(__nv_bfloat16());
    default: return f(__half());
  }
}

// Raises a kernel's dynamic shared memory limit to the device's, once a device
// (`done`: a static of the caller, one a kernel).
struct SmemRaised {
  std::atomic<uint64_t> devices{0};
};
template <class K>
cudaError_t raise_smem(K* kernel, int device, int most, SmemRaised& done) {
  const uint64_t bit = 1ull << (device & 63);
  if (done.devices.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e == cudaSuccess) done.devices.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

inline uint32_t type_bytes(uint32_t dtype) { return dtype == TESSA_F32 ? 4u : 2u; }

inline uint64_t div_up(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// The most elements (a power of two up to `most`) that every row of a matrix
// can be accessed by at once: base, stride and columns are multiples of it.
inline uint32_t vector_elems(const void* base, uint64_t rows, uint64_t cols, uint64_t stride, uint32_t bytes,
                             uint32_t most) {
  uint32_t v = most;
  while (v > 1 && (reinterpret_cast<uintptr_t>(base) % (v * bytes) || cols % v || (rows > 1 && stride % v))) v >>= 1;
  return v;
}

}  // namespace train
}  // namespace tessa
