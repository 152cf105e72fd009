// az_types.h -- element types and small helpers of the layer kernels (az_dense.hip, az_norm.hip,
// az_sample.hip): float32, bfloat16 and float16 storage, float32 arithmetic.
#ifndef AZ_TYPES_H_
#define AZ_TYPES_H_

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/az_layers.h"

typedef __bf16 az_bf16;
typedef _Float16 az_f16;
typedef float az_f32x4 __attribute__((ext_vector_type(4)));

// A workgroup barrier that orders LDS accesses alone: __syncthreads also waits for the global loads in flight, the
// ones that run ahead among them.
static __device__ __forceinline__ void az_lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// sixteen bytes of T
template <typename T>
struct alignas(16) AzPack {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};

template <typename T>
static __device__ __forceinline__ AzPack<T> az_load16(const T* p) {
  AzPack<T> r;
  *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(p);
  return r;
}

template <typename T>
static __device__ __forceinline__ void az_store16(T* p, const AzPack<T>& r) {
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r);
}

// V elements, V * sizeof(T) bytes aligned to their own size
template <typename T, int V>
struct alignas(sizeof(T) * V) AzVec {
  T v[V];
};

template <typename T, int V>
static __device__ __forceinline__ void az_storev(T* p, const AzVec<T, V>& r) {
  *reinterpret_cast<AzVec<T, V>*>(p) = r;
}

// V elements at any element's address: gfx950 loads and stores 16 bytes at any address, and the compiler, told the
// true alignment, emits just that.
template <typename T, int V>
static __device__ __forceinline__ AzVec<T, V> az_loadu(const T* p) {
  AzVec<T, V> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}

template <typename T, int V>
static __device__ __forceinline__ void az_storeu(T* p, const AzVec<T, V>& r) {
  __builtin_memcpy(p, &r, sizeof(r));
}

static inline bool az_aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

static inline int64_t az_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A launch holds fewer than 2^32 threads along an axis.
static inline bool az_grid_fits(int64_t blocks, int threads) { return blocks * threads <= 0xffffffffll; }

// f.template operator()<T>() for an AZ_TYPE_ code
template <typename F>
static int az_dispatch_type(int dtype, F&& f) {
  if (dtype == AZ_TYPE_F32) return f.template operator()<float>();
  if (dtype == AZ_TYPE_BF16) return f.template operator()<az_bf16>();
  return f.template operator()<az_f16>();
}

#endif  // AZ_TYPES_H_
