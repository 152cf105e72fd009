// az_dense.h -- what the product kernels of az_dense.hip and az_dense_wide.hip share: activations, the
// epilogues, the matrix instructions.
#ifndef AZ_DENSE_H_
#define AZ_DENSE_H_

#include <hip/hip_runtime.h>

#include "az_host.h"
#include "az_types.h"

namespace az_dense {

// ---------------------------------------------------------------------------
// activations, in float32
// exp(-z): the exponent's product with log2(e) in two parts, the second one (below 2^-24 of the first) to first
// order.  Off by three units in the last place where the result is normal.
__device__ __forceinline__ float exp_minus(float z) {
  const float hi = -1.44269502f * z;
  const float lo = fmaf(z, -1.92596303e-8f, fmaf(z, -1.44269502f, -hi));
  const float e = __builtin_amdgcn_exp2f(hi);
  return fabsf(lo) < 1.0f ? e * fmaf(0.693147182f, lo, 1.0f) : e;   // (infinite z)
}

__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + exp_minus(z)); }

// The normal distribution's integral up to z: 1 + erf(z / sqrt 2) would cancel for negative z, down to nothing below -5.6.
__device__ __forceinline__ float normal_cdf(float z) { return 0.5f * erfcf(z * -0.70710678f); }

__device__ __forceinline__ float act_value(float z, int act) {
  if (act == AZ_ACT_RELU) return z != z ? z : fmaxf(z, 0.0f);
  if (act == AZ_ACT_SWISH) return z * sigmoid(z);
  if (act == AZ_ACT_GELU) return z * normal_cdf(z);
  return z;
}

__device__ __forceinline__ float act_slope(float z, int act) {
  if (act == AZ_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  if (act == AZ_ACT_SWISH) {
    const float p = sigmoid(z);
    return p * (1.0f + z * (1.0f - p));
  }
  if (act == AZ_ACT_GELU)
    return normal_cdf(z) + z * (0.39894228f * exp_minus(0.5f * z * z));
  return 1.0f;
}

// The kept pre-activation.  A 16-bit layer keeps it as float16 for both 16-bit types: it is read only for the
// slope, whose relative error from this rounding is at most 2^-11 |z act''(z) / act'(z)|, an eighth of what
// bfloat16 would give, and the slope does not change beyond +-65504, where a finite z is clamped.  A positive z
// too small for float16 stays positive (the slope of relu).  float32 would take twice the memory between the passes for
// gradients' errors of 1.00 instead of 1.05 times their last rounding's in float16 (bfloat16: 1.00 either way).
template <typename T>
struct Kept {
  typedef az_f16 type;
};
template <>
struct Kept<float> {
  typedef float type;
};
__device__ __forceinline__ void keep(float* p, float z) { *p = z; }
__device__ __forceinline__ void keep(az_f16* p, float z) {
  if (fabsf(z) < INFINITY) z = fminf(fmaxf(z, -65504.0f), 65504.0f);
  if (z > 0.0f) z = fmaxf(z, 5.9604645e-8f);
  *p = (az_f16)z;
}

// ---------------------------------------------------------------------------
// dz of a 16-bit layer whose slope is not 0 or 1 is kept as two values of its type, dz = hi + lo 2^-p with p the type's
// significant bits: to 2^-16 of itself at least (bfloat16; float16: 2^-22), where rounding it to the type alone would add as much
// to the gradients' errors as their own last rounding does (1.41 to 1.46 times that rounding's error in all, measured from
// 300 x 520 x 264 on; 1.00 with two planes, float16 1.05 by its z).  The products run over the lo plane, scale, and go on over the
// hi plane: twice the matrix instructions, dx and dkernel of 16384 x 4096 x 4096 bfloat16 830 and 791 us (418 and 398 over one
// plane, as a layer without an activation or with relu has it).
template <typename T>
struct Low {
  static constexpr float UP = 1.0f, DOWN = 1.0f;
};
template <>
struct Low<az_bf16> {
  static constexpr float UP = 0x1p8f, DOWN = 0x1p-8f;
};
template <>
struct Low<az_f16> {
  static constexpr float UP = 0x1p11f, DOWN = 0x1p-11f;
};

// Between the planes.  A lo sum that is not finite comes from the other operand, which reaches the hi plane's sum itself.
template <typename T>
__device__ __forceinline__ void scale_low(az_f32x4& c) {
  for (int e = 0; e < 4; ++e) c[e] = fabsf(c[e]) < INFINITY ? c[e] * Low<T>::DOWN : 0.0f;
}

enum { EPI_FORWARD, EPI_STORE, EPI_PARTIAL };

struct Prod {
  const void* a;
  const void* b;
  int64_t lda, ldb;
  int M, N, K;
  int k_chunk;          // reduction length of one split (blockIdx.z)
  int planes;           // of dz in a 16-bit layer: 2 (hi, lo) or 1
  int tiles_m, tiles_n;
  // epilogue
  int act;
  const void* bias;
  const void* residual;
  void* z;
  void* out;
  float* partial;       // [splits][M][N]
  // operands as planes (float32 as three bfloat16 ones in the wide kernel; dz of 16 bits): elements from one to the
  // next, 0 for an operand that has one only; and the float32 operands
  int64_t a_plane, b_plane;
  const float* a32;
  const float* b32;
  int64_t lda32, ldb32;
};

// Four consecutive outputs of row m from column n, at any address.  `early`: the caller has loaded their residual.
template <typename T, int EPI>
__device__ __forceinline__ void finish(const Prod& p, int m, int n, const float* v, bool early = false,
                                       AzVec<T, 4> loaded = {}) {
  if (m >= p.M || n >= p.N) return;
  const int64_t at = (int64_t)m * p.N + n;
  const int have = p.N - n;
  if constexpr (EPI == EPI_PARTIAL) {
    float* out = p.partial + (int64_t)blockIdx.z * p.M * p.N + at;
    if (have >= 4) {
      az_storeu<float, 4>(out, AzVec<float, 4>{v[0], v[1], v[2], v[3]});
    } else {
      for (int i = 0; i < have; ++i) out[i] = v[i];
    }
  } else {
    T* out = (T*)p.out + at;
    if constexpr (EPI == EPI_STORE) {
      if (have >= 4) {
        AzVec<T, 4> o;
        for (int i = 0; i < 4; ++i) o.v[i] = (T)v[i];
        az_storeu<T, 4>(out, o);
      } else {
        for (int i = 0; i < have; ++i) out[i] = (T)v[i];
      }
    } else {
      typedef typename Kept<T>::type Z;
      const T* bias = (const T*)p.bias;
      const T* res = p.residual ? (const T*)p.residual + at : nullptr;
      Z* z = p.z ? (Z*)p.z + at : nullptr;
      if (have >= 4) {
        AzVec<T, 4> o, r = loaded, b;
        AzVec<Z, 4> zz;
        if (bias) b = az_loadu<T, 4>(bias + n);
        if (res && !early) r = az_loadu<T, 4>(res);
        for (int i = 0; i < 4; ++i) {
          const float s = v[i] + (bias ? (float)b.v[i] : 0.0f);
          keep(&zz.v[i], s);
          o.v[i] = (T)(act_value(s, p.act) + (res ? (float)r.v[i] : 0.0f));
        }
        if (z) az_storeu<Z, 4>(z, zz);
        az_storeu<T, 4>(out, o);
      } else {
        for (int i = 0; i < have; ++i) {
          const float s = v[i] + (bias ? (float)bias[n + i] : 0.0f);
          if (z) keep(z + i, s);
          out[i] = (T)(act_value(s, p.act) + (res ? (float)res[i] : 0.0f));
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// The matrix instructions on 64 bytes of reduction: 16 float32 values (four 16x16x4 steps) or 32 of 16 bits
// (one 16x16x32 step).  Lane l gives 16 bytes of row l % 16, those at (l / 16) * 16; which reduction
// index a lane's j-th element stands for is the same for both operands, so any order does.
__device__ __forceinline__ az_f32x4 mma(const AzPack<float>& a, const AzPack<float>& b, az_f32x4 c) {
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], c, 0, 0, 0);
  return c;
}
typedef az_bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef az_f16 f16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ az_f32x4 mma(const AzPack<az_bf16>& a, const AzPack<az_bf16>& b, az_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                 0, 0);
}
__device__ __forceinline__ az_f32x4 mma(const AzPack<az_f16>& a, const AzPack<az_f16>& b, az_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                0);
}


}  // namespace

// az_dense_wide.hip: the products C = A B of the three passes on the wide kernel, tiles of 256 x 256 or 128 x 128.
// T: the operands' type; SPLIT: float32 operands as bfloat16 planes (T is then float).  Splits > 1 write p.partial.
enum { PASS_Y, PASS_DX, PASS_DW };
int az_product_wide(int dtype, int pass, bool split_k, bool big, const az_dense::Prod* p, int splits, hipStream_t stream);

#endif  // AZ_DENSE_H_
