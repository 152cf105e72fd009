// az_dense.hip -- the dense layer y = act(x W + b) + r and its backward pass (include/az_layers.h).
// Part of libaz_mcts.so (gfx950 only).
//
// All three products of a layer are C[M, N] = sum_k A(m, k) B(k, n) over row-major arrays, and differ in
// which axis of an operand is contiguous:
//   forward  y  = x W      A = x  [m][k]   B = W  [k][n]
//   backward dx = dz W^T   A = dz [m][k]   B = W  [n][k]
//            dW = x^T dz   A = x  [k][m]   B = dz [k][n]
// so a kernel takes, for each operand, whether its reduction axis is the contiguous one.
#include <hip/hip_runtime.h>

#include "az_host.h"
#include "az_types.h"

namespace {

// ---------------------------------------------------------------------------
// activations, in float32
__device__ __forceinline__ float act_value(float z, int act) {
  if (act == AZ_ACT_RELU) return z != z ? z : fmaxf(z, 0.0f);
  if (act == AZ_ACT_SWISH) return z / (1.0f + expf(-z));
  if (act == AZ_ACT_GELU) return 0.5f * z * (1.0f + erff(z * 0.70710678f));
  return z;
}

__device__ __forceinline__ float act_slope(float z, int act) {
  if (act == AZ_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  if (act == AZ_ACT_SWISH) {
    const float p = 1.0f / (1.0f + expf(-z));
    return p * (1.0f + z * (1.0f - p));
  }
  if (act == AZ_ACT_GELU)
    return 0.5f * (1.0f + erff(z * 0.70710678f)) + z * (0.39894228f * expf(-0.5f * z * z));
  return 1.0f;
}

// The kept pre-activation.  A 16-bit layer keeps it as float16 for both 16-bit types: it is read only for the
// slope, whose relative error from this rounding is at most 2^-11 |z act''(z) / act'(z)|, an eighth of what
// bfloat16 would give, and the slope does not change beyond +-65504, where a finite z is clamped.  A positive z
// too small for float16 stays positive (the slope of relu).
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
enum { EPI_FORWARD, EPI_STORE, EPI_PARTIAL };

struct Prod {
  const void* a;
  const void* b;
  int64_t lda, ldb;
  int M, N, K;
  int k_chunk;          // reduction length of one split (blockIdx.z)
  int a_vec, b_vec;     // 16-byte loads are aligned
  int tiles_m, tiles_n;
  // epilogue
  int act, out_vec;     // out_vec: rows of the outputs can be read and written four elements at a time
  const void* bias;
  const void* residual;
  void* z;
  void* out;
  float* partial;       // [splits][M][N]
};

// Four consecutive outputs of row m from column n.
template <typename T, int EPI>
__device__ __forceinline__ void finish(const Prod& p, int m, int n, const float* v) {
  if (m >= p.M || n >= p.N) return;
  const int64_t at = (int64_t)m * p.N + n;
  const int have = p.N - n < 4 ? p.N - n : 4;
  if constexpr (EPI == EPI_PARTIAL) {
    float* out = p.partial + (int64_t)blockIdx.z * p.M * p.N + at;
    if (p.out_vec) {
      *reinterpret_cast<float4*>(out) = float4{v[0], v[1], v[2], v[3]};
    } else {
      for (int i = 0; i < have; ++i) out[i] = v[i];
    }
  } else {
    T* out = (T*)p.out + at;
    if constexpr (EPI == EPI_STORE) {
      if (p.out_vec) {
        AzVec<T, 4> o;
        for (int i = 0; i < 4; ++i) o.v[i] = (T)v[i];
        az_storev<T, 4>(out, o);
      } else {
        for (int i = 0; i < have; ++i) out[i] = (T)v[i];
      }
    } else {
      typedef typename Kept<T>::type Z;
      const T* bias = (const T*)p.bias;
      const T* res = p.residual ? (const T*)p.residual + at : nullptr;
      Z* z = p.z ? (Z*)p.z + at : nullptr;
      if (p.out_vec) {
        AzVec<T, 4> o, r, b;
        AzVec<Z, 4> zz;
        if (bias) b = az_loadv<T, 4>(bias + n);
        if (res) r = az_loadv<T, 4>(res);
        for (int i = 0; i < 4; ++i) {
          const float s = v[i] + (bias ? (float)b.v[i] : 0.0f);
          keep(&zz.v[i], s);
          o.v[i] = (T)(act_value(s, p.act) + (res ? (float)r.v[i] : 0.0f));
        }
        if (z) az_storev<Z, 4>(z, zz);
        az_storev<T, 4>(out, o);
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

// ---------------------------------------------------------------------------
// Any sizes and alignments: 64 x 64 outputs a workgroup, four waves of 32 x 32, 64 bytes of reduction a step.
// Operands go through registers (one step ahead, every element guarded, zero outside) into LDS, each row's reduction
// contiguous, rows 80 bytes apart so that the 16 rows of an operand read fall on different banks.
constexpr int TILE = 64, ROW_BYTES = 80;

template <typename T, bool KC>
struct Stage {
  static constexpr int E = AzPack<T>::N, BK = 4 * E;
  AzPack<T> r;
  // row / first reduction index (KC) or first row / reduction index (not KC) of this thread's 16 bytes
  __device__ static int row(int t) { return KC ? t / 4 : (t % (TILE / E)) * E; }
  __device__ static int red(int t) { return KC ? (t % 4) * E : t / (TILE / E); }
  __device__ void load(const T* p, int64_t ld, int rows, int r0, int k0, int k1, bool vec) {
    const int r_ = r0 + row(threadIdx.x), k_ = k0 + red(threadIdx.x);
    const int cont = KC ? k_ : r_, cont_end = KC ? k1 : rows;
    const bool line = KC ? r_ < rows : k_ < k1;
    const T* q = p + (KC ? (int64_t)r_ * ld + k_ : (int64_t)k_ * ld + r_);
    if (line && vec && cont + E <= cont_end) {
      r = az_load16(q);
    } else {
      for (int e = 0; e < E; ++e) r.v[e] = line && cont + e < cont_end ? q[e] : (T)0.0f;
    }
  }
  __device__ void store(char* lds) const {
    if constexpr (KC) {
      az_store16((T*)(lds + row(threadIdx.x) * ROW_BYTES) + red(threadIdx.x), r);
    } else {
      for (int e = 0; e < E; ++e) ((T*)(lds + (row(threadIdx.x) + e) * ROW_BYTES))[red(threadIdx.x)] = r.v[e];
    }
  }
};

template <typename T, bool AKC, bool BKC, int EPI>
__global__ __launch_bounds__(256) void k_product_tile(Prod p) {
  constexpr int BK = Stage<T, true>::BK;
  __shared__ alignas(16) char lds[2][2][TILE * ROW_BYTES];
  const int m0 = (blockIdx.x % p.tiles_m) * TILE, n0 = (blockIdx.x / p.tiles_m) * TILE;
  const int k_begin = blockIdx.z * p.k_chunk, k_end = min(p.K, k_begin + p.k_chunk);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
  Stage<T, AKC> sa;
  Stage<T, BKC> sb;
  az_f32x4 acc[2][2] = {};
  sa.load((const T*)p.a, p.lda, p.M, m0, k_begin, k_end, p.a_vec);
  sb.load((const T*)p.b, p.ldb, p.N, n0, k_begin, k_end, p.b_vec);
  int buf = 0;
  for (int k = k_begin; k < k_end; k += BK, buf ^= 1) {
    sa.store(lds[buf][0]);
    sb.store(lds[buf][1]);
    __syncthreads();   // (the other buffer's readers passed the barrier of the step before)
    if (k + BK < k_end) {
      sa.load((const T*)p.a, p.lda, p.M, m0, k + BK, k_end, p.a_vec);
      sb.load((const T*)p.b, p.ldb, p.N, n0, k + BK, k_end, p.b_vec);
    }
    AzPack<T> fa[2], fb[2];
    for (int i = 0; i < 2; ++i) {
      const int off = (lane & 15) * ROW_BYTES + (lane >> 4) * 16;
      fa[i] = az_load16((const T*)(lds[buf][0] + (wm + i * 16) * ROW_BYTES + off));
      fb[i] = az_load16((const T*)(lds[buf][1] + (wn + i * 16) * ROW_BYTES + off));
    }
    // operands exchanged: a lane then holds four consecutive columns of one output row
    for (int i = 0; i < 2; ++i)
      for (int j = 0; j < 2; ++j) acc[i][j] = mma(fb[j], fa[i], acc[i][j]);
  }
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2; ++j) {
      const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
      finish<T, EPI>(p, m0 + wm + i * 16 + (lane & 15), n0 + wn + j * 16 + (lane >> 4) * 4, v);
    }
}

// ---------------------------------------------------------------------------
// Joins split sums in the order of the splits: 64 groups of four outputs a workgroup, the splits dealt to four
// waves whose sums are added in their order.  Segment 0 takes the epilogue, segment 1 (the bias' gradient) is
// stored as it is.
struct Join {
  const float* part[2];
  int64_t length[2];
  int splits[2];
  void* out1;
  int64_t blocks0;
};

template <typename T, int EPI>
__global__ __launch_bounds__(256) void k_join(Join q, Prod p) {
  __shared__ float sums[4][64][4];
  const int seg = (int64_t)blockIdx.x >= q.blocks0;
  const int64_t L = q.length[seg];
  const int g = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t at = (((int64_t)blockIdx.x - (seg ? q.blocks0 : 0)) * 64 + g) * 4;
  const int have = (int)max((int64_t)0, min((int64_t)4, L - at));
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (have > 0) {
    const float* part = q.part[seg] + at;
    const bool vec = L % 4 == 0;
#pragma unroll 4
    for (int i = w; i < q.splits[seg]; i += 4) {
      const float* r = part + (int64_t)i * L;
      if (vec) {
        const float4 x = *reinterpret_cast<const float4*>(r);
        s[0] += x.x, s[1] += x.y, s[2] += x.z, s[3] += x.w;
      } else {
        for (int e = 0; e < have; ++e) s[e] += r[e];
      }
    }
  }
  for (int e = 0; e < 4; ++e) sums[w][g][e] = s[e];
  __syncthreads();
  if (w != 0 || have == 0) return;
  for (int e = 0; e < 4; ++e) s[e] = ((sums[0][g][e] + sums[1][g][e]) + sums[2][g][e]) + sums[3][g][e];
  if (seg) {
    for (int e = 0; e < have; ++e) ((T*)q.out1)[at + e] = (T)s[e];
  } else if (p.out_vec) {   // N is a multiple of four: the group is in one row
    finish<T, EPI>(p, (int)(at / p.N), (int)(at % p.N), s);
  } else {
    for (int e = 0; e < have; ++e) {
      Prod one = p;
      const int64_t i = at + e;
      const int n = (int)(i % p.N);
      one.N = n + 1;       // one element of the row
      one.out = (T*)p.out + (int64_t)(i / p.N) * (p.N - one.N);
      if (p.residual) one.residual = (const T*)p.residual + (int64_t)(i / p.N) * (p.N - one.N);
      if (p.z) one.z = (typename Kept<T>::type*)p.z + (int64_t)(i / p.N) * (p.N - one.N);
      finish<T, EPI>(one, (int)(i / p.N), n, s + e);
    }
  }
}

// ---------------------------------------------------------------------------
// dz = dy act'(z), rounded to T, and the partial column sums of dz before the rounding: a workgroup takes 64 V
// columns (V a thread) of a chunk of rows, four rows at a time.
struct Slope {
  const void* dy;
  const void* z;
  void* dz;            // may be null (no activation: dy itself is dz)
  float* partial;      // [chunks][N], may be null
  int M, N, act, rows_per_chunk;
};

template <typename T, int V>
__global__ __launch_bounds__(256) void k_slope(Slope p) {
  typedef typename Kept<T>::type Z;
  __shared__ float sums[3][64][V];
  const int g = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int n = (blockIdx.x * 64 + g) * V;
  const int m_end = min(p.M, (int)(blockIdx.y + 1) * p.rows_per_chunk);
  float s[V] = {};
  if (n < p.N) {
    for (int m = blockIdx.y * p.rows_per_chunk + w; m < m_end; m += 4) {
      const int64_t at = (int64_t)m * p.N + n;
      const AzVec<T, V> dy = az_loadv<T, V>((const T*)p.dy + at);
      AzVec<Z, V> z;
      if (p.act != AZ_ACT_NONE) z = az_loadv<Z, V>((const Z*)p.z + at);
      AzVec<T, V> o;
      for (int i = 0; i < V; ++i) {
        const float d = p.act == AZ_ACT_NONE ? (float)dy.v[i] : (float)dy.v[i] * act_slope((float)z.v[i], p.act);
        s[i] += d;
        o.v[i] = (T)d;
      }
      if (p.dz) az_storev<T, V>((T*)p.dz + at, o);
    }
  }
  if (!p.partial) return;
  if (w > 0)
    for (int i = 0; i < V; ++i) sums[w - 1][g][i] = s[i];
  __syncthreads();
  if (w > 0 || n >= p.N) return;
  for (int i = 0; i < V; ++i)
    p.partial[(int64_t)blockIdx.y * p.N + n + i] = ((s[i] + sums[0][g][i]) + sums[1][g][i]) + sums[2][g][i];
}

template <typename T>
__global__ void k_zero(T* p, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) p[i] = (T)0.0f;
}

// ---------------------------------------------------------------------------
int size_of(int dtype) { return dtype == AZ_TYPE_F32 ? 4 : 2; }
int64_t round16(int64_t n) { return (n + 15) & ~(int64_t)15; }

// Splits of a reduction of K for tiles x splits workgroups: enough to give every compute unit two, at least 128
// elements each.
int splits_of(int64_t tiles, int64_t K) {
  const int64_t want = az_ceil(512, tiles), most = az_ceil(K, 128);
  int64_t s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

// Rows of dz that one workgroup of k_slope takes: 1024 workgroups in all, 64 chunks at most (the join reads them).
int slope_chunks(int64_t rows, int64_t col_tiles) {
  int64_t c = az_ceil(1024, col_tiles);
  if (c > 64) c = 64;
  const int64_t most = az_ceil(rows, 16);
  return (int)(c < most ? c : most);
}

struct Plan {
  int splits_y, splits_dx, splits_dw, chunks;
  int64_t partial_floats;   // of the largest product's splits
};

Plan plan_of(int64_t M, int64_t K, int64_t N) {
  auto tiles = [](int64_t a, int64_t b) { return az_ceil(a, TILE) * az_ceil(b, TILE); };
  Plan p;
  p.splits_y = splits_of(tiles(M, N), K);
  p.splits_dx = splits_of(tiles(M, K), N);
  p.splits_dw = splits_of(tiles(K, N), M);
  p.chunks = slope_chunks(M, az_ceil(N, 64 * (N % 4 == 0 ? 4 : 1)));
  return p;
}

int check(int dtype, int act, int64_t rows, int64_t fan_in, int64_t fan_out) {
  if (dtype < AZ_TYPE_F32 || dtype > AZ_TYPE_F16) return az_fail(AZ_ERR_INVALID, "dense: unknown type %d", dtype);
  if (act < AZ_ACT_NONE || act > AZ_ACT_GELU) return az_fail(AZ_ERR_INVALID, "dense: unknown activation %d", act);
  if (rows < 0 || fan_in < 1 || fan_out < 1)
    return az_fail(AZ_ERR_INVALID, "dense: rows=%lld fan_in=%lld fan_out=%lld", (long long)rows, (long long)fan_in,
                   (long long)fan_out);
  if (rows > 0x7fff0000) return az_fail(AZ_ERR_UNSUPPORTED, "dense: rows up to %d", 0x7fff0000);
  if (fan_in > AZ_DENSE_MAX_WIDTH || fan_out > AZ_DENSE_MAX_WIDTH)
    return az_fail(AZ_ERR_UNSUPPORTED, "dense: widths up to %d", AZ_DENSE_MAX_WIDTH);
  return AZ_OK;
}

// One product (and, with `bias_part`, the join of the bias' gradient).  `partial` holds splits x M x N floats.
template <typename T, bool AKC, bool BKC, int EPI>
int product(Prod p, int splits, float* partial, const Join* extra, hipStream_t stream) {
  const int E = AzPack<T>::N;
  p.a_vec = p.lda % E == 0 && az_aligned16(p.a);
  p.b_vec = p.ldb % E == 0 && az_aligned16(p.b);
  auto four = [](const void* q) { return ((uintptr_t)q & (4 * sizeof(T) - 1)) == 0; };
  p.out_vec = p.N % 4 == 0 && four(p.out) && four(p.bias) && four(p.residual) && az_aligned16(p.z);
  p.tiles_m = (int)az_ceil(p.M, TILE), p.tiles_n = (int)az_ceil(p.N, TILE);
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  if (tiles > 0x7fffffff) return az_fail(AZ_ERR_UNSUPPORTED, "dense: too many output tiles");
  const int BK = Stage<T, true>::BK;
  p.k_chunk = (int)(az_ceil(az_ceil(p.K, splits), BK) * BK);
  splits = (int)az_ceil(p.K, p.k_chunk);
  const dim3 grid((unsigned)tiles, 1, splits), block(256);
  if (splits == 1) {
    k_product_tile<T, AKC, BKC, EPI><<<grid, block, 0, stream>>>(p);
    AZ_LAUNCH_CHECK();
  } else {
    Prod q = p;
    q.partial = partial;
    q.out_vec = p.N % 4 == 0;
    k_product_tile<T, AKC, BKC, EPI_PARTIAL><<<grid, block, 0, stream>>>(q);
    AZ_LAUNCH_CHECK();
  }
  if (splits > 1 || extra) {
    Join j = extra ? *extra : Join{};
    if (splits > 1) {
      j.part[0] = partial, j.length[0] = (int64_t)p.M * p.N, j.splits[0] = splits;
      j.blocks0 = az_ceil(j.length[0], 256);
    }
    const int64_t blocks = j.blocks0 + az_ceil(j.length[1], 256);
    k_join<T, EPI><<<dim3((unsigned)blocks), dim3(256), 0, stream>>>(j, p);
    AZ_LAUNCH_CHECK();
  }
  return AZ_OK;
}

// Workspace layout of a backward pass: [dz][bias partials][split sums]
struct Layout {
  int64_t dz, bias, partial, total;
};

Layout layout_of(int dtype, int64_t M, int64_t K, int64_t N, int pass) {
  const Plan p = plan_of(M, K, N);
  Layout l = {0, 0, 0, 0};
  if (pass == 0) {
    l.total = p.splits_y > 1 ? p.splits_y * M * N * 4 : 0;
    return l;
  }
  l.bias = round16(M * N * size_of(dtype));
  l.partial = l.bias + round16((int64_t)p.chunks * N * 4);
  const int64_t dx = p.splits_dx > 1 ? p.splits_dx * M * K : 0, dw = p.splits_dw > 1 ? p.splits_dw * K * N : 0;
  l.total = l.partial + 4 * (dx > dw ? dx : dw);
  return l;
}

}  // namespace

extern "C" int64_t az_dense_workspace_bytes(int32_t dtype, int32_t rows, int32_t fan_in, int32_t fan_out,
                                            int32_t pass) {
  if (check(dtype, AZ_ACT_NONE, rows, fan_in, fan_out) != AZ_OK || pass < 0 || pass > 1) return -1;
  return rows == 0 ? 0 : layout_of(dtype, rows, fan_in, fan_out, pass).total;
}

extern "C" int az_dense_forward(int32_t dtype, int32_t act, int32_t rows, int32_t fan_in, int32_t fan_out,
                                const void* x, const void* kernel, const void* bias, const void* residual, void* y,
                                void* z, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check(dtype, act, rows, fan_in, fan_out)) return rc;
  if (rows == 0) return AZ_OK;
  if (!x || !kernel || !y) return az_fail(AZ_ERR_INVALID, "dense: null x, kernel or y");
  const Layout l = layout_of(dtype, rows, fan_in, fan_out, 0);
  if (workspace_bytes < l.total || (l.total && (!workspace || !az_aligned16(workspace))))
    return az_fail(AZ_ERR_INVALID, "dense: the workspace must hold %lld bytes, 16-byte aligned", (long long)l.total);
  return az_dispatch_type(dtype, [&]<typename T>() {
    Prod p = {};
    p.a = x, p.lda = fan_in, p.b = kernel, p.ldb = fan_out;
    p.M = rows, p.N = fan_out, p.K = fan_in;
    p.act = act, p.bias = bias, p.residual = residual, p.z = act == AZ_ACT_NONE ? nullptr : z, p.out = y;
    const Plan plan = plan_of(rows, fan_in, fan_out);
    return product<T, true, false, EPI_FORWARD>(p, plan.splits_y, (float*)workspace, nullptr, (hipStream_t)stream);
  });
}

extern "C" int az_dense_backward(int32_t dtype, int32_t act, int32_t rows, int32_t fan_in, int32_t fan_out,
                                 const void* x, const void* kernel, const void* z, const void* dy, void* dx,
                                 void* dkernel, void* dbias, void* workspace, int64_t workspace_bytes,
                                 void* stream_) {
  if (int rc = check(dtype, act, rows, fan_in, fan_out)) return rc;
  hipStream_t stream = (hipStream_t)stream_;
  if (!dx && !dkernel && !dbias) return AZ_OK;
  return az_dispatch_type(dtype, [&]<typename T>() -> int {
    if (rows == 0) {
      const int64_t n = (int64_t)fan_in * fan_out;
      if (dkernel) k_zero<T><<<dim3((unsigned)az_ceil(n, 256)), dim3(256), 0, stream>>>((T*)dkernel, n);
      if (dbias) k_zero<T><<<dim3((unsigned)az_ceil(fan_out, 256)), dim3(256), 0, stream>>>((T*)dbias, fan_out);
      AZ_LAUNCH_CHECK();
      return AZ_OK;
    }
    if (!dy || (dkernel && !x) || (dx && !kernel) || (act != AZ_ACT_NONE && !z))
      return az_fail(AZ_ERR_INVALID, "dense backward: null dy, or x / kernel / z where it is needed");
    const Layout l = layout_of(dtype, rows, fan_in, fan_out, 1);
    if (workspace_bytes < l.total || !workspace || !az_aligned16(workspace))
      return az_fail(AZ_ERR_INVALID, "dense: the workspace must hold %lld bytes, 16-byte aligned",
                     (long long)l.total);
    char* ws = (char*)workspace;
    const Plan plan = plan_of(rows, fan_in, fan_out);
    const void* dz = dy;
    if (act != AZ_ACT_NONE || dbias) {
      Slope s = {};
      s.dy = dy, s.z = z, s.dz = act != AZ_ACT_NONE ? ws + l.dz : nullptr;
      s.partial = dbias ? (float*)(ws + l.bias) : nullptr;
      s.M = rows, s.N = fan_out, s.act = act, s.rows_per_chunk = (int)az_ceil(rows, plan.chunks);
      const bool vec = fan_out % 4 == 0 && ((uintptr_t)dy & (4 * sizeof(T) - 1)) == 0 && az_aligned16(z);
      const int V = vec ? 4 : 1;
      const dim3 grid((unsigned)az_ceil(fan_out, 64 * V), plan.chunks), block(256);
      if (vec)
        k_slope<T, 4><<<grid, block, 0, stream>>>(s);
      else
        k_slope<T, 1><<<grid, block, 0, stream>>>(s);
      AZ_LAUNCH_CHECK();
      if (s.dz) dz = s.dz;
    }
    if (dx) {
      Prod p = {};
      p.a = dz, p.lda = fan_out, p.b = kernel, p.ldb = fan_out;
      p.M = rows, p.N = fan_in, p.K = fan_out, p.out = dx;
      if (int rc = product<T, true, true, EPI_STORE>(p, plan.splits_dx, (float*)(ws + l.partial), nullptr, stream))
        return rc;
    }
    Join j = {};
    j.part[1] = (const float*)(ws + l.bias), j.length[1] = fan_out, j.splits[1] = plan.chunks, j.out1 = dbias;
    if (dkernel) {
      Prod p = {};
      p.a = x, p.lda = fan_in, p.b = dz, p.ldb = fan_out;
      p.M = fan_in, p.N = fan_out, p.K = rows, p.out = dkernel;
      return product<T, false, false, EPI_STORE>(p, plan.splits_dw, (float*)(ws + l.partial), dbias ? &j : nullptr,
                                                 stream);
    }
    if (dbias) {
      k_join<T, EPI_STORE><<<dim3((unsigned)az_ceil(fan_out, 256)), dim3(256), 0, stream>>>(j, Prod{});
      AZ_LAUNCH_CHECK();
    }
    return AZ_OK;
  });
}
