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

#include <type_traits>

#include "az_dense.h"

using namespace az_dense;

namespace {

// ---------------------------------------------------------------------------
// Any sizes and alignments (gfx950 loads 16 bytes at any address): 64 x 64 outputs a workgroup, four waves of 32 x 32,
// 256 bytes of reduction a step (64 float32 elements, 128 of 16 bits).  Operands go through registers (one step ahead,
// every element guarded, zero outside) into LDS as they lie in memory.  One whose reduction is contiguous: 64 rows, 272
// bytes apart so that the 16 rows of a read fall on different banks, read 16 bytes a lane.  The other: a row of 64
// elements for each reduction index, read element by element (float32; rows 320 bytes apart, the four of a read on
// different banks) or by the transposing read (16 bits; rows 160 bytes apart).  Writing it transposed instead cost as many
// LDS cycles as the matrix instructions take.  A step this long keeps the loads of the next one in flight for two
// thousand cycles of matrix instructions; with 64 bytes a step the loop waited for memory.
// 8192 x 256 x 256 float32: 20.5 us with swish, 16.5 us for dx and, in splits, dkernel (at the rate of a large library
// product in float32, 150 TFLOP/s, 7 us: with two workgroups a compute unit the first loads and last stores of four steps
// are not hidden).
constexpr int TILE = 64, PACKS = 4;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <typename T, bool KC>
struct Stage {
  static constexpr int E = AzPack<T>::N, BK = 4 * PACKS * E;
  static constexpr int PITCH = KC ? 272 : sizeof(T) == 4 ? 320 : 160, BYTES = PITCH * (KC ? TILE : BK);
  AzPack<T> r[PACKS];
  // output row / first reduction index (KC) or first output row / reduction index (not KC) of this thread's pack q
  __device__ static int row(int q) {
    return KC ? threadIdx.x / (4 * PACKS) + q * (TILE / PACKS) : (threadIdx.x % (TILE / E)) * E;
  }
  __device__ static int red(int q) {
    return KC ? (threadIdx.x % (4 * PACKS)) * E : threadIdx.x / (TILE / E) + q * (BK / PACKS);
  }
  __device__ void load(const T* p, int64_t ld, int rows, int r0, int k0, int k1) {
    if (r0 + TILE <= rows && k0 + BK <= k1) {   // the whole step: loads without a branch between them, in flight together
#pragma unroll
      for (int q = 0; q < PACKS; ++q) {
        const int r_ = r0 + row(q), k_ = k0 + red(q);
        __builtin_memcpy(&r[q], p + (KC ? (int64_t)r_ * ld + k_ : (int64_t)k_ * ld + r_), 16);
      }
      return;
    }
#pragma unroll
    for (int q = 0; q < PACKS; ++q) {
      const int r_ = r0 + row(q), k_ = k0 + red(q);
      const int cont = KC ? k_ : r_, cont_end = KC ? k1 : rows;
      const bool line = KC ? r_ < rows : k_ < k1;
      const T* at = p + (KC ? (int64_t)r_ * ld + k_ : (int64_t)k_ * ld + r_);
      if (line && cont + E <= cont_end) {
        __builtin_memcpy(&r[q], at, 16);   // (at any address)
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) r[q].v[e] = line && cont + e < cont_end ? at[e] : (T)0.0f;
      }
    }
  }
  __device__ void store(char* lds) const {
#pragma unroll
    for (int q = 0; q < PACKS; ++q)
      az_store16((T*)(lds + (KC ? row(q) : red(q)) * PITCH) + (KC ? red(q) : row(q)), r[q]);
  }
  // the 16 rows from r0, 64 bytes of reduction from the q-th on: lane l has row l % 16, those at (l / 16) * 16 bytes
  __device__ static AzPack<T> fragment(const char* lds, int r0, int q, int lane) {
    if constexpr (KC) {
      return az_load16((const T*)(lds + (r0 + (lane & 15)) * PITCH + q * 64 + (lane >> 4) * 16));
    } else if constexpr (sizeof(T) == 4) {
      AzPack<T> x;
      const char* p = lds + (q * 16 + (lane >> 4) * 4) * PITCH + (r0 + (lane & 15)) * 4;
#pragma unroll
      for (int e = 0; e < 4; ++e) x.v[e] = *reinterpret_cast<const T*>(p + e * PITCH);
      return x;
    } else {
      // the transposing read hands lane i of 16 the i-th column of the four rows of 16 that the lanes point into
      const char* p = lds + (q * 32 + (lane >> 4) * 8 + ((lane >> 2) & 3)) * PITCH + (r0 + (lane & 3) * 4) * 2;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * PITCH));
      AzPack<T> x;
      __builtin_memcpy(&x, &lo, 8);
      __builtin_memcpy((char*)&x + 8, &hi, 8);
      return x;
    }
  }
};

// PLANES: of dz.
template <typename T, bool AKC, bool BKC, int EPI, int PLANES>
__global__ __launch_bounds__(256) void k_product_tile(Prod p) {
  typedef Stage<T, AKC> StageA;
  typedef Stage<T, BKC> StageB;
  constexpr int BK = StageA::BK;
  __shared__ alignas(16) char lds[2][StageA::BYTES + StageB::BYTES];
  const int m0 = (blockIdx.x % p.tiles_m) * TILE, n0 = (blockIdx.x / p.tiles_m) * TILE;
  const int k_begin = blockIdx.z * p.k_chunk, k_end = min(p.K, k_begin + p.k_chunk);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
  StageA sa;
  StageB sb;
  az_f32x4 acc[2][2] = {};
  int buf = 0;
  auto run = [&](const T* a, const T* b) {
    sa.load(a, p.lda, p.M, m0, k_begin, k_end);
    sb.load(b, p.ldb, p.N, n0, k_begin, k_end);
    for (int k = k_begin; k < k_end; k += BK, buf ^= 1) {
      char* la = lds[buf];
      char* lb = la + StageA::BYTES;
      sa.store(la);
      sb.store(lb);
      __syncthreads();   // (the other buffer's readers passed the barrier of the step before)
      if (k + BK < k_end) {
        sa.load(a, p.lda, p.M, m0, k + BK, k_end);
        sb.load(b, p.ldb, p.N, n0, k + BK, k_end);
      }
#pragma unroll
      for (int q = 0; q < PACKS; ++q) {
        if (k + q * (BK / PACKS) >= k_end) break;   // zeros from here on
        AzPack<T> fa[2], fb[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          fa[i] = StageA::fragment(la, wm + i * 16, q, lane);
          fb[i] = StageB::fragment(lb, wn + i * 16, q, lane);
        }
        // operands exchanged: a lane then holds four consecutive columns of one output row
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[i][j] = mma(fb[j], fa[i], acc[i][j]);
      }
    }
  };
  if constexpr (PLANES > 1) {
    run((const T*)p.a + p.a_plane, (const T*)p.b + p.b_plane);
    for (int i = 0; i < 2; ++i)
      for (int j = 0; j < 2; ++j) scale_low<T>(acc[i][j]);
  }
  run((const T*)p.a, (const T*)p.b);
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2; ++j) {
      const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
      finish<T, EPI>(p, m0 + wm + i * 16 + (lane & 15), n0 + wn + j * 16 + (lane >> 4) * 4, v);
    }
}

// ---------------------------------------------------------------------------
// Few outputs: 16 x 16 a workgroup, whose waves share the reduction (each takes every WAVES-th piece of 64 bytes) and
// whose sums are added in the waves' order.  One launch where splitting over workgroups needs two; operands go straight
// into registers, element by element where the reduction is not contiguous.
constexpr int WAVES = 16;

// Row r's elements k .. (WHOLE: all of them below K).
template <typename T, bool KC, bool WHOLE>
__device__ __forceinline__ AzPack<T> piece(const T* p, int64_t ld, int K, int r, int k) {
  constexpr int E = AzPack<T>::N;
  AzPack<T> x;
  if constexpr (KC && WHOLE) {
    __builtin_memcpy(&x, p + (int64_t)r * ld + k, 16);   // (at any address)
  } else {
    const T* at = p + (KC ? (int64_t)r * ld + k : (int64_t)k * ld + r);
#pragma unroll
    for (int e = 0; e < E; ++e) x.v[e] = WHOLE || k + e < K ? at[KC ? e : e * ld] : (T)0.0f;
  }
  return x;
}

// One workgroup's 16 x 16 outputs.  Rows and columns beyond the edge read the last one's operands and are not stored.
template <typename T, bool AKC, bool BKC, int EPI, int PLANES>
__device__ __forceinline__ void few_outputs(const Prod& p, int block, az_f32x4 (*sums)[64]) {
  constexpr int E = AzPack<T>::N;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m0 = (block % p.tiles_m) * 16, n0 = (block / p.tiles_m) * 16;
  const int m = min(m0 + (lane & 15), p.M - 1), n = min(n0 + (lane & 15), p.N - 1);
  az_f32x4 acc = {};
  auto run = [&](const T* pa, const T* pb) {
    int k = wave * 4 * E;
#pragma unroll 4
    for (; k + 4 * E <= p.K; k += WAVES * 4 * E) {
      const int at = k + (lane >> 4) * E;
      const AzPack<T> a = piece<T, AKC, true>(pa, p.lda, p.K, m, at);
      const AzPack<T> b = piece<T, BKC, true>(pb, p.ldb, p.K, n, at);
      acc = mma(b, a, acc);
    }
    if (k < p.K) {
      const int at = k + (lane >> 4) * E;
      const AzPack<T> a = piece<T, AKC, false>(pa, p.lda, p.K, m, at);
      const AzPack<T> b = piece<T, BKC, false>(pb, p.ldb, p.K, n, at);
      acc = mma(b, a, acc);
    }
  };
  if constexpr (PLANES > 1) {
    run((const T*)p.a + p.a_plane, (const T*)p.b + p.b_plane);
    scale_low<T>(acc);
  }
  run((const T*)p.a, (const T*)p.b);
  sums[wave][lane] = acc;
  __syncthreads();
  if (wave > 0) return;
  for (int w = 1; w < WAVES; ++w) acc += sums[w][lane];
  const float v[4] = {acc[0], acc[1], acc[2], acc[3]};
  finish<T, EPI>(p, m0 + (lane & 15), n0 + (lane >> 4) * 4, v);
}

template <typename T, bool AKC, bool BKC, int EPI, int PLANES>
__global__ __launch_bounds__(WAVES * 64) void k_product_few(Prod p) {
  __shared__ az_f32x4 sums[WAVES][64];
  few_outputs<T, AKC, BKC, EPI, PLANES>(p, blockIdx.x, sums);
}

// The bias' gradient from `chunks` rows of partial column sums, added in k_join's order: 64 columns a workgroup.
template <typename T>
__device__ __forceinline__ void join_columns(const float* part, int N, int chunks, T* out, int block, float (*sums)[64]) {
  const int c = threadIdx.x & 63, w = threadIdx.x >> 6, n = block * 64 + c;
  float s = 0.0f;
  if (n < N) {
#pragma unroll 4
    for (int i = w; i < chunks; i += WAVES) s += part[(int64_t)i * N + n];
  }
  sums[w][c] = s;
  __syncthreads();
  if (w > 0 || n >= N) return;
  for (int i = 1; i < WAVES; ++i) s += sums[i][c];
  out[n] = (T)s;
}

// All of a small layer's backward pass behind dz in one launch (each launch costs the host three microseconds): dx,
// then dkernel, then the bias' gradient.
template <typename T, int PLANES>
__global__ __launch_bounds__(WAVES * 64) void k_gradients_few(Prod dx, Prod dw, int dx_blocks, int dw_blocks,
                                                              const float* part, int chunks, T* dbias) {
  __shared__ az_f32x4 sums[WAVES][64];
  const int block = blockIdx.x;
  if (block < dx_blocks)
    few_outputs<T, true, true, EPI_STORE, PLANES>(dx, block, sums);
  else if (block < dx_blocks + dw_blocks)
    few_outputs<T, false, false, EPI_STORE, PLANES>(dw, block - dx_blocks, sums);
  else
    join_columns(part, dw.N, chunks, dbias, block - dx_blocks - dw_blocks, reinterpret_cast<float(*)[64]>(sums));
}

// ---------------------------------------------------------------------------
// Joins split sums in the order of the splits.  Segment 0 (the product; few splits, many outputs) takes the epilogue,
// 64 groups of four outputs a workgroup and its splits dealt to four threads; segment 1 (the bias' gradient; many
// splits, few outputs) is stored as it is, 16 groups a workgroup and 16 threads each.
struct Join {
  const float* part[2];
  int64_t length[2];
  int splits[2];
  void* out1;
  int64_t blocks0;
};

template <typename T, int EPI>
__global__ __launch_bounds__(256) void k_join(Join q, Prod p) {
  __shared__ float sums[256][4];
  const int seg = (int64_t)blockIdx.x >= q.blocks0;
  const int64_t L = q.length[seg];
  const int groups = seg ? 16 : 64, lanes = 256 / groups, g = threadIdx.x % groups, w = threadIdx.x / groups;
  const int64_t at = (((int64_t)blockIdx.x - (seg ? q.blocks0 : 0)) * groups + g) * 4;
  const int have = (int)max((int64_t)0, min((int64_t)4, L - at));
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (have > 0) {
    const float* part = q.part[seg] + at;
    if (L % 4 == 0) {
#pragma unroll 4
      for (int i = w; i < q.splits[seg]; i += lanes) {
        const float4 x = *reinterpret_cast<const float4*>(part + (int64_t)i * L);
        s[0] += x.x, s[1] += x.y, s[2] += x.z, s[3] += x.w;
      }
    } else {
#pragma unroll 4
      for (int i = w; i < q.splits[seg]; i += lanes)
        for (int e = 0; e < 4; ++e) s[e] += e < have ? part[(int64_t)i * L + e] : 0.0f;
    }
  }
  for (int e = 0; e < 4; ++e) sums[threadIdx.x][e] = s[e];
  __syncthreads();
  if (w != 0 || have == 0) return;
  for (int i = 1; i < lanes; ++i)
    for (int e = 0; e < 4; ++e) s[e] += sums[i * groups + g][e];
  if (seg) {
    for (int e = 0; e < have; ++e) ((T*)q.out1)[at + e] = (T)s[e];
  } else if (p.N % 4 == 0) {   // the group is in one row
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
// The three bfloat16 planes of a float32 value: each the rounding of what is left.  (A value that is not finite has
// no such planes; the wide kernel works its outputs out again.)
__device__ __forceinline__ void planes_of(float x, az_bf16* p) {
  p[0] = (az_bf16)x;
  x -= (float)p[0];
  p[1] = (az_bf16)x;
  x -= (float)p[1];
  p[2] = (az_bf16)x;
}

// dz = dy act'(z), rounded to T (and, for 16 bits, what that rounding leaves as a second plane), and the partial column sums of
// dz before the rounding: a workgroup takes 256 columns (four a thread) of a chunk of rows, four rows at a time.  Bound by
// memory: 16384 x 4096 bfloat16 97 us with both planes, 537 MB; 8192 x 256 float32 10 us.
struct Slope {
  const void* dy;
  const void* z;
  void* dz;            // may be null (no activation: dy itself is dz)
  az_bf16* planes;     // float32 only: dz as planes, may be null
  int64_t plane;       // elements from one plane to the next
  bool low;            // 16 bits only: the lo plane too, behind dz
  float* partial;      // [chunks][N], may be null
  int M, N, act, rows_per_chunk;
  int ld;              // of dz and the planes: columns N .. ld are set to zero
};

// EXACT: N and ld are multiples of four.
template <typename T, bool EXACT>
__global__ __launch_bounds__(256) void k_slope(Slope p) {
  typedef typename Kept<T>::type Z;
  constexpr int V = 4;
  __shared__ float sums[3][64][V];
  const int g = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int n = (blockIdx.x * 64 + g) * V;
  const int m_end = min(p.M, (int)(blockIdx.y + 1) * p.rows_per_chunk);
  const int have = min(V, p.N - n), room = p.dz || p.planes ? min(V, p.ld - n) : 0;   // columns to read, to write
  float s[V] = {};
  if (have > 0 || room > 0) {
#pragma unroll 2
    for (int m = blockIdx.y * p.rows_per_chunk + w; m < m_end; m += 4) {
      const int64_t at = (int64_t)m * p.N + n, to = (int64_t)m * p.ld + n;
      float d[V] = {}, z[V] = {};
      if (EXACT ? have > 0 : have == V) {
        const AzVec<T, V> dy = az_loadu<T, V>((const T*)p.dy + at);
        for (int i = 0; i < V; ++i) d[i] = (float)dy.v[i];
        if (p.act != AZ_ACT_NONE) {
          const AzVec<Z, V> k = az_loadu<Z, V>((const Z*)p.z + at);
          for (int i = 0; i < V; ++i) z[i] = (float)k.v[i];
        }
      } else if (!EXACT) {
        for (int i = 0; i < V; ++i)
          if (i < have) {
            d[i] = (float)((const T*)p.dy)[at + i];
            if (p.act != AZ_ACT_NONE) z[i] = (float)((const Z*)p.z)[at + i];
          }
      }
      if (p.act != AZ_ACT_NONE)
        for (int i = 0; i < V; ++i) d[i] = EXACT || i < have ? d[i] * act_slope(z[i], p.act) : 0.0f;
      for (int i = 0; i < V; ++i) s[i] += d[i];
      auto put = [&](auto* out, const auto& vec) {
        if (EXACT || room == V)
          az_storeu(out, vec);
        else
          for (int i = 0; i < V; ++i)
            if (i < room) out[i] = vec.v[i];
      };
      const AzVec<T, V> hi = {(T)d[0], (T)d[1], (T)d[2], (T)d[3]};
      if (p.dz) put((T*)p.dz + to, hi);
      if constexpr (sizeof(T) == 2) {
        if (p.low) {
          AzVec<T, V> lo;   // (exact but for its own rounding; 0 where dz or its rounding is not finite)
          for (int i = 0; i < V; ++i) {
            const float h = (float)hi.v[i];
            lo.v[i] = (T)(fabsf(h) < INFINITY ? (d[i] - h) * Low<T>::UP : 0.0f);
          }
          put((T*)p.dz + p.plane + to, lo);
        }
      } else {
        if (p.planes) {
          AzVec<az_bf16, V> o[3];
          for (int i = 0; i < V; ++i) {
            az_bf16 q[3];
            planes_of(d[i], q);
            for (int k = 0; k < 3; ++k) o[k].v[i] = q[k];
          }
          for (int k = 0; k < 3; ++k) put(p.planes + k * p.plane + to, o[k]);
        }
      }
    }
  }
  if (!p.partial) return;
  if (w > 0)
    for (int i = 0; i < V; ++i) sums[w - 1][g][i] = s[i];
  __syncthreads();
  if (w > 0) return;
  for (int i = 0; i < V; ++i)
    if (i < have)
      p.partial[(int64_t)blockIdx.y * p.N + n + i] = ((s[i] + sums[0][g][i]) + sums[1][g][i]) + sums[2][g][i];
}

// Copies an operand for the wide kernel: rows of `ld` elements, the last ones zero; float32 as planes.  Bound by memory:
// 8192 x 2048 float32 about 31 us, 168 MB.
template <typename T>
__global__ __launch_bounds__(256) void k_pack(const T* src, int rows, int cols, int ld, void* dst, int64_t plane) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per = ld / 8;
  if (i >= (int64_t)rows * per) return;
  const int64_t m = i / per;
  const int n = (int)(i % per) * 8;
  const T* from = src + m * cols + n;
  AzVec<T, 8> x;
  if (n + 8 <= cols) {
    x = az_loadu<T, 8>(from);
  } else {
    for (int e = 0; e < 8; ++e) x.v[e] = n + e < cols ? from[e] : (T)0.0f;
  }
  const int64_t to = m * ld + n;
  if constexpr (sizeof(T) == 4) {
    AzVec<az_bf16, 8> o[3];
    for (int e = 0; e < 8; ++e) {
      az_bf16 q[3];
      planes_of(x.v[e], q);
      for (int k = 0; k < 3; ++k) o[k].v[e] = q[k];
    }
    for (int k = 0; k < 3; ++k) az_storev<az_bf16, 8>((az_bf16*)dst + k * plane + to, o[k]);
  } else {
    az_storev<T, 8>((T*)dst + to, x);
  }
}

template <typename T>
__global__ void k_zero(T* p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) p[i] = (T)0.0f;
}

// ---------------------------------------------------------------------------
int size_of(int dtype) { return dtype == AZ_TYPE_F32 ? 4 : 2; }
int64_t round16(int64_t n) { return (n + 15) & ~(int64_t)15; }

// Chunks of rows that k_slope is dealt in: 2048 workgroups in all, 256 chunks at most (the join reads them), at least
// 16 rows each.
int slope_chunks(int64_t rows, int64_t col_tiles) {
  int64_t c = az_ceil(2048, col_tiles);
  if (c > 256) c = 256;
  const int64_t most = az_ceil(rows, 16);
  return (int)(c < most ? c : most);
}

int64_t round64(int64_t n) { return (n + 63) & ~(int64_t)63; }

// How one product C[M, N] over K runs.
struct Plan {
  bool wide, big, few;
  int splits;
};

// As many splits as bring `tiles` tiles to `want` workgroups, each at least `least` steps of the reduction long.
int64_t splits_for(int64_t tiles, int64_t want, int64_t K, int64_t least) {
  const int64_t s = az_ceil(want, tiles), most = K / least;
  return s < most ? s : most;
}

// Measured over layers of 64 to 16384 rows and 256 to 4096 columns, in microseconds (wide / 64 x 64 tiles):
//   16 bits: 4096 x 1024 x 1024 19 / 53, 64 x 1024 x 1024 9 / 9, 8192 x 256 x 256 10 / 10, 8 x 4096 x 4096 11 / 19; operands
//     that have to be copied first: 1003 x 401 x 517 23 / 19
//   float32: 4096 x 1024 x 1024 83 / 114, 1024 x 1024 x 1024 38 / 40, 256 x 2048 x 2048 43 / 38
// 256 x 256 tiles pay from one for each compute unit on: 16384 x 512 x 2048 59 against 62 with 128 x 128 (512 tiles),
// its dx 57 against 37 (128 tiles).  With fewer tiles they pay where the splits that fill the compute units stay long:
// dkernel of 16384 x 2048 x 2048 in bfloat16 125 (4 splits of 4096) against 149, of 8192 x 2048 x 2048 83 (4 of 2048)
// against 77; in float32, where every step is six, 389 against 436.
// Few outputs, up to 1024 tiles of 16 x 16, as long as the reduction is not too long for the waves of one workgroup, and for
// all of them together (k_product_few / the best other form; y reads its second operand element by element): 64 x 256 x 256
// float32 3.2 / 7.1, bfloat16 3.0 / 7.0, 512 x 512 x 512 float32 9.6 / 11.6, 256 x 1024 x 1024 bfloat16 y 9.1 / 11.5, dx 9.5 /
// 10.4, 200 x 1500 x 1100 y 13.8 / 19.3, float32 23.5 / 27.9, 8 x 4096 x 4096 bfloat16 dx 8.5 / 11.6 (two planes of dz 17.6 / 19.9,
// with dz); but 32 x 4096 x 4096 bfloat16 dx 17.1 / 13.7, 128 x 2048 x 2048 y 21 / 11, dx 17 / 9.8 (float32 33 / 21, 31 / 21), 64 x
// 4096 x 4096 dx 31 / 15 (two planes 64 / 25, float32 59 / 34).
// Up to 2560 tiles of 16-bit operands that the wide kernel would have to copy, if dx and dkernel are both so small: they then
// share one launch.  A backward pass that way / on 64 x 64 tiles, relu: 1003 x 401 x 517 32 / 39, 700 x 391 x 900 28 / 37,
// 1001 x 257 x 600 21 / 35, 2003 x 129 x 301 28 / 30, 611 x 333 x 999 32 / 42; swish 56 / 61, 46 / 58, 35 / 54, 42 / 46,
// 58 / 73.  With one product alone it does not pay: 1003 x 1003 x 403 50 / 40, 901 x 901 x 450 47 / 38, 515 x 515 x 1111 49 / 45,
// 1025 x 517 x 401 40 / 35, and for y 1001 x 257 x 600 16.1 / 13.0, 901 x 901 x 450 20.3 / 16.8, 2003 x 129 x 301 12.4 / 10.3,
// 1025 x 517 x 401 12.9 / 17.1.
bool small_pair(int dtype, int64_t M, int64_t N, int64_t K, bool in_place) {
  return dtype != AZ_TYPE_F32 && !in_place && az_ceil(M, 16) * az_ceil(N, 16) <= 2560 && K <= 1024;
}

// in_place: a 16-bit operand need not be copied for the wide kernel.  contiguous: operands with a contiguous reduction.
// pair: dx and dkernel are both small enough for the launch that they share.
Plan plan_of(int dtype, int64_t M, int64_t N, int64_t K, bool in_place, int contiguous, bool pair = false) {
  Plan p = {};
  const double work = (double)M * N * K;
  const bool f32 = dtype == AZ_TYPE_F32;
  const int64_t pieces = az_ceil(M, 16) * az_ceil(N, 16);
  p.few = pair || (pieces <= 1024 && pieces * K <= 0x180000 &&
                   K <= (contiguous == 2 ? 4096 : contiguous == 1 ? (f32 ? 4096 : 2048) : 1024));
  p.wide = !p.few && work >= (f32 ? 0x1p31 : in_place ? 0x1p25 : 0x1p29);
  int64_t s = 1;
  if (!p.few && !p.wide) {
    // two workgroups a compute unit for a long reduction, one otherwise, of two steps at least; a few tiles are split
    // further
    const int64_t tiles = az_ceil(M, TILE) * az_ceil(N, TILE);
    s = splits_for(tiles, K >= 1024 ? 512 : 256, K, tiles <= 16 ? 32 : f32 ? 128 : 256);
  } else if (p.wide) {
    const int64_t large = az_ceil(M, 256) * az_ceil(N, 256), steps = f32 ? 6 * K : K;
    const int64_t share = 256 / large;   // splits that give each compute unit a large tile
    p.big = large >= 256 || (share >= 1 && large * share >= 192 && steps / share >= 4096);
    if (p.big) {
      s = large >= 256 ? 1 : share;
    } else {
      const int64_t tiles = az_ceil(M, 128) * az_ceil(N, 128);
      const int64_t one = splits_for(tiles, 256, steps, 512), two = splits_for(tiles, 512, steps, 2048);
      s = one > two ? one : two;
      if (s > K / 64) s = K / 64;
    }
  }
  p.splits = (int)(s < 1 ? 1 : s > 64 ? 64 : s);
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

// The tiles of a product; their number.
int64_t prepare(Prod& p, int tile) {
  p.tiles_m = (int)az_ceil(p.M, tile), p.tiles_n = (int)az_ceil(p.N, tile);
  return (int64_t)p.tiles_m * p.tiles_n;
}

// One product (and, with `extra`, the join of the bias' gradient).  `partial` holds splits x M x N floats.
template <typename T, bool AKC, bool BKC, int EPI>
int product(Prod p, const Plan& plan, float* partial, const Join* extra, hipStream_t stream) {
  const int pass = EPI == EPI_FORWARD ? PASS_Y : AKC ? PASS_DX : PASS_DW;
  const int dtype = sizeof(T) == 4 ? AZ_TYPE_F32 : std::is_same_v<T, az_bf16> ? AZ_TYPE_BF16 : AZ_TYPE_F16;
  const int64_t tiles = prepare(p, plan.wide ? (plan.big ? 256 : 128) : plan.few ? 16 : TILE);
  if (!az_grid_fits(tiles, plan.few ? WAVES * 64 : 512) || !az_grid_fits(az_ceil((int64_t)p.M * p.N, 256), 256))
    return az_fail(AZ_ERR_UNSUPPORTED, "dense: %d x %d outputs are too many for one launch", p.M, p.N);
  const int step = plan.wide ? 64 : Stage<T, true>::BK;
  p.k_chunk = (int)(az_ceil(az_ceil(p.K, plan.splits), step) * step);
  const int splits = (int)az_ceil(p.K, p.k_chunk);
  Prod q = p;
  if (splits > 1) q.partial = partial;
  auto run = [&]<int PLANES>() {
    if (plan.few) {
      k_product_few<T, AKC, BKC, EPI, PLANES><<<dim3((unsigned)tiles), dim3(WAVES * 64), 0, stream>>>(q);
    } else {
      const dim3 grid((unsigned)tiles, 1, splits), block(256);
      if (splits == 1)
        k_product_tile<T, AKC, BKC, EPI, PLANES><<<grid, block, 0, stream>>>(q);
      else
        k_product_tile<T, AKC, BKC, EPI_PARTIAL, PLANES><<<grid, block, 0, stream>>>(q);
    }
  };
  if (plan.wide) {
    if (int rc = az_product_wide(dtype, pass, splits > 1, plan.big, &q, splits, stream)) return rc;
  } else {
    bool two = false;
    if constexpr (sizeof(T) == 2 && EPI == EPI_STORE) {
      two = p.planes > 1;
      if (two) run.template operator()<2>();
    }
    if (!two) run.template operator()<1>();
    AZ_LAUNCH_CHECK();
  }
  if (splits > 1 || extra) {
    Join j = extra ? *extra : Join{};
    if (splits > 1) {
      j.part[0] = partial, j.length[0] = (int64_t)p.M * p.N, j.splits[0] = splits;
      j.blocks0 = az_ceil(j.length[0], 256);
    }
    const int64_t blocks = j.blocks0 + az_ceil(j.length[1], 64);
    k_join<T, EPI><<<dim3((unsigned)blocks), dim3(256), 0, stream>>>(j, p);
    AZ_LAUNCH_CHECK();
  }
  return AZ_OK;
}

// A pass' plans and its workspace: copies of the operands for the wide kernel where it cannot read them in place
// (always room for them), dz, the partial sums of the bias' gradient, the partial sums of a split product.
struct Layout {
  Plan y, dx, dw;
  int chunks;
  int64_t x, kernel, dz, dz_planes, bias, partial, total;
};

Layout layout_of(int dtype, int64_t M, int64_t K, int64_t N, int pass) {
  Layout l = {};
  const int64_t Kp = round64(K), Np = round64(N), each = dtype == AZ_TYPE_F32 ? 6 : 2;
  int64_t at = 0;
  auto room = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) & ~(int64_t)255;
    return here;
  };
  if (pass == 0) {
    l.y = plan_of(dtype, M, N, K, K % 64 == 0 && N % 8 == 0, 1);
    if (l.y.wide) l.x = room(M * Kp * each), l.kernel = room(K * Np * each);
    if (l.y.splits > 1) l.partial = room(l.y.splits * M * N * 4);
  } else {
    const bool dx_in_place = N % 64 == 0, dw_in_place = K % 8 == 0 && N % 8 == 0;
    l.dx = plan_of(dtype, M, K, N, dx_in_place, 2), l.dw = plan_of(dtype, K, N, M, dw_in_place, 0);
    const bool small_dx = small_pair(dtype, M, K, N, dx_in_place), small_dw = small_pair(dtype, K, N, M, dw_in_place);
    if ((l.dx.few || small_dx) && (l.dw.few || small_dw))
      l.dx = plan_of(dtype, M, K, N, dx_in_place, 2, true), l.dw = plan_of(dtype, K, N, M, dw_in_place, 0, true);
    l.chunks = slope_chunks(M, az_ceil(N, 256));
    l.dz = room(M * Np * 4);   // float32, or two planes of 16 bits
    if (dtype == AZ_TYPE_F32 && (l.dx.wide || l.dw.wide)) l.dz_planes = room(M * Np * 6);
    l.bias = room((int64_t)l.chunks * N * 4);
    if (l.dw.wide) l.x = room(M * Kp * each);
    if (l.dx.wide) l.kernel = room(K * Np * each);
    const int64_t a = l.dx.splits > 1 ? l.dx.splits * M * K : 0, b = l.dw.splits > 1 ? l.dw.splits * K * N : 0;
    l.partial = room(4 * (a > b ? a : b));
  }
  l.total = at;
  return l;
}

// An operand [rows, cols] as the wide kernel reads it: in place, or copied to `to` (float32 always: planes).
// along: its rows are the reduction's axis and have to be whole steps long.  plane: elements between its planes, 0 for one.
struct Source {
  const void* p;
  int64_t ld, plane;
};

template <typename T>
int source(const void* src, int64_t rows, int64_t cols, bool along, void* to, hipStream_t stream, Source* out) {
  if (sizeof(T) == 2 && az_aligned16(src) && cols % (along ? 64 : 8) == 0) {
    *out = {src, cols, 0};
    return AZ_OK;
  }
  const int64_t ld = round64(cols), threads = rows * (ld / 8);
  if (!az_grid_fits(az_ceil(threads, 256), 256)) return az_fail(AZ_ERR_UNSUPPORTED, "dense: operand too large");
  *out = {to, ld, sizeof(T) == 4 ? rows * ld : 0};
  k_pack<T><<<dim3((unsigned)az_ceil(threads, 256)), dim3(256), 0, stream>>>((const T*)src, (int)rows, (int)cols,
                                                                             (int)ld, to, rows * ld);
  AZ_LAUNCH_CHECK();
  return AZ_OK;
}

void operand_a(Prod& p, const Source& s, const void* raw, int64_t ld) {
  p.a = s.p, p.lda = s.ld, p.a_plane = s.plane, p.a32 = (const float*)raw, p.lda32 = ld;
}
void operand_b(Prod& p, const Source& s, const void* raw, int64_t ld) {
  p.b = s.p, p.ldb = s.ld, p.b_plane = s.plane, p.b32 = (const float*)raw, p.ldb32 = ld;
}

}  // namespace

extern "C" int64_t az_dense_workspace_bytes(int32_t dtype, int32_t rows, int32_t fan_in, int32_t fan_out,
                                            int32_t pass) {
  if (check(dtype, AZ_ACT_NONE, rows, fan_in, fan_out) != AZ_OK || pass < 0 || pass > 1) return -1;
  return rows == 0 ? 0 : layout_of(dtype, rows, fan_in, fan_out, pass).total;
}

extern "C" int az_dense_forward(int32_t dtype, int32_t act, int32_t rows, int32_t fan_in, int32_t fan_out,
                                const void* x, const void* kernel, const void* bias, const void* residual, void* y,
                                void* z, void* workspace, int64_t workspace_bytes, void* stream_) {
  if (int rc = check(dtype, act, rows, fan_in, fan_out)) return rc;
  if (rows == 0) return AZ_OK;
  if (!x || !kernel || !y) return az_fail(AZ_ERR_INVALID, "dense: null x, kernel or y");
  const Layout l = layout_of(dtype, rows, fan_in, fan_out, 0);
  if (workspace_bytes < l.total || (l.total && (!workspace || !az_aligned16(workspace))))
    return az_fail(AZ_ERR_INVALID, "dense: the workspace must hold %lld bytes, 16-byte aligned", (long long)l.total);
  hipStream_t stream = (hipStream_t)stream_;
  char* ws = (char*)workspace;
  return az_dispatch_type(dtype, [&]<typename T>() -> int {
    Prod p = {};
    Source sx = {x, fan_in, 0}, sk = {kernel, fan_out, 0};
    if (l.y.wide) {
      if (int rc = source<T>(x, rows, fan_in, true, ws + l.x, stream, &sx)) return rc;
      if (int rc = source<T>(kernel, fan_in, fan_out, false, ws + l.kernel, stream, &sk)) return rc;
    }
    operand_a(p, sx, x, fan_in);
    operand_b(p, sk, kernel, fan_out);
    p.M = rows, p.N = fan_out, p.K = fan_in, p.planes = 1;
    p.act = act, p.bias = bias, p.residual = residual, p.z = act == AZ_ACT_NONE ? nullptr : z, p.out = y;
    return product<T, true, false, EPI_FORWARD>(p, l.y, (float*)(ws + l.partial), nullptr, stream);
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
      if (dkernel) k_zero<T><<<dim3((unsigned)(n < 1 << 20 ? az_ceil(n, 256) : 4096)), dim3(256), 0, stream>>>((T*)dkernel, n);
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
    const bool wide_dx = dx && l.dx.wide, wide_dw = dkernel && l.dw.wide, wide = wide_dx || wide_dw;
    // dz: dy itself, or written by k_slope (padded for the wide kernel: it reduces along dz's rows for dx), for
    // float32 also or only as planes
    const int64_t ld = wide ? round64(fan_out) : fan_out;
    constexpr bool F32 = sizeof(T) == 4;
    const bool copy = act != AZ_ACT_NONE ||
                      (wide && !F32 && (!az_aligned16(dy) || fan_out % 8 || (wide_dx && fan_out % 64)));
    // (without an activation or with relu, whose slope is 0 or 1, dz has the 16 bits of dy)
    const bool low = !F32 && act != AZ_ACT_NONE && act != AZ_ACT_RELU;
    Source sdz = {dy, fan_out, 0}, sdzw = sdz;
    if (copy) sdz = sdzw = {ws + l.dz, ld, low ? rows * ld : 0};
    if (F32 && wide) sdzw = {ws + l.dz_planes, ld, rows * ld};
    if (copy || dbias || (F32 && wide)) {
      Slope s = {};
      s.dy = dy, s.z = z, s.dz = copy ? ws + l.dz : nullptr, s.plane = rows * ld, s.low = low;
      if (F32 && wide) s.planes = (az_bf16*)(ws + l.dz_planes);
      s.partial = dbias ? (float*)(ws + l.bias) : nullptr;
      s.M = rows, s.N = fan_out, s.act = act, s.rows_per_chunk = (int)az_ceil(rows, l.chunks), s.ld = (int)ld;
      const dim3 grid((unsigned)az_ceil(ld, 256), l.chunks);
      if (fan_out % 4 == 0)
        k_slope<T, true><<<grid, dim3(256), 0, stream>>>(s);
      else
        k_slope<T, false><<<grid, dim3(256), 0, stream>>>(s);
      AZ_LAUNCH_CHECK();
    }
    // (the float32 operands of an output that the planes leave not finite)
    const void* dz32 = copy ? ws + l.dz : dy;
    const int64_t ld32 = copy ? ld : fan_out;
    float* partial = (float*)(ws + l.partial);
    if (dx && dkernel && l.dx.few && l.dw.few) {
      Prod px = {}, pw = {};
      operand_a(px, sdz, nullptr, 0);
      operand_b(px, Source{kernel, fan_out, 0}, nullptr, 0);
      px.M = rows, px.N = fan_in, px.K = fan_out, px.out = dx;
      operand_a(pw, Source{x, fan_in, 0}, nullptr, 0);
      operand_b(pw, sdz, nullptr, 0);
      pw.M = fan_in, pw.N = fan_out, pw.K = rows, pw.out = dkernel;
      const int64_t nx = prepare(px, 16), nw = prepare(pw, 16);
      const int64_t nb = dbias ? az_ceil(fan_out, 64) : 0;
      if (!az_grid_fits(nx + nw + nb, WAVES * 64)) return az_fail(AZ_ERR_UNSUPPORTED, "dense: too many outputs");
      auto run = [&]<int PLANES>() {
        k_gradients_few<T, PLANES><<<dim3((unsigned)(nx + nw + nb)), dim3(WAVES * 64), 0, stream>>>(
            px, pw, (int)nx, (int)nw, (const float*)(ws + l.bias), l.chunks, (T*)dbias);
      };
      if constexpr (F32)
        run.template operator()<1>();
      else if (low)
        run.template operator()<2>();
      else
        run.template operator()<1>();
      AZ_LAUNCH_CHECK();
      return AZ_OK;
    }
    if (dx) {
      Prod p = {};
      Source sk = {kernel, fan_out, 0};
      if (wide_dx)
        if (int rc = source<T>(kernel, fan_in, fan_out, true, ws + l.kernel, stream, &sk)) return rc;
      operand_a(p, wide_dx ? sdzw : sdz, dz32, ld32);
      operand_b(p, sk, kernel, fan_out);
      p.M = rows, p.N = fan_in, p.K = fan_out, p.out = dx, p.planes = 1 + low;
      if (int rc = product<T, true, true, EPI_STORE>(p, l.dx, partial, nullptr, stream)) return rc;
    }
    Join j = {};
    j.part[1] = (const float*)(ws + l.bias), j.length[1] = fan_out, j.splits[1] = l.chunks, j.out1 = dbias;
    if (dkernel) {
      Prod p = {};
      Source sx = {x, fan_in, 0};
      if (wide_dw)
        if (int rc = source<T>(x, rows, fan_in, false, ws + l.x, stream, &sx)) return rc;
      operand_a(p, sx, x, fan_in);
      operand_b(p, wide_dw ? sdzw : sdz, dz32, ld32);
      p.M = fan_in, p.N = fan_out, p.K = rows, p.out = dkernel, p.planes = 1 + low;
      return product<T, false, false, EPI_STORE>(p, l.dw, partial, dbias ? &j : nullptr, stream);
    }
    if (dbias) {
      k_join<T, EPI_STORE><<<dim3((unsigned)az_ceil(fan_out, 64)), dim3(256), 0, stream>>>(j, Prod{});
      AZ_LAUNCH_CHECK();
    }
    return AZ_OK;
  });
}
