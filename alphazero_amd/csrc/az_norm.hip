// az_norm.hip -- layer norm over the last axis and its backward pass (include/az_layers.h).
// Part of libaz_mcts.so (gfx950 only).
//
// Bound by memory: the forward pass reads x and writes y once, the backward pass reads x and dy and writes dx once.
// A row stays in the registers of NT threads between its sums and its outputs, so the variance is taken from the
// differences to the mean (no cancellation), and the backward pass adds its row's share of the scale's and bias'
// gradients to registers that a thread keeps for its columns over all rows of its workgroup.  Up to 1024 columns a wave
// takes a row, up to 4096 four waves, up to 16384 sixteen: 16 elements a thread, what leaves room for the two gradients.
// Odd widths are read 16 bytes at a time all the same (gfx950 loads at any address), the row's last piece by elements.
// 16384 x 4096 bfloat16: forward 58-63 us (268 MB), backward 80 us (402 MB), a large copy 5.2 TB/s; 8191 x 1001
// float32: 14 and 21 us (66 and 98 MB), with 4 us for the join.
#include <hip/hip_runtime.h>

#include "az_host.h"
#include "az_types.h"

namespace {

struct Norm {
  const void* x;
  const void* scale;
  const void* bias;
  const void* dy;
  void* out;            // y or dx
  float* mean;
  float* rstd;
  float* partial;       // [blocks][2][width]: scale's, bias' gradient
  float eps;
  int rows, width;
};

// V elements of a row from column c as they are, 0 beyond its end.  EXACT: the width is a multiple of V; the load
// is then made by every thread, without a branch (behind which the compiler would wait for it).
template <typename T, int V, bool EXACT>
__device__ __forceinline__ AzVec<T, V> fetch_row(const T* row, int c, int width) {
  AzVec<T, V> r;
  if constexpr (EXACT) {
    r = az_loadu<T, V>(row + (c < width ? c : 0));
    for (int i = 0; i < V; ++i) r.v[i] = c < width ? r.v[i] : (T)0.0f;
  } else if (c + V <= width) {
    r = az_loadu<T, V>(row + c);
  } else {
    for (int i = 0; i < V; ++i) r.v[i] = c + i < width ? row[c + i] : (T)0.0f;
  }
  return r;
}

template <typename T, int V, bool EXACT>
__device__ __forceinline__ void load_row(const T* row, int c, int width, float* v) {
  const AzVec<T, V> r = fetch_row<T, V, EXACT>(row, c, width);
  for (int i = 0; i < V; ++i) v[i] = (float)r.v[i];
}

template <typename T, int V>
__device__ __forceinline__ void store_row(T* row, int c, int width, const float* v) {
  if (c + V <= width) {
    AzVec<T, V> r;
    for (int i = 0; i < V; ++i) r.v[i] = (T)v[i];
    az_storeu<T, V>(row + c, r);
  } else {
    for (int i = 0; i < V; ++i)
      if (c + i < width) row[c + i] = (T)v[i];
  }
}

// Sum over the NT threads of a row, the same in each of them.  `scratch` holds NT / 64 floats and may be used again
// after the next barrier.
template <int NT>
__device__ __forceinline__ float row_sum(float s, float* scratch) {
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
  if constexpr (NT > 64) {
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.0f;
    for (int i = 0; i < NT / 64; ++i) s += scratch[i];
  }
  return s;
}

template <typename T>
constexpr int vec_of() {
  return 16 / sizeof(T);
}

// NT threads a row, R 16-byte loads a thread; workgroups of max(NT, 256) threads.
template <typename T, typename P, int NT, int R, bool EXACT>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void k_norm_forward(Norm p) {
  constexpr int V = vec_of<T>(), ROWS = NT < 256 ? 256 / NT : 1;
  __shared__ float scratch[2][NT / 64];   // (each is written again behind the other's barrier)
  const int t = threadIdx.x % NT;
  for (int64_t m = (int64_t)blockIdx.x * ROWS + threadIdx.x / NT; m < p.rows; m += (int64_t)gridDim.x * ROWS) {
    const T* x = (const T*)p.x + m * p.width;
    float v[R][V];
    float s = 0.0f;
    for (int r = 0; r < R; ++r) {
      load_row<T, V, EXACT>(x, (r * NT + t) * V, p.width, v[r]);
      for (int i = 0; i < V; ++i) s += v[r][i];
    }
    const float mean = row_sum<NT>(s, scratch[0]) / p.width;
    s = 0.0f;
    for (int r = 0; r < R; ++r)
      for (int i = 0; i < V; ++i) {
        v[r][i] -= mean;
        if ((r * NT + t) * V + i < p.width) s += v[r][i] * v[r][i];
      }
    const float rstd = 1.0f / sqrtf(row_sum<NT>(s, scratch[1]) / p.width + p.eps);
    T* y = (T*)p.out + m * p.width;
    for (int r = 0; r < R; ++r) {
      const int c = (r * NT + t) * V;
      float g[V], b[V];
      if (p.scale) load_row<P, V, EXACT>((const P*)p.scale, c, p.width, g);
      if (p.bias) load_row<P, V, EXACT>((const P*)p.bias, c, p.width, b);
      for (int i = 0; i < V; ++i) {
        float o = v[r][i] * rstd;
        if (p.scale) o *= g[i];
        if (p.bias) o += b[i];
        v[r][i] = o;
      }
      store_row<T, V>(y, c, p.width, v[r]);
    }
    if (t == 0 && p.mean) p.mean[m] = mean, p.rstd[m] = rstd;
  }
}

// A row's x and dy are loaded while the row before is worked on (not with 1024 threads a row, which have 128 registers
// each).  16384 x 4096 bfloat16: 80 us, 402 MB; 138 us while the loads waited for each other and for the barriers.
template <typename T, typename P, int NT, int R, bool EXACT>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void k_norm_backward(Norm p) {
  constexpr int V = vec_of<T>(), ROWS = NT < 256 ? 256 / NT : 1, W = NT * V * R;
  __shared__ float scratch[2][2 * (NT / 64)];
  __shared__ float joined[ROWS > 1 ? 2 * W : 1];
  const int t = threadIdx.x % NT, g = threadIdx.x / NT;
  float ds[R][V] = {}, db[R][V] = {};
  AzVec<P, V> gain[R];
  for (int r = 0; r < R; ++r) {
    if (p.scale)
      gain[r] = fetch_row<P, V, EXACT>((const P*)p.scale, (r * NT + t) * V, p.width);
    else
      for (int i = 0; i < V; ++i) gain[r].v[i] = (P)1.0f;
  }
  AzVec<T, V> next_x[R], next_h[R];
  float next_mean = 0.0f, next_rstd = 0.0f;
  auto fetch = [&](int m) {
    m = min(m, p.rows - 1);   // (beyond the last row: loaded, not used)
    const int64_t at = (int64_t)m * p.width;
    next_mean = p.mean[m], next_rstd = p.rstd[m];
    for (int r = 0; r < R; ++r) {
      next_x[r] = fetch_row<T, V, EXACT>((const T*)p.x + at, (r * NT + t) * V, p.width);
      next_h[r] = fetch_row<T, V, EXACT>((const T*)p.dy + at, (r * NT + t) * V, p.width);
    }
  };
  constexpr bool AHEAD = NT < 1024;
  const int stride = gridDim.x * ROWS;
  int phase = 0;
  if (AHEAD) fetch(blockIdx.x * ROWS + g);
  for (int64_t m64 = blockIdx.x * ROWS + g; m64 < p.rows; m64 += stride, phase ^= 1) {
    const int m = (int)m64;
    if (!AHEAD) fetch(m);
    const float mean = next_mean, rstd = next_rstd;
    float x[R][V], h[R][V], s1 = 0.0f, s2 = 0.0f;
    for (int r = 0; r < R; ++r)
      for (int i = 0; i < V; ++i) x[r][i] = (float)next_x[r].v[i], h[r][i] = (float)next_h[r].v[i];
    if (AHEAD) fetch(m + stride);
    for (int r = 0; r < R; ++r)
      for (int i = 0; i < V; ++i) {
        x[r][i] = (x[r][i] - mean) * rstd;
        ds[r][i] += h[r][i] * x[r][i];
        db[r][i] += h[r][i];
        h[r][i] *= (float)gain[r].v[i];
        s1 += h[r][i];          // (beyond the row's end h is 0)
        s2 += h[r][i] * x[r][i];
      }
    if (!p.out) continue;
    for (int off = 32; off > 0; off >>= 1) s1 += __shfl_xor(s1, off), s2 += __shfl_xor(s2, off);
    if constexpr (NT > 64) {
      // (two scratches in turn: one is written again only behind the other's barrier)
      if ((t & 63) == 0) scratch[phase][2 * (t >> 6)] = s1, scratch[phase][2 * (t >> 6) + 1] = s2;
      az_lds_barrier();
      s1 = s2 = 0.0f;
      for (int i = 0; i < NT / 64; ++i) s1 += scratch[phase][2 * i], s2 += scratch[phase][2 * i + 1];
    }
    s1 /= p.width, s2 /= p.width;
    const int64_t at = (int64_t)m * p.width;
    for (int r = 0; r < R; ++r) {
      for (int i = 0; i < V; ++i) h[r][i] = rstd * (h[r][i] - s1 - x[r][i] * s2);
      store_row<T, V>((T*)p.out + at, (r * NT + t) * V, p.width, h[r]);
    }
  }
  if (!p.partial) return;
  if constexpr (ROWS > 1) {   // the workgroup's rows, in their order
    for (int k = 0; k < ROWS; ++k) {
      if (g == k)
        for (int r = 0; r < R; ++r)
          for (int i = 0; i < V; ++i) {
            const int c = (r * NT + t) * V + i;
            joined[c] = k ? joined[c] + ds[r][i] : ds[r][i];
            joined[W + c] = k ? joined[W + c] + db[r][i] : db[r][i];
          }
      __syncthreads();
    }
    float* out = p.partial + (int64_t)blockIdx.x * 2 * p.width;
    for (int c = threadIdx.x; c < p.width; c += ROWS * NT) out[c] = joined[c], out[p.width + c] = joined[W + c];
  } else {
    float* out = p.partial + (int64_t)blockIdx.x * 2 * p.width;
    for (int r = 0; r < R; ++r) {
      store_row<float, V>(out, (r * NT + t) * V, p.width, ds[r]);
      store_row<float, V>(out + p.width, (r * NT + t) * V, p.width, db[r]);
    }
  }
}

// Rows too wide for the registers: a workgroup a row, which it reads again from L2 for each sum.  3000 x 20000 float32: 223 us,
// backward 260 and the columns 100 (480 and 720 MB at least: 93 and 139 us at a large copy's rate).
template <typename T, typename P>
__global__ __launch_bounds__(1024) void k_norm_forward_wide(Norm p) {
  __shared__ float scratch[2][16];
  for (int64_t m = blockIdx.x; m < p.rows; m += gridDim.x) {
    const int64_t at = m * p.width;
    const T* x = (const T*)p.x + at;
    float s = 0.0f;
    for (int c = threadIdx.x; c < p.width; c += 1024) s += (float)x[c];
    const float mean = row_sum<1024>(s, scratch[0]) / p.width;
    s = 0.0f;
    for (int c = threadIdx.x; c < p.width; c += 1024) {
      const float d = (float)x[c] - mean;
      s += d * d;
    }
    const float rstd = 1.0f / sqrtf(row_sum<1024>(s, scratch[1]) / p.width + p.eps);
    for (int c = threadIdx.x; c < p.width; c += 1024) {
      float o = ((float)x[c] - mean) * rstd;
      if (p.scale) o *= (float)((const P*)p.scale)[c];
      if (p.bias) o += (float)((const P*)p.bias)[c];
      ((T*)p.out)[at + c] = (T)o;
    }
    if (threadIdx.x == 0 && p.mean) p.mean[m] = mean, p.rstd[m] = rstd;
  }
}

template <typename T, typename P>
__global__ __launch_bounds__(1024) void k_norm_backward_wide(Norm p) {
  __shared__ float scratch[2][16];
  for (int64_t m = blockIdx.x; m < p.rows; m += gridDim.x) {
    const int64_t at = m * p.width;
    const float mean = p.mean[m], rstd = p.rstd[m];
    auto h_of = [&](int c) {
      const float d = (float)((const T*)p.dy)[at + c];
      return p.scale ? d * (float)((const P*)p.scale)[c] : d;
    };
    auto x_of = [&](int c) { return ((float)((const T*)p.x)[at + c] - mean) * rstd; };
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = threadIdx.x; c < p.width; c += 1024) {
      const float h = h_of(c);
      s1 += h;
      s2 += h * x_of(c);
    }
    s1 = row_sum<1024>(s1, scratch[0]) / p.width;
    s2 = row_sum<1024>(s2, scratch[1]) / p.width;
    for (int c = threadIdx.x; c < p.width; c += 1024)
      ((T*)p.out)[at + c] = (T)(rstd * (h_of(c) - s1 - x_of(c) * s2));
  }
}

template <typename T>
__global__ __launch_bounds__(256) void k_norm_columns_wide(Norm p) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= p.width) return;
  float ds = 0.0f, db = 0.0f;
  for (int m = blockIdx.y; m < p.rows; m += gridDim.y) {
    const int64_t at = (int64_t)m * p.width + c;
    const float d = (float)((const T*)p.dy)[at];
    ds += d * (((float)((const T*)p.x)[at] - p.mean[m]) * p.rstd[m]);
    db += d;
  }
  p.partial[(int64_t)blockIdx.y * 2 * p.width + c] = ds;
  p.partial[(int64_t)blockIdx.y * 2 * p.width + p.width + c] = db;
}

// Column sums of the workgroups' partial gradients, in their order: 64 columns a workgroup, 16 threads a column.
template <typename P>
__global__ __launch_bounds__(1024) void k_norm_join(const float* partial, int blocks, int width, P* dscale, P* dbias) {
  __shared__ float sums[16][64];
  const int which = blockIdx.y, g = threadIdx.x & 63, w = threadIdx.x >> 6;
  P* out = which ? dbias : dscale;
  if (!out) return;
  const int c = blockIdx.x * 64 + g;
  float s = 0.0f;
  if (c < width) {
#pragma unroll 8
    for (int i = w; i < blocks; i += 16) s += partial[((int64_t)i * 2 + which) * width + c];
  }
  sums[w][g] = s;
  __syncthreads();
  if (w != 0 || c >= width) return;
  s = 0.0f;
  for (int i = 0; i < 16; ++i) s += sums[i][g];
  out[c] = (P)s;
}

template <typename P>
__global__ void k_norm_zero(P* a, P* b, int n) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  if (a) a[i] = (P)0.0f;
  if (b) b[i] = (P)0.0f;
}

// ---------------------------------------------------------------------------
constexpr int IN_REGISTERS = 16384;   // widest row of the register form: 1024 threads x 16 elements

// Threads a row, in microseconds (forward, backward): a wave / four waves 16384 x 1024 float32 24, 38 / 27, 45, bfloat16 16, 26 /
// 35, 53, 16384 x 512 float32 15, 23 / 26, 42 (64 x 1024 4.4, 7.4 / 3.9, 8.4); four waves / sixteen 8192 x 4096 float32 43, 82 /
// 104, 105, bfloat16 27, 40 / 94, 79, 64 x 4096 4.6, 8.2 / 5.2, 11.
int threads_of(int width) { return width <= 1024 ? 64 : width <= 4096 ? 256 : 1024; }

// Workgroups of a forward pass: one a row (or four rows) as long as a launch holds them, then they go on to further rows.
int64_t few(int64_t blocks) { return blocks < (1 << 20) ? blocks : 1 << 20; }

// Workgroups of the backward pass, each of which leaves a row of partial column sums.
int backward_blocks(int64_t rows, int width) {
  const int64_t per = width <= 1024 ? 4 : 1, most = width <= 4096 ? 512 : 256;
  const int64_t n = az_ceil(rows, per);
  return (int)(n < most ? n : most);
}

// Calls f.operator()<NT, R, EXACT>() for the row's threads and loads.
template <typename T, typename P, typename F>
void with_shape(int width, F&& f) {
  constexpr int V = vec_of<T>(), FULL = 16 / V;   // 16 elements a thread
  const int nt = threads_of(width);
  auto with = [&]<int NT, int R>() {
    if (width % V == 0)
      f.template operator()<NT, R, true>();
    else
      f.template operator()<NT, R, false>();
  };
  if (nt == 64) {
    if (width <= 64 * V) return with.template operator()<64, 1>();
    if constexpr (FULL > 2)
      if (width <= 128 * V) return with.template operator()<64, 2>();
    return with.template operator()<64, FULL>();
  }
  if (nt == 256) {
    if (width <= 256 * 2 * V && FULL > 2) return with.template operator()<256, 2>();
    return with.template operator()<256, FULL>();
  }
  return with.template operator()<1024, FULL>();
}

int check(int dtype, int param_dtype, int64_t rows, int64_t width) {
  if (dtype < AZ_TYPE_F32 || dtype > AZ_TYPE_F16 || (param_dtype != dtype && param_dtype != AZ_TYPE_F32))
    return az_fail(AZ_ERR_INVALID, "layer norm: types %d and %d", dtype, param_dtype);
  if (rows < 0 || width < 1)
    return az_fail(AZ_ERR_INVALID, "layer norm: rows=%lld width=%lld", (long long)rows, (long long)width);
  if (rows > 0x7fff0000 || width > AZ_NORM_MAX_WIDTH)
    return az_fail(AZ_ERR_UNSUPPORTED, "layer norm: rows up to %d, width up to %d", 0x7fff0000, AZ_NORM_MAX_WIDTH);
  return AZ_OK;
}

template <typename F>
int with_types(int dtype, int param_dtype, F&& f) {
  return az_dispatch_type(dtype, [&]<typename T>() -> int {
    if (param_dtype == AZ_TYPE_F32) return f.template operator()<T, float>();
    return f.template operator()<T, T>();
  });
}

}  // namespace

extern "C" int az_layer_norm_forward(int32_t dtype, int32_t param_dtype, int32_t rows, int32_t width, const void* x,
                                     const void* scale, const void* bias, float eps, void* y, float* mean,
                                     float* rstd, void* stream_) {
  if (int rc = check(dtype, param_dtype, rows, width)) return rc;
  if (rows == 0) return AZ_OK;
  if (!x || !y || !mean != !rstd) return az_fail(AZ_ERR_INVALID, "layer norm: null x or y, or one of mean and rstd");
  hipStream_t stream = (hipStream_t)stream_;
  Norm p = {};
  p.x = x, p.scale = scale, p.bias = bias, p.out = y, p.mean = mean, p.rstd = rstd, p.eps = eps;
  p.rows = rows, p.width = width;
  return with_types(dtype, param_dtype, [&]<typename T, typename P>() -> int {
    if (width > IN_REGISTERS) {
      k_norm_forward_wide<T, P><<<dim3((unsigned)few(rows)), dim3(1024), 0, stream>>>(p);
    } else {
      with_shape<T, P>(width, [&]<int NT, int R, bool EXACT>() {
        constexpr int ROWS = NT < 256 ? 256 / NT : 1;
        k_norm_forward<T, P, NT, R, EXACT><<<dim3((unsigned)few(az_ceil(rows, ROWS))), dim3(NT < 256 ? 256 : NT), 0, stream>>>(p);
      });
    }
    AZ_LAUNCH_CHECK();
    return AZ_OK;
  });
}

extern "C" int64_t az_layer_norm_workspace_bytes(int32_t rows, int32_t width) {
  if (check(AZ_TYPE_F32, AZ_TYPE_F32, rows, width) != AZ_OK) return -1;
  return rows == 0 ? 0 : (int64_t)backward_blocks(rows, width) * 2 * width * 4;
}

extern "C" int az_layer_norm_backward(int32_t dtype, int32_t param_dtype, int32_t rows, int32_t width, const void* x,
                                      const void* scale, const float* mean, const float* rstd, const void* dy,
                                      void* dx, void* dscale, void* dbias, void* workspace, int64_t workspace_bytes,
                                      void* stream_) {
  if (int rc = check(dtype, param_dtype, rows, width)) return rc;
  hipStream_t stream = (hipStream_t)stream_;
  const bool columns = dscale || dbias;
  if (!columns && !dx) return AZ_OK;
  return with_types(dtype, param_dtype, [&]<typename T, typename P>() -> int {
    if (rows == 0) {
      if (columns)
        k_norm_zero<P><<<dim3((unsigned)az_ceil(width, 256)), dim3(256), 0, stream>>>((P*)dscale, (P*)dbias, width);
      AZ_LAUNCH_CHECK();
      return AZ_OK;
    }
    if (!x || !mean || !rstd || !dy) return az_fail(AZ_ERR_INVALID, "layer norm backward: null x, mean, rstd or dy");
    const int blocks = backward_blocks(rows, width);
    if (columns && (workspace_bytes < (int64_t)blocks * 2 * width * 4 || !workspace || !az_aligned16(workspace)))
      return az_fail(AZ_ERR_INVALID, "layer norm: the workspace must hold %lld bytes, 16-byte aligned",
                     (long long)blocks * 2 * width * 4);
    Norm p = {};
    p.x = x, p.scale = scale, p.dy = dy, p.out = dx, p.mean = const_cast<float*>(mean);
    p.rstd = const_cast<float*>(rstd), p.partial = columns ? (float*)workspace : nullptr;
    p.rows = rows, p.width = width;
    if (width > IN_REGISTERS) {
      if (dx) k_norm_backward_wide<T, P><<<dim3((unsigned)few(rows)), dim3(1024), 0, stream>>>(p);
      if (columns)
        k_norm_columns_wide<T><<<dim3((unsigned)az_ceil(width, 256), blocks), dim3(256), 0, stream>>>(p);
    } else {
      with_shape<T, P>(width, [&]<int NT, int R, bool EXACT>() {
        k_norm_backward<T, P, NT, R, EXACT><<<dim3(blocks), dim3(NT < 256 ? 256 : NT), 0, stream>>>(p);
      });
    }
    AZ_LAUNCH_CHECK();
    if (columns) {
      k_norm_join<P><<<dim3((unsigned)az_ceil(width, 64), 2), dim3(1024), 0, stream>>>((const float*)workspace, blocks,
                                                                                     width, (P*)dscale, (P*)dbias);
      AZ_LAUNCH_CHECK();
    }
    return AZ_OK;
  });
}
