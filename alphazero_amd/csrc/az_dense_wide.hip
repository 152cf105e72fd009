// az_dense_wide.hip -- the large products of a dense layer on the 16-bit matrix instructions.
// Part of libaz_mcts.so (gfx950 only).
//
// A workgroup computes BM x BN outputs, 64 reduction steps at a time: the next step's operands go from global memory
// straight into LDS (16 bytes a lane, no registers) while the waves multiply the current ones, two buffers in
// turn.  An operand whose reduction axis is contiguous lies in LDS as rows of 128 bytes and is read 16 bytes a lane;
// one whose other axis is contiguous lies as 64 rows of BM (BN) elements and is read by the transposing LDS read, which
// hands lane i column i of a 4 x 16 block.  Both are swizzled in 16-byte chunks so that the lanes of
// one read fall on all banks: a direct load puts lane l's bytes at l * 16, so the swizzle is in the global address that a
// lane loads from.  The buffer descriptor ends where the matrix ends: what is loaded beyond it is zero, which
// covers the ragged edges (rows beyond M or N are not stored; a reduction over rows that ends inside a step adds
// zeros; a reduction along contiguous rows is a multiple of 64 here).
//
// Bound: 16384 x 4096 x 4096 bfloat16 takes 398 us at best and 431 on average for dkernel, 418 and 453 for dx (1.2-1.4
// PFLOP/s; a library product of that size reaches 1.2), at which the matrix pipes are busy 0.69 and 0.63 of the cycles of a
// clock that the power limit holds near 2 GHz; over dz's two planes 791 and 850, 830 and 887 us.  The forward pass takes
// 522-552 us at best, 563-584 on average, its pipes busy 0.5 of the cycles: its epilogue moves another 400 MB that nothing
// overlaps (one workgroup a compute unit: two stages are 128 KB).  LDS is busy a quarter of the cycles, without bank
// conflicts.  Measured and not kept: four waves of 128 x 128 (fewer LDS reads, but one wave a SIMD: 1.83 ms a step instead of 1.52), three to five stages for the
// 128 x 128 tiles (8192 x 1024 x 1024: 44 us instead of 28: their loads already fill the way from L2, 64 bytes a cycle).
//
// float32 products run on the same instructions: an operand is split into three bfloat16 planes x = x0 + x1 + x2
// (each the rounding of what the planes before it left, so the three hold all 24 bits), and of the nine products the
// six that matter, x0 y0, x0 y1, x1 y0, x1 y1, x0 y2, x2 y0, are added in one float32 accumulator, the small ones
// first.  What is left out is below 2^-26 of the terms' magnitudes; operands below 2^-110 lose bits of their last plane
// (products of values around 2^-114 are off by 6e-7 instead of 1.2e-7 at 1400 x 1300 x 1400, around 2^-118 by 9e-6).  Six
// bfloat16 products cost 6 / 16 of the float32 instruction's time.  An infinity or an overflow turns into NaN on the way (inf - inf, inf * 0): an output
// that is not finite is worked out again from the float32 operands by the float32 instruction, 16 rows of a wave at a time.
#include <hip/hip_runtime.h>

#include "az_dense.h"

using namespace az_dense;

namespace {

typedef __attribute__((address_space(3))) void lds_void;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int STEP = 64;   // reduction steps per stage

typedef int i32x4 __attribute__((ext_vector_type(4)));

// A buffer descriptor of the bytes from p to end: what is loaded from beyond is zero.
__device__ __forceinline__ i32x4 descriptor(const char* p, const char* end) {
  const int64_t left = end - p;
  const uint32_t n = left <= 0 ? 0u : left > 0xffffffffll ? 0xffffffffu : (uint32_t)left;
  const uint64_t at = (uint64_t)p;
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)at);
  r[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32) & 0xffff);
  r[2] = __builtin_amdgcn_readfirstlane((int)n);
  r[3] = 0x00027000;
  return r;
}

// Lane l's 16 bytes at `offset` behind the descriptor's start go to LDS byte `to` + 16 l.  In assembly, because for the
// builtin the compiler waits for every load in flight in front of each LDS read; the kernel's own waits are in front
// of its barriers.  (No register is written; the load reads M0 one instruction after it is set.)
__device__ __forceinline__ void load_to_lds(i32x4 r, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(to), "v"(offset), "s"(r)
               : "memory", "m0");
}

// chunk swizzle of reduction row k of an operand that is not reduction-contiguous: the eight 32-byte pieces that two
// groups of 16 lanes read at once (rows k..k+3 and k+8..k+11) go to eight places
__device__ __forceinline__ int row_swizzle(int k) { return 2 * ((k & 3) | ((k >> 1) & 4)); }

// One operand's stage: R rows (or columns) of the output, NW waves that load it.
template <bool KC, int R, int NW>
struct Operand {
  static constexpr int BYTES = R * STEP * 2, LOADS = BYTES / 1024 / NW;
  uint32_t offset[LOADS];   // this lane's byte offset from the stage's first element
  const char* base;
  const char* end;
  int64_t step;             // bytes from one stage to the next

  __device__ void init(const void* p, int64_t ld, int rows, int K, int r0, int wave, int lane) {
    for (int i = 0; i < LOADS; ++i) {
      const int ins = wave * LOADS + i;
      if constexpr (KC) {
        offset[i] = (uint32_t)((ins * 8 + (lane >> 3)) * ld * 2) + (((lane & 7) ^ (lane >> 3)) * 16);
      } else {
        constexpr int LANES = R / 8;   // lanes (16-byte chunks) a reduction row
        const int k = ins * (64 / LANES) + lane / LANES;
        offset[i] = (uint32_t)(k * ld * 2) + (((lane % LANES) ^ row_swizzle(k)) * 16);
      }
    }
    end = (const char*)p + (KC ? (int64_t)rows : (int64_t)K) * ld * 2;
    base = (const char*)p + (KC ? r0 * ld : (int64_t)r0) * 2;
    step = KC ? STEP * 2 : STEP * ld * 2;
  }
  // stage t (of the plane `plane` bytes further) into lds
  __device__ __forceinline__ void load(int t, int64_t plane, uint32_t lds, int wave) const {
    const i32x4 r = descriptor(base + plane + t * step, end + plane);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) load_to_lds(r, offset[i], lds + (wave * LOADS + i) * 1024);
  }
};

// The 16 x 32 fragment of rows r0.. and reduction steps sub * 32.. of a stage.
template <bool KC, int R>
__device__ __forceinline__ uint4 fragment(const char* lds, int r0, int sub, int lane) {
  if constexpr (KC) {
    const int row = r0 + (lane & 15), chunk = sub * 4 + (lane >> 4);
    return *reinterpret_cast<const uint4*>(lds + row * 128 + ((chunk ^ (row & 7)) * 16));
  } else {
    const int k = sub * 32 + (lane >> 4) * 8 + ((lane >> 2) & 3);
    const int chunk = r0 / 8 + ((lane >> 1) & 1), byte = (lane & 1) * 8;
    // rows k and k + 4 have the same swizzle
    const char* p = lds + k * (R * 2) + ((chunk ^ row_swizzle(k)) * 16) + byte;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * (R * 2)));
    uint4 r;
    __builtin_memcpy(&r, &lo, 8);
    __builtin_memcpy((char*)&r + 8, &hi, 8);
    return r;
  }
}

// The pairs of planes of float32 operands, a hexadecimal digit each from the left: (0,2) (2,0) (1,1) (0,1) (1,0) (0,0), so
// that what is small has been added up before the accumulator has its full size.
constexpr int PAIRS = 6, A_PLANES = 0x021010, B_PLANES = 0x201100;
constexpr int plane_of(int planes, int pair) { return (planes >> (4 * (PAIRS - 1 - pair))) & 15; }
constexpr bool small_first() {
  int seen = 0;   // a bit for each pair
  for (int i = 0; i < PAIRS; ++i) {
    const int a = plane_of(A_PLANES, i), b = plane_of(B_PLANES, i);
    if (a + b > 2 || (i > 0 && a + b > plane_of(A_PLANES, i - 1) + plane_of(B_PLANES, i - 1))) return false;
    seen |= 1 << (3 * a + b);
  }
  return seen == 0b1011111;
}
static_assert(small_first());

template <typename T>
__device__ __forceinline__ az_f32x4 mma16(uint4 a, uint4 b, az_f32x4 c) {
  return mma(__builtin_bit_cast(AzPack<T>, a), __builtin_bit_cast(AzPack<T>, b), c);
}

// Workgroups go to the eight dies in turn, each with an L2 of its own: a die takes a contiguous run of tiles, and
// the run goes down columns of GROUP tiles, so that the operands of the tiles in flight on a die are few.
__device__ __forceinline__ void tile_of(int id, int tiles_m, int tiles_n, int* tm, int* tn) {
  const int n = tiles_m * tiles_n, per = n / 8, rest = n % 8, die = id % 8;
  const int at = die * per + min(die, rest) + id / 8;
  constexpr int GROUP = 4;
  const int group = at / (GROUP * tiles_n), first = group * GROUP, height = min(GROUP, tiles_m - first);
  const int in = at - group * GROUP * tiles_n;
  *tm = first + in % height;
  *tn = in / height;
}

// T: type of the operands in memory and LDS; TO: of the outputs; SPLIT: T is bfloat16 planes of float32 operands; LOW: one
// operand is dz as a hi and a lo plane.
template <typename T, typename TO, int BM, int BN, int WM, int WN, bool AKC, bool BKC, int EPI, bool SPLIT, bool LOW>
__global__ __launch_bounds__(WM* WN * 64, 2) void k_product_wide(Prod p) {
  constexpr int NW = WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
  typedef Operand<AKC, BM, NW> OpA;
  typedef Operand<BKC, BN, NW> OpB;
  constexpr int STAGE = OpA::BYTES + OpB::BYTES;
  __shared__ alignas(16) char lds[2 * STAGE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t lds_at = (uint32_t)(uintptr_t)(lds_void*)lds;
  int tm, tn;
  tile_of(blockIdx.x, p.tiles_m, p.tiles_n, &tm, &tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);
  OpA a;
  OpB b;
  a.init(p.a, p.lda, p.M, p.K, m0, wave, lane);
  b.init(p.b, p.ldb, p.N, p.K, n0, wave, lane);
  // stages of this split; float32 operands go through them once for each pair of planes, dz for each of its two
  const int t0 = blockIdx.z * (p.k_chunk / STEP), t1 = min((p.K + STEP - 1) / STEP, t0 + p.k_chunk / STEP);
  const int stages = (t1 - t0) * (SPLIT ? PAIRS : LOW ? 2 : 1);
  auto load = [&](int s, int buf) {
    int t = t0 + s;
    int64_t pa = 0, pb = 0;
    if constexpr (SPLIT) {
      const int pair = s / (t1 - t0);
      t -= pair * (t1 - t0);
      pa = plane_of(A_PLANES, pair) * p.a_plane * 2;
      pb = plane_of(B_PLANES, pair) * p.b_plane * 2;
    }
    if constexpr (LOW) {   // the lo plane first
      if (s < t1 - t0)
        pa = p.a_plane * 2, pb = p.b_plane * 2;
      else
        t -= t1 - t0;
    }
    a.load(t, pa, lds_at + buf * STAGE, wave);
    b.load(t, pb, lds_at + buf * STAGE + OpA::BYTES, wave);
  };
  az_f32x4 acc[FM][FN] = {};
  // Two sets of fragments: while one half of a stage is multiplied, the next half (of this stage, or of the next one
  // behind the barrier) is read.
  uint4 fa[2][FM], fb[2][FN];
  auto read = [&](int s, int sub) {
    const char* la = lds + (s & 1) * STAGE;
#pragma unroll
    for (int j = 0; j < FN; ++j) fb[sub][j] = fragment<BKC, BN>(la + OpA::BYTES, wn + j * 16, sub, lane);
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[sub][i] = fragment<AKC, BM>(la, wm + i * 16, sub, lane);
  };
  auto multiply = [&](int sub) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = mma16<T>(fb[sub][j], fa[sub][i], acc[i][j]);
  };
  // one LDS read, then its share of the matrix instructions: left to itself the compiler puts each read in front of its
  // use and waits for it (16384 x 4096 x 4096, three products and the rest of a step: 1.52 ms, 1.46 ms this way)
  auto interleave = [&] {
    constexpr int READS = FM * (AKC ? 1 : 2) + FN * (BKC ? 1 : 2), PER = FM * FN / READS;
#pragma unroll
    for (int i = 0; i < READS; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x8, PER, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, FM * FN - READS * PER, 0);
  };
  load(0, 0);
  if (stages > 1) load(1, 1);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  read(0, 0);
  auto run = [&](int first, int last) {
    for (int s = first; s < last; ++s) {
      read(s, 1);
      multiply(0);
      interleave();
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();   // the next stage is in LDS, and this one's readers are done
      if (s + 2 < stages) load(s + 2, s & 1);
      read(s + 1, 0);    // (behind the last stage: read, not used)
      multiply(1);
      interleave();
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if constexpr (LOW) {
    run(0, t1 - t0);
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) scale_low<T>(acc[i][j]);
    run(t1 - t0, stages);
  } else {
    run(0, stages);
  }
  // The outputs leave through LDS, up to 64 rows of a wave at a time, so that a row's columns are written together; the
  // sixteen groups of four columns are exchanged by the row, which spreads the rows over the banks.
  constexpr int ROUND = FM < 4 ? FM : 4;
  static_assert(FN % 4 == 0 && FM % ROUND == 0 && NW * ROUND * 16 * 64 * 4 <= 2 * STAGE);
  float* out = reinterpret_cast<float*>(lds) + wave * (ROUND * 16 * 64);
  __syncthreads();
#pragma unroll
  for (int part = 0; part < FM / ROUND * (FN / 4); ++part) {
    const int i0 = part / (FN / 4) * ROUND, j0 = part % (FN / 4) * 4;
#pragma unroll
    for (int i = 0; i < ROUND; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = i * 16 + (lane & 15), quad = j * 4 + (lane >> 4);
        *reinterpret_cast<az_f32x4*>(out + row * 64 + ((quad ^ (row & 15)) * 4)) = acc[i0 + i][j0 + j];
      }
    if constexpr (SPLIT) {
      // outputs that are not finite, 16 rows at a time, from the float32 operands (a row and column beyond the edge
      // stand for the last one)
#pragma unroll 1
      for (int i = 0; i < ROUND; ++i) {
        const int row = i * 16 + (lane & 15);
        auto at = [&](int j) {
          return reinterpret_cast<az_f32x4*>(out + row * 64 + (((j * 4 + (lane >> 4)) ^ (row & 15)) * 4));
        };
        bool bad = false;
        for (int j = 0; j < 4; ++j)
          for (int e = 0; e < 4; ++e) bad |= !(fabsf((*at(j))[e]) < INFINITY);
        if (__ballot(bad) == 0) continue;
        const int64_t m = min(m0 + wm + i0 * 16 + row, p.M - 1);
        const int k1 = min(p.K, t1 * STEP);
        az_f32x4 sum[4] = {};
        for (int k = t0 * STEP; k < k1; k += 16) {
          const int kk = k + (lane >> 4) * 4;
          AzPack<float> x;
          for (int e = 0; e < 4; ++e)
            x.v[e] = kk + e < k1 ? p.a32[AKC ? m * p.lda32 + kk + e : (kk + e) * p.lda32 + m] : 0.0f;
          for (int j = 0; j < 4; ++j) {
            const int64_t n = min(n0 + wn + (j0 + j) * 16 + (lane & 15), p.N - 1);
            AzPack<float> y;
            for (int e = 0; e < 4; ++e)
              y.v[e] = kk + e < k1 ? p.b32[BKC ? n * p.ldb32 + kk + e : (kk + e) * p.ldb32 + n] : 0.0f;
            sum[j] = mma(y, x, sum[j]);
          }
        }
        for (int j = 0; j < 4; ++j) {
          az_f32x4 v = *at(j);
          for (int e = 0; e < 4; ++e)
            if (!(fabsf(v[e]) < INFINITY)) v[e] = sum[j][e];
          *at(j) = v;
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
    const int n = n0 + wn + j0 * 16 + (lane & 15) * 4;
    // the residual of the next rows is loaded while these are worked on: 64 bytes a lane in flight
    constexpr int AHEAD = 8;
    AzVec<TO, 4> next[AHEAD];
    const bool early = EPI == EPI_FORWARD && p.residual && n + 4 <= p.N;
    auto fetch = [&](int r0) {
      if (!early) return;
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int m = m0 + wm + i0 * 16 + r0 + k * 4 + (lane >> 4);
        if (m < p.M) next[k] = az_loadu<TO, 4>((const TO*)p.residual + (int64_t)m * p.N + n);
      }
    };
    fetch(0);
#pragma unroll 1
    for (int r0 = 0; r0 < ROUND * 16; r0 += 4 * AHEAD) {
      AzVec<TO, 4> res[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) res[k] = next[k];
      if (r0 + 4 * AHEAD < ROUND * 16) fetch(r0 + 4 * AHEAD);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int row = r0 + 4 * k + (lane >> 4), m = m0 + wm + i0 * 16 + row;
        const az_f32x4 x = *reinterpret_cast<const az_f32x4*>(out + row * 64 + (((lane & 15) ^ (row & 15)) * 4));
        float v[4] = {x[0], x[1], x[2], x[3]};
        finish<TO, EPI>(p, m, n, v, early, res[k]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
  }
}

template <typename T, typename TO, bool AKC, bool BKC, int EPI, bool SPLIT, bool LOW = false>
int launch(const Prod& p, bool big, int splits, hipStream_t stream) {
  const dim3 grid(p.tiles_m * p.tiles_n, 1, splits);
  if (big)
    k_product_wide<T, TO, 256, 256, 2, 4, AKC, BKC, EPI, SPLIT, LOW><<<grid, dim3(512), 0, stream>>>(p);
  else if constexpr (AKC && !SPLIT)
    // Eight waves of 32 x 64: a compute unit with one tile hides more of its latencies than with four of 64 x 64, whose
    // fewer LDS reads win where both operands take transposing reads (dkernel) and over float32's long reductions:
    // 2048 x 512 x 512 bfloat16 y 10.6 / 13.3 us, dx 7.5 / 8.5, but dkernel of 4096 x 2048 x 2048 55.5 / 50.8 and float32
    // y of 4096 x 1024 x 1024 91 / 79
    k_product_wide<T, TO, 128, 128, 4, 2, AKC, BKC, EPI, SPLIT, LOW><<<grid, dim3(512), 0, stream>>>(p);
  else
    k_product_wide<T, TO, 128, 128, 2, 2, AKC, BKC, EPI, SPLIT, LOW><<<grid, dim3(256), 0, stream>>>(p);
  AZ_LAUNCH_CHECK();
  return AZ_OK;
}

}  // namespace

int az_product_wide(int dtype, int pass, bool split_k, bool big, const Prod* p, int splits, hipStream_t stream) {
  auto run = [&]<typename T, typename TO, bool SPLIT>() -> int {
    if (pass == PASS_Y)
      return split_k ? launch<T, TO, true, false, EPI_PARTIAL, SPLIT>(*p, big, splits, stream)
                     : launch<T, TO, true, false, EPI_FORWARD, SPLIT>(*p, big, splits, stream);
    if constexpr (!SPLIT) {
      if (p->planes > 1) {
        if (pass == PASS_DX)
          return split_k ? launch<T, TO, true, true, EPI_PARTIAL, SPLIT, true>(*p, big, splits, stream)
                         : launch<T, TO, true, true, EPI_STORE, SPLIT, true>(*p, big, splits, stream);
        return split_k ? launch<T, TO, false, false, EPI_PARTIAL, SPLIT, true>(*p, big, splits, stream)
                       : launch<T, TO, false, false, EPI_STORE, SPLIT, true>(*p, big, splits, stream);
      }
    }
    if (pass == PASS_DX)
      return split_k ? launch<T, TO, true, true, EPI_PARTIAL, SPLIT>(*p, big, splits, stream)
                     : launch<T, TO, true, true, EPI_STORE, SPLIT>(*p, big, splits, stream);
    return split_k ? launch<T, TO, false, false, EPI_PARTIAL, SPLIT>(*p, big, splits, stream)
                   : launch<T, TO, false, false, EPI_STORE, SPLIT>(*p, big, splits, stream);
  };
  if (dtype == AZ_TYPE_F32) return run.template operator()<az_bf16, float, true>();
  if (dtype == AZ_TYPE_BF16) return run.template operator()<az_bf16, az_bf16, false>();
  return run.template operator()<az_f16, az_f16, false>();
}
