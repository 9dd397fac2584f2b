// The product kernels behind linear.hip, instantiated per element type (linear_f32 / bf16 / f16.hip).
#pragma once
#include "linear.h"
#include "mm_tile.h"

namespace dtf {

struct LinTileArgs {
  MmProduct p;
  float* partial;      // splits > 1: [split][M][N4] sums, N4 = N rounded up to 4; the epilogue runs in the reduction
  long long N4;
  int k_per_split;
  int gx, gy, total;   // tiles of C, and tiles x splits
  int rows_a, rows_b;  // M and N for the loads: padded where the operand's contiguous dimension is
  int vec;             // four consecutive n can be read and written at once in every [M,N] tensor
  int splits;
  AbortRef abort;
};

// Exponential and logistic function: the library's for fp32 tensors; for 16-bit ones, which round to 2^-9 and 2^-12, the hardware's
// base-2 exponential and reciprocal (a few 2^-23 relative for the arguments that matter).
template <MmKind KIND>
__device__ __forceinline__ float lin_exp(float x) {
  return KIND == MM_F32 ? expf(x) : __builtin_amdgcn_exp2f(x * 1.4426950408889634f);
}
template <MmKind KIND>
__device__ __forceinline__ float lin_logistic(float x) {
  const float d = 1.f + lin_exp<KIND>(-x);
  return KIND == MM_F32 ? 1.f / d : __builtin_amdgcn_rcpf(d);
}
// Phi(z), the normal distribution function, and e^(-z^2/2). 16-bit tensors: erfc(x) = (a1 t + ... + a5 t^5) e^(-x^2), t = 1 / (1 + p x), off by
// at most 1.5e-7 (Abramowitz and Stegun, 7.1.26) - erff and the like cost 35 us of the 450 of an 8192 x 4096 x 8192 product.
template <MmKind KIND>
__device__ __forceinline__ float lin_phi(float z, float& gauss) {
  gauss = lin_exp<KIND>(-0.5f * z * z);
  if (KIND == MM_F32) return 0.5f * (1.f + erff(z * 0.70710678118654752f));
  const float t = __builtin_amdgcn_rcpf(1.f + 0.3275911f * 0.70710678118654752f * fabsf(z));
  const float tail = 0.5f * gauss * t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
  return z < 0.f ? tail : 1.f - tail;
}
// A value before the activation -> act(z). NaN stays NaN.
template <MmKind KIND>
__device__ __forceinline__ float lin_act(int act, float z) {
  float gauss;
  switch (act) {
    case ACT_RELU: return z < 0.f ? 0.f : z;
    case ACT_GELU: return z * lin_phi<KIND>(z, gauss);
    case ACT_GELU_TANH: return z * lin_logistic<KIND>(1.5957691216057308f * (z + 0.044715f * z * z * z));   // (1 + tanh u) / 2 = 1 / (1 + e^-2u)
    case ACT_SILU: return z * lin_logistic<KIND>(z);
    default: return z;
  }
}
// dy act'(z). ReLU selects: whatever arrives at a unit that is off stays there.
template <MmKind KIND>
__device__ __forceinline__ float lin_act_bwd(int act, float dy, float z) {
  float gauss;
  // Every slope has reached its limit long before: no z^2 that overflows and no infinity times zero. NaN stays.
  z = z > 1e4f ? 1e4f : z < -1e4f ? -1e4f : z;
  switch (act) {
    case ACT_RELU: return z > 0.f ? dy : z <= 0.f ? 0.f : z;
    case ACT_GELU: {
      const float phi = lin_phi<KIND>(z, gauss);
      return dy * (phi + z * gauss * 0.39894228040143268f);
    }
    case ACT_GELU_TANH: {
      const float q = lin_logistic<KIND>(1.5957691216057308f * (z + 0.044715f * z * z * z));
      return dy * (q + z * q * (1.f - q) * (1.5957691216057308f * (1.f + 0.134145f * z * z)));
    }
    case ACT_SILU: {
      const float q = lin_logistic<KIND>(z);
      return dy * (q * (1.f + z * (1.f - q)));
    }
    default: return dy;
  }
}

// Four consecutive values of a tensor <-> fp32. `vec`: they are there and aligned. Otherwise `have` of them are there, four in one
// unaligned access, fewer one by one.
template <MmKind KIND>
__device__ __forceinline__ floatx4 lin_load4(const void* base, long long at, int vec, int have) {
  using E = typename MmElem<KIND>::type;
  typedef E E4 __attribute__((ext_vector_type(4)));
  const E* p = reinterpret_cast<const E*>(base) + at;
  floatx4 v = {0.f, 0.f, 0.f, 0.f};
  if (vec) {
    v = __builtin_convertvector(*reinterpret_cast<const E4*>(p), floatx4);
  } else if (have >= 4) {
    typedef E4 __attribute__((aligned(2))) loose;
    v = __builtin_convertvector(*reinterpret_cast<const loose*>(p), floatx4);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < have) v[i] = (float)p[i];
  }
  return v;
}
template <MmKind KIND>
__device__ __forceinline__ void lin_store4(void* base, long long at, int vec, int have, const floatx4& v) {
  using E = typename MmElem<KIND>::type;
  typedef E E4 __attribute__((ext_vector_type(4)));
  E* p = reinterpret_cast<E*>(base) + at;
  if (vec) {
    *reinterpret_cast<E4*>(p) = __builtin_convertvector(v, E4);
  } else if (have >= 4) {
    typedef E4 __attribute__((aligned(2))) loose;
    *reinterpret_cast<loose*>(p) = __builtin_convertvector(v, E4);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < have) p[i] = (E)v[i];
  }
}

// The epilogue of four consecutive n of row m: every tensor is rounded once, from the fp32 value. What it reads comes apart, so that
// a caller can have several rows' reads in flight.
template <MmKind KIND>
struct LinRead { floatx4 res, old; };
template <MmKind KIND>
__device__ __forceinline__ LinRead<KIND> lin_read(const MmProduct& p, int vec, int m, int n) {
  LinRead<KIND> r;
  if (p.res) r.res = lin_load4<KIND>(p.res, (long long)m * p.ldr + n, vec, p.N - n);
  if (p.accumulate) r.old = lin_load4<KIND>(p.c, (long long)m * p.ldc + n, vec, p.N - n);
  return r;
}
template <MmKind KIND>
__device__ __forceinline__ void lin_finish(const MmProduct& p, int vec, int m, int n, floatx4 v, const floatx4& bias, const LinRead<KIND>& r) {
  const int have = p.N - n;
  v = v * p.scale + bias;
  if (p.pre) lin_store4<KIND>(p.pre, (long long)m * p.ldp + n, vec, have, v);
  if (p.act != ACT_NONE) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = lin_act<KIND>(p.act, v[i]);
  }
  if (p.res) v += r.res;
  if (p.accumulate) v += r.old;
  lin_store4<KIND>(p.c, (long long)m * p.ldc + n, vec, have, v);
}
template <MmKind KIND>
__device__ __forceinline__ floatx4 lin_bias(const MmProduct& p, int vec, int n) {
  return p.bias ? lin_load4<KIND>(p.bias, n, vec, p.N - n) : floatx4{0.f, 0.f, 0.f, 0.f};
}
template <MmKind KIND>
__device__ __forceinline__ void lin_finish(const MmProduct& p, int vec, int m, int n, const floatx4& v) {
  lin_finish<KIND>(p, vec, m, n, v, lin_bias<KIND>(p, vec, n), lin_read<KIND>(p, vec, m, n));
}

// Lanes of a wave that hand each other values through LDS: a wave's accesses of LDS happen in order, so all it takes is that the compiler
// keeps every access on its side of this point, and the lanes together at it. No instruction.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

template <int NJ>
struct LinEpilogue { static constexpr int PITCH = NJ * 16 + 4; };   // floats; the 16 bytes spread a column over the banks
template <class Loop, int WAVES>
constexpr int lin_lds() {
  constexpr int epi = WAVES * 32 * LinEpilogue<Loop::NJ>::PITCH * 4;
  return epi > Loop::LDS ? epi : Loop::LDS;
}

template <MmKind KIND, class Loop, int BM, int BN, int WGM, int WGN>
__global__ __launch_bounds__(64 * WGM * WGN) void linear_tile_kernel(LinTileArgs a) {
  DTF_ABORT_GUARD(a);
  extern __shared__ __attribute__((aligned(16))) char lin_smem[];
  const int t = mm_item(blockIdx.x, a.total);
  if (t >= a.total) return;
  const MmProduct& p = a.p;
  const int tiles = a.gx * a.gy, split = t / tiles;
  int tx, ty;
  mm_tile_of(t - split * tiles, a.gx, a.gy, tx, ty);
  const int m0 = ty * BM, n0 = tx * BN;
  const int k_begin = split * a.k_per_split, k_end = min(p.K, k_begin + a.k_per_split);
  constexpr int MI = BM / WGM / 16, NJ = BN / WGN / 16;
  floatx4 acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  const MmOperands o{reinterpret_cast<const char*>(p.a), reinterpret_cast<const char*>(p.b), p.lda, p.ldb, a.rows_a, a.rows_b};
  Loop::run(o, m0, n0, k_begin, k_end, lin_smem, acc);

  // The sums leave through LDS, 32 rows of a wave's tile at a time: a loop over whole rows with 16 lanes to a row, so the
  // tensors are read and written 64 columns at once and the epilogue's code exists once. Each wave has its own rows: no barrier.
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));   // what follows from it is computed here, not kept in registers over the product
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), q = lane >> 4, l15 = lane & 15;
  const int wm = (wave / WGN) * (BM / WGM), wn = (wave % WGN) * (BN / WGN);
  constexpr int PITCH = LinEpilogue<NJ>::PITCH, LANES = NJ * 4, RSTEP = 64 / LANES, U = RSTEP > 8 ? 32 / RSTEP : 4;   // lanes to a row, rows at once, reads ahead
  static_assert(64 % LANES == 0 && 32 % (RSTEP * U) == 0, "a lane keeps its columns");
  float* rows = reinterpret_cast<float*>(lin_smem) + wave * (32 * PITCH);
  const int c = (lane % LANES) * 4, n = n0 + wn + c, r0 = lane / LANES;
  floatx4 bias = {0.f, 0.f, 0.f, 0.f};
  if (a.splits == 1 && n < p.N) bias = lin_bias<KIND>(p, a.vec, n);
#pragma unroll
  for (int i0 = 0; i0 < MI; i0 += 2) {
    const int mb = m0 + wm + i0 * 16;
    if (mb >= p.M) break;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) *reinterpret_cast<floatx4*>(rows + (i * 16 + l15) * PITCH + j * 16 + 4 * q) = acc[i0 + i][j];
    wave_lds_fence();
    if (n < p.N) {   // the lanes without a column wait at the fence below
#pragma unroll 1
      for (int r = r0; r < 32; r += RSTEP * U) {
        if (a.splits > 1) {
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (mb + r + u * RSTEP < p.M)   // N4 covers the last n
              *reinterpret_cast<floatx4*>(a.partial + ((long long)split * p.M + mb + r + u * RSTEP) * a.N4 + n) =
                  *reinterpret_cast<const floatx4*>(rows + (r + u * RSTEP) * PITCH + c);
          continue;
        }
        LinRead<KIND> rd[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (mb + r + u * RSTEP < p.M) rd[u] = lin_read<KIND>(p, a.vec, mb + r + u * RSTEP, n);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (mb + r + u * RSTEP < p.M)
            lin_finish<KIND>(p, a.vec, mb + r + u * RSTEP, n, *reinterpret_cast<const floatx4*>(rows + (r + u * RSTEP) * PITCH + c), bias, rd[u]);
      }
    }
    wave_lds_fence();
  }
}

// Sums of the splits in a fixed order, then the epilogue. One thread per four n of a row.
template <MmKind KIND>
__global__ __launch_bounds__(256) void linear_join_kernel(LinTileArgs a) {
  DTF_ABORT_GUARD(a);
  const long long per_row = a.N4 >> 2, count = per_row * a.p.M, plane = a.N4 * a.p.M;
  const long long stride = (long long)gridDim.x * 256;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < count; i += stride) {
    const float* src = a.partial + 4 * i;
    floatx4 v = *reinterpret_cast<const floatx4*>(src);
    for (int s = 1; s < a.splits; ++s) v += *reinterpret_cast<const floatx4*>(src + s * plane);
    const int m = (int)(i / per_row), n = (int)(i - m * per_row) * 4;
    lin_finish<KIND>(a.p, a.vec, m, n, v);
  }
}

// ---- A few rows: the weights are read once and that is all the time there is. 16 waves a workgroup, as many 16-byte
// loads in flight as a wave has use for, fp32 multiply-adds on the vector pipe, sums in a fixed order.
constexpr int kRowWaves = 16;
template <MmKind KIND>
__device__ __forceinline__ void row_unpack(const uintx4& v, float (&f)[16 / sizeof(typename MmElem<KIND>::type)]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (KIND == MM_F32) {
      f[i] = __uint_as_float(v[i]);
    } else if constexpr (KIND == MM_BF16) {
      f[2 * i] = pair_lo(v[i]);
      f[2 * i + 1] = pair_hi(v[i]);
    } else {
      f[2 * i] = (float)__builtin_bit_cast(_Float16, (unsigned short)v[i]);
      f[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (unsigned short)(v[i] >> 16));
    }
  }
}
// Sums of a workgroup's waves: part[wave][m][cols] -> the epilogue, or the split's partial sums.
template <MmKind KIND, int MR>
__device__ __forceinline__ void row_finish(const LinTileArgs& a, const float* part, int cols, int n0, int split) {
  __syncthreads();
  const int per_row = cols / 4;
  for (int e = threadIdx.x; e < MR * per_row; e += 64 * kRowWaves) {
    const int m = e / per_row, c = (e - m * per_row) * 4, n = n0 + c;
    if (m >= a.p.M || n >= a.p.N) continue;
    floatx4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kRowWaves; ++w) v += *reinterpret_cast<const floatx4*>(part + (w * MR + m) * cols + c);
    if (a.splits > 1) *reinterpret_cast<floatx4*>(a.partial + ((long long)split * a.p.M + m) * a.N4 + n) = v;
    else lin_finish<KIND>(a.p, a.vec, m, n, v);
  }
}
// W [K,N]: a lane owns one 16-byte chunk of columns and eight consecutive k; LPR lanes side by side make the columns of a
// workgroup, the 64 / LPR others go along k.
template <MmKind KIND, int MR, int LPR>
__global__ __launch_bounds__(64 * kRowWaves) void linear_row_n_kernel(LinTileArgs a) {
  DTF_ABORT_GUARD(a);
  using E = typename MmElem<KIND>::type;
  constexpr int EPC = 16 / sizeof(E), COLS = LPR * EPC, KL = 64 / LPR;   // lanes along k
  extern __shared__ __attribute__((aligned(16))) char lin_smem[];
  float* part = reinterpret_cast<float*>(lin_smem);
  const int t = mm_item(blockIdx.x, a.total);   // neighbours in n, which share cache lines, on one XCD
  if (t >= a.total) return;
  const MmProduct& p = a.p;
  const int split = t / a.gx, n0 = (t - split * a.gx) * COLS;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = n0 + (lane & (LPR - 1)) * EPC, kl = lane / LPR;
  const int k_begin = split * a.k_per_split, k_end = min(p.K, k_begin + a.k_per_split);   // multiples of 8
  const E* w = reinterpret_cast<const E*>(p.b) + n;
  const E* x = reinterpret_cast<const E*>(p.a);
  float acc[MR][EPC];
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int e = 0; e < EPC; ++e) acc[m][e] = 0.f;
  for (int k0 = k_begin + (wave * KL + kl) * 8; k0 < k_end; k0 += kRowWaves * KL * 8) {
    if (n >= p.N) break;
    uintx4 wv[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) wv[u] = *reinterpret_cast<const uintx4*>(w + (long long)(k0 + u) * p.ldb);
    uintx4 xv[MR][8 / EPC];   // packed, to spare registers
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
      for (int h = 0; h < 8 / EPC; ++h) xv[m][h] = reinterpret_cast<const uintx4*>(x + (long long)min(m, p.M - 1) * p.lda + k0)[h];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      float f[EPC];
      row_unpack<KIND>(wv[u], f);
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        float g[EPC];
        row_unpack<KIND>(xv[m][u / EPC], g);
#pragma unroll
        for (int e = 0; e < EPC; ++e) acc[m][e] = fmaf(g[u % EPC], f[e], acc[m][e]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int e = 0; e < EPC; ++e) {
      float v = acc[m][e];
#pragma unroll
      for (int off = LPR; off < 64; off <<= 1) v += __shfl_xor(v, off);
      acc[m][e] = v;
    }
  if (kl == 0) {
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
      for (int e = 0; e < EPC; e += 4)
        *reinterpret_cast<floatx4*>(part + (wave * MR + m) * COLS + lane * EPC + e) = floatx4{acc[m][e], acc[m][e + 1], acc[m][e + 2], acc[m][e + 3]};
  }
  row_finish<KIND, MR>(a, part, COLS, n0, split);
}
// W [N,K] (rows of k): a wave owns one column of C at a time and its lanes go along k; 16 columns a workgroup and a
// copy of x in LDS. The waves' sums need no joining.
template <MmKind KIND, int MR>
__global__ __launch_bounds__(64 * kRowWaves) void linear_row_k_kernel(LinTileArgs a) {
  DTF_ABORT_GUARD(a);
  using E = typename MmElem<KIND>::type;
  constexpr int EPC = 16 / sizeof(E), DEEP = 4;
  extern __shared__ __attribute__((aligned(16))) char lin_smem[];
  const int t = mm_item(blockIdx.x, a.total);
  if (t >= a.total) return;
  const MmProduct& p = a.p;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int chunks = p.K / EPC;   // whole: K is a multiple of 8
  uintx4* xs = reinterpret_cast<uintx4*>(lin_smem);   // [MR][chunks]
  float* part = reinterpret_cast<float*>(lin_smem + (size_t)MR * chunks * 16);   // [MR][16]
  const int n = t * kRowWaves + wave;
  const uintx4* w = reinterpret_cast<const uintx4*>(reinterpret_cast<const E*>(p.b) + (long long)min(n, p.N - 1) * p.ldb);
  uintx4 wv[DEEP];
#pragma unroll
  for (int u = 0; u < DEEP; ++u) wv[u] = lane + 64 * u < chunks ? w[lane + 64 * u] : uintx4{0, 0, 0, 0};
  for (int e = threadIdx.x; e < MR * chunks; e += 64 * kRowWaves) {
    const int m = e / chunks;
    xs[e] = reinterpret_cast<const uintx4*>(reinterpret_cast<const E*>(p.a) + (long long)min(m, p.M - 1) * p.lda)[e - m * chunks];
  }
  __syncthreads();
  float acc[MR];
#pragma unroll
  for (int m = 0; m < MR; ++m) acc[m] = 0.f;
  for (int c0 = lane; c0 < chunks; c0 += 64 * DEEP) {
#pragma unroll
    for (int u = 0; u < DEEP; ++u) {
      const int c = c0 + 64 * u;
      if (c < chunks) {
        float f[EPC];
        row_unpack<KIND>(wv[u], f);
        if (c + 64 * DEEP < chunks) wv[u] = w[c + 64 * DEEP];
#pragma unroll
        for (int m = 0; m < MR; ++m) {
          float g[EPC];
          row_unpack<KIND>(xs[m * chunks + c], g);
#pragma unroll
          for (int e = 0; e < EPC; ++e) acc[m] = fmaf(g[e], f[e], acc[m]);
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MR; ++m) {
    const float v = wave_sum(acc[m]);
    if (lane == 0) part[m * kRowWaves + wave] = v;
  }
  __syncthreads();
  if (threadIdx.x < MR * 4) {
    const int m = threadIdx.x >> 2, c = (threadIdx.x & 3) * 4;
    if (m < p.M && t * kRowWaves + c < p.N) lin_finish<KIND>(p, a.vec, m, t * kRowWaves + c, *reinterpret_cast<const floatx4*>(part + m * kRowWaves + c));
  }
}

// dz = dy act'(pre) and the sums of its columns. dz is rounded to the tensors' type, which is what the matrix pipe multiplies: dx and dW of 16-bit tensors are off by
// 1.4 times their own rounding (8192 x 4096 x 4096 bf16 2.3e-3 of 64 bits, with dz in fp32 1.7e-3); the column sums take the unrounded values. A block takes 256 columns (four per thread) and rows_per_block
// rows, a quarter of them per wave; the waves' sums are added in wave order, the blocks' by lin_colsum_kernel.
struct LinDzArgs {
  const void* dy; long long lddy;
  const void* pre; long long ldp;
  void* dz; long long lddz;    // null: only the sums
  float* part;                 // [row blocks][N4], null: no sums
  long long N4;
  int M, N, act, rows_per_block;
  float dz_scale;              // dz is stored times this
  int vec;
  AbortRef abort;
};
template <MmKind KIND>
__global__ __launch_bounds__(256) void linear_dz_kernel(LinDzArgs a) {
  DTF_ABORT_GUARD(a);
  __shared__ floatx4 sums[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = blockIdx.x * 256 + lane * 4, have = a.N - n;
  const int m_begin = blockIdx.y * a.rows_per_block, m_end = min(a.M, m_begin + a.rows_per_block);
  floatx4 s = {0.f, 0.f, 0.f, 0.f};
  if (have > 0) {
    constexpr int U = 2;   // rows whose loads are in flight together
    for (int m0 = m_begin + wave; m0 < m_end; m0 += 4 * U) {
      floatx4 v[U], z[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int m = min(m0 + 4 * u, m_end - 1);
        v[u] = lin_load4<KIND>(a.dy, (long long)m * a.lddy + n, a.vec, have);
        if (a.act != ACT_NONE) z[u] = lin_load4<KIND>(a.pre, (long long)m * a.ldp + n, a.vec, have);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int m = m0 + 4 * u;
        if (m >= m_end) break;
        if (a.act != ACT_NONE) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i < have) v[u][i] = lin_act_bwd<KIND>(a.act, v[u][i], z[u][i]);
        }
        if (a.dz) lin_store4<KIND>(a.dz, (long long)m * a.lddz + n, 1, 4, v[u] * a.dz_scale);   // zeros past N
        s += v[u];
      }
    }
  } else if (a.dz && n < a.lddz) {
    for (int m = m_begin + wave; m < m_end; m += 4) lin_store4<KIND>(a.dz, (long long)m * a.lddz + n, 1, 4, s);
  }
  if (!a.part) return;
  sums[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && have > 0)
    *reinterpret_cast<floatx4*>(a.part + (long long)blockIdx.y * a.N4 + n) = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
}
// Copies of operands that are not 16-byte aligned, lines padded with zeros: one pass over a matrix that a product reads many times.
struct LinPadArgs {
  const void* src[2]; void* dst[2];
  long long ld[2], ld_dst[2];   // elements; ld_dst a multiple of 16 bytes
  int rows[2], cols[2];
  AbortRef abort;
};
template <MmKind KIND>
__global__ __launch_bounds__(256) void linear_pad_kernel(LinPadArgs a) {
  DTF_ABORT_GUARD(a);
  using Raw = std::conditional_t<KIND == MM_F32, unsigned, unsigned short>;
  constexpr int EPC = MmTraits<KIND>::EPC;
  typedef Raw Chunk __attribute__((ext_vector_type(EPC)));
  typedef Chunk __attribute__((aligned(2))) loose;
  const int z = blockIdx.y, lane = threadIdx.x & 63;
  const Raw* src = reinterpret_cast<const Raw*>(a.src[z]);
  if (!src) return;
  const int per_row = (int)(a.ld_dst[z] / EPC);
  for (int row = blockIdx.x * 4 + (threadIdx.x >> 6); row < a.rows[z]; row += gridDim.x * 4) {
    const Raw* s = src + row * a.ld[z];
    Chunk* d = reinterpret_cast<Chunk*>(reinterpret_cast<Raw*>(a.dst[z]) + row * a.ld_dst[z]);
    for (int c = lane; c < per_row; c += 64) {
      const int have = a.cols[z] - c * EPC;
      Chunk v = 0;
      if (have >= EPC) {
        v = *reinterpret_cast<const loose*>(s + c * EPC);
      } else {
#pragma unroll
        for (int e = 0; e < EPC; ++e)
          if (e < have) v[e] = s[c * EPC + e];
      }
      d[c] = v;
    }
  }
}
struct LinColSumArgs { const float* part; long long N4; int blocks, N, accumulate; void* db; AbortRef abort; };
template <MmKind KIND>
__global__ __launch_bounds__(256) void linear_colsum_kernel(LinColSumArgs a) {
  DTF_ABORT_GUARD(a);
  // 64 columns a workgroup; a wave adds every fourth block's sums, eight loads in flight, and the waves are added in order
  __shared__ float sums[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = blockIdx.x * 64 + lane;
  float s = 0.f;
  if (n < a.N) {
    for (int b = wave; b < a.blocks; b += 32) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = a.part[(long long)min(b + 4 * u, a.blocks - 1) * a.N4 + n];
#pragma unroll
      for (int u = 0; u < 8; ++u) s += b + 4 * u < a.blocks ? v[u] : 0.f;
    }
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave || n >= a.N) return;
  using E = typename MmElem<KIND>::type;
  E* out = reinterpret_cast<E*>(a.db) + n;
  float v = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
  if (a.accumulate) v += (float)*out;
  *out = (E)v;
}

// The launches of one element type. Variants of the product kernel: see linear.hip.
struct LinLaunch {
  void (*tile)(const LinTileArgs&, int variant, hipStream_t);
  void (*join)(const LinTileArgs&, hipStream_t);
  void (*dz)(const LinDzArgs&, dim3 grid, hipStream_t);
  void (*colsum)(const LinColSumArgs&, hipStream_t);
  void (*pad)(const LinPadArgs&, hipStream_t);
};
const LinLaunch& lin_launch_f32();
const LinLaunch& lin_launch_bf16();
const LinLaunch& lin_launch_f16();

// The variants of the product kernel: tile, waves over it, stages in LDS, 128-byte pieces of k per stage.
enum LinVariant { LIN_REGS = 0, LIN_64 = 1, LIN_128 = 2, LIN_256 = 3, LIN_32 = 4, LIN_ROWS = 5 };
struct LinTile { int tm, tn, wgm, wgn, stages, subs; };
constexpr LinTile kLinTiles[] = {{128, 128, 2, 2, 1, 1}, {64, 64, 2, 2, 4, 1}, {128, 128, 2, 4, 2, 2}, {256, 256, 2, 4, 2, 1}, {32, 64, 1, 4, 4, 1}};

template <MmKind KIND, bool KCA, bool KCB, int V>
struct LinLoopOf {
  static constexpr LinTile T = kLinTiles[V];
  using type = MmDirect<KIND, KCA, KCB, T.tm, T.tn, T.wgm, T.wgn, true, T.stages, T.subs>;
};
template <MmKind KIND, bool KCA, bool KCB>
struct LinLoopOf<KIND, KCA, KCB, LIN_REGS> {
  using type = MmRegs<KIND, KCA, KCB, 128, 128, 2, 2, true>;
};
template <MmKind KIND, bool KCA, bool KCB, int V>
void lin_tile_launch_as(const LinTileArgs& a, hipStream_t stream) {
  constexpr LinTile T = kLinTiles[V];
  constexpr int WAVES = T.wgm * T.wgn;
  using Loop = typename LinLoopOf<KIND, KCA, KCB, V>::type;
  launch("linear", linear_tile_kernel<KIND, Loop, T.tm, T.tn, T.wgm, T.wgn>, dim3((unsigned)((a.total + 7) / 8 * 8)), dim3(64 * WAVES), lin_lds<Loop, WAVES>(),
         stream, a);
}
// columns of a workgroup of the few-rows kernel over W [K,N], by lanes side by side
inline int lin_row_lanes(int N, int elems) {
  const int groups = ceil_div(N, elems);   // chunks of columns
  return groups >= 8 * 256 ? 8 : groups >= 4 * 256 ? 4 : 2;
}
template <MmKind KIND, int MR, bool KCB>
void lin_row_launch_as(const LinTileArgs& a, hipStream_t stream) {
  constexpr int EPC = MmTraits<KIND>::EPC;
  const dim3 grid((unsigned)((a.total + 7) / 8 * 8)), block(64 * kRowWaves);
  if (KCB) {
    launch("linear_rows", linear_row_k_kernel<KIND, MR>, grid, block, (size_t)MR * a.p.K * (16 / EPC) + MR * kRowWaves * 4, stream, a);
    return;
  }
  auto lds = [](int lanes) { return (size_t)kRowWaves * MR * lanes * EPC * 4; };
  switch (lin_row_lanes(a.p.N, EPC)) {
    case 2: launch("linear_rows", linear_row_n_kernel<KIND, MR, 2>, grid, block, lds(2), stream, a); break;
    case 4: launch("linear_rows", linear_row_n_kernel<KIND, MR, 4>, grid, block, lds(4), stream, a); break;
    default: launch("linear_rows", linear_row_n_kernel<KIND, MR, 8>, grid, block, lds(8), stream, a);
  }
}
template <MmKind KIND, bool KCB>
void lin_row_launch(const LinTileArgs& a, hipStream_t stream) {
  if (a.p.M <= 1) return lin_row_launch_as<KIND, 1, KCB>(a, stream);
  if constexpr (KIND == MM_F32 || KCB)
    if (a.p.M <= 2) return lin_row_launch_as<KIND, 2, KCB>(a, stream);
  if constexpr (KIND == MM_F32)
    if (a.p.M <= 4) return lin_row_launch_as<KIND, 4, KCB>(a, stream);
  throw std::runtime_error("linear: too many rows");
}
template <MmKind KIND, bool KCA, bool KCB>
void lin_tile_launch(const LinTileArgs& a, int variant, hipStream_t stream) {
  switch (variant) {
    case LIN_REGS: return lin_tile_launch_as<KIND, KCA, KCB, LIN_REGS>(a, stream);
    case LIN_64: return lin_tile_launch_as<KIND, KCA, KCB, LIN_64>(a, stream);
    case LIN_128: return lin_tile_launch_as<KIND, KCA, KCB, LIN_128>(a, stream);
    case LIN_256: return lin_tile_launch_as<KIND, KCA, KCB, LIN_256>(a, stream);
    case LIN_32:
      if constexpr (KCA) return lin_tile_launch_as<KIND, KCA, KCB, LIN_32>(a, stream);
      [[fallthrough]];
    case LIN_ROWS:
      if constexpr (KCA) return lin_row_launch<KIND, KCB>(a, stream);
      [[fallthrough]];
    default: throw std::runtime_error("linear: unknown variant");
  }
}
template <MmKind KIND>
LinLaunch lin_make_launch() {
  LinLaunch l;
  l.tile = [](const LinTileArgs& a, int variant, hipStream_t s) {
    if (a.p.kc_a) {
      if (a.p.kc_b) lin_tile_launch<KIND, true, true>(a, variant, s);
      else lin_tile_launch<KIND, true, false>(a, variant, s);
    } else {
      if (a.p.kc_b) throw std::runtime_error("linear: no product of a row-contiguous A with a k-contiguous B");
      lin_tile_launch<KIND, false, false>(a, variant, s);
    }
  };
  l.join = [](const LinTileArgs& a, hipStream_t s) {
    long long blocks = (a.N4 / 4 * a.p.M + 255) / 256;
    launch("linear_join", linear_join_kernel<KIND>, dim3((unsigned)(blocks > 4096 ? 4096 : blocks)), dim3(256), 0, s, a);
  };
  l.dz = [](const LinDzArgs& a, dim3 grid, hipStream_t s) { launch("linear_dz", linear_dz_kernel<KIND>, grid, dim3(256), 0, s, a); };
  l.pad = [](const LinPadArgs& a, hipStream_t s) {
    const int rows = a.rows[0] > a.rows[1] ? a.rows[0] : a.rows[1];
    launch("linear_pad", linear_pad_kernel<KIND>, dim3((unsigned)(rows > 8192 ? 2048 : ceil_div(rows, 4)), 2), dim3(256), 0, s, a);
  };
  l.colsum = [](const LinColSumArgs& a, hipStream_t s) {
    launch("linear_colsum", linear_colsum_kernel<KIND>, dim3((unsigned)ceil_div(a.N, 64)), dim3(256), 0, s, a);
  };
  return l;
}

}  // namespace dtf
