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
  int vec;             // four consecutive n can be read and written at once in every [M,N] tensor
  int splits;
  AbortRef abort;
};

// A value before the activation -> act(z). NaN stays NaN.
__device__ __forceinline__ float lin_act(int act, float z) {
  switch (act) {
    case ACT_RELU: return z < 0.f ? 0.f : z;
    case ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    case ACT_GELU_TANH: return z / (1.f + expf(-1.5957691216057308f * (z + 0.044715f * z * z * z)));   // (1 + tanh u) / 2 = 1 / (1 + e^-2u)
    case ACT_SILU: return z / (1.f + expf(-z));
    default: return z;
  }
}
__device__ __forceinline__ float lin_act_grad(int act, float z) {
  switch (act) {
    case ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case ACT_GELU: return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * expf(-0.5f * z * z) * 0.39894228040143268f;
    case ACT_GELU_TANH: {
      const float q = 1.f / (1.f + expf(-1.5957691216057308f * (z + 0.044715f * z * z * z)));
      return q + z * q * (1.f - q) * (1.5957691216057308f * (1.f + 0.134145f * z * z));
    }
    case ACT_SILU: {
      const float q = 1.f / (1.f + expf(-z));
      return q * (1.f + z * (1.f - q));
    }
    default: return 1.f;
  }
}

// Four consecutive values of a tensor <-> fp32. `vec`: the address allows one access; else `have` of them, one by one.
template <MmKind KIND>
__device__ __forceinline__ floatx4 lin_load4(const void* base, long long at, int vec, int have) {
  using E = typename MmElem<KIND>::type;
  typedef E E4 __attribute__((ext_vector_type(4)));
  const E* p = reinterpret_cast<const E*>(base) + at;
  floatx4 v = {0.f, 0.f, 0.f, 0.f};
  if (vec) {
    v = __builtin_convertvector(*reinterpret_cast<const E4*>(p), floatx4);
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
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < have) p[i] = (E)v[i];
  }
}

// The epilogue of four consecutive n of row m: every tensor is rounded once, from the fp32 value.
template <MmKind KIND>
__device__ __forceinline__ void lin_finish(const MmProduct& p, int vec, int m, int n, floatx4 v) {
  const int have = p.N - n;
  if (p.bias) v += lin_load4<KIND>(p.bias, n, vec, have);
  if (p.pre) lin_store4<KIND>(p.pre, (long long)m * p.ldp + n, vec, have, v);
  if (p.act != ACT_NONE) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = lin_act(p.act, v[i]);
  }
  if (p.res) v += lin_load4<KIND>(p.res, (long long)m * p.ldr + n, vec, have);
  const long long at = (long long)m * p.ldc + n;
  if (p.accumulate) v += lin_load4<KIND>(p.c, at, vec, have);
  lin_store4<KIND>(p.c, at, vec, have, v);
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
  const MmOperands o{reinterpret_cast<const char*>(p.a), reinterpret_cast<const char*>(p.b), p.lda, p.ldb, p.M, p.N};
  Loop::run(o, m0, n0, k_begin, k_end, lin_smem, acc);

  // The sums leave through LDS, 32 rows of a wave's tile at a time: a loop over whole rows with 16 lanes to a row, so the
  // tensors are read and written 64 columns at once and the epilogue's code exists once. Each wave has its own rows: no barrier.
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, l15 = lane & 15;
  const int wm = (wave / WGN) * (BM / WGM), wn = (wave % WGN) * (BN / WGN);
  float* rows = reinterpret_cast<float*>(lin_smem) + wave * (32 * LinEpilogue<NJ>::PITCH);
#pragma unroll
  for (int i0 = 0; i0 < MI; i0 += 2) {
    if (m0 + wm + i0 * 16 >= p.M) break;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        *reinterpret_cast<floatx4*>(rows + (i * 16 + l15) * LinEpilogue<NJ>::PITCH + j * 16 + 4 * q) = acc[i0 + i][j];
#pragma unroll 1
    for (int e = lane; e < 32 * NJ * 4; e += 64) {
      const int r = e / (NJ * 4), c = (e % (NJ * 4)) * 4;
      const int m = m0 + wm + i0 * 16 + r, n = n0 + wn + c;
      if (m >= p.M || n >= p.N) continue;
      const floatx4 v = *reinterpret_cast<const floatx4*>(rows + r * LinEpilogue<NJ>::PITCH + c);
      if (a.splits > 1) *reinterpret_cast<floatx4*>(a.partial + ((long long)split * p.M + m) * a.N4 + n) = v;   // N4 covers the last n
      else lin_finish<KIND>(p, a.vec, m, n, v);
    }
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

// dz = dy act'(pre) and the sums of its columns. A block takes 256 columns (four per thread) and rows_per_block
// rows, a quarter of them per wave; the waves' sums are added in wave order, the blocks' by lin_colsum_kernel.
struct LinDzArgs {
  const void* dy; long long lddy;
  const void* pre; long long ldp;
  void* dz; long long lddz;    // null: only the sums
  float* part;                 // [row blocks][N4], null: no sums
  long long N4;
  int M, N, act, rows_per_block;
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
    for (int m = m_begin + wave; m < m_end; m += 4) {
      floatx4 v = lin_load4<KIND>(a.dy, (long long)m * a.lddy + n, a.vec, have);
      if (a.act != ACT_NONE) {
        const floatx4 z = lin_load4<KIND>(a.pre, (long long)m * a.ldp + n, a.vec, have);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] *= lin_act_grad(a.act, z[i]);
      }
      if (a.dz) lin_store4<KIND>(a.dz, (long long)m * a.lddz + n, a.vec, have, v);
      s += v;
    }
  }
  if (!a.part) return;
  sums[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && have > 0)
    *reinterpret_cast<floatx4*>(a.part + (long long)blockIdx.y * a.N4 + n) = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
}
struct LinColSumArgs { const float* part; long long N4; int blocks, N, accumulate; void* db; AbortRef abort; };
template <MmKind KIND>
__global__ __launch_bounds__(256) void linear_colsum_kernel(LinColSumArgs a) {
  DTF_ABORT_GUARD(a);
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n >= a.N) return;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  int b = 0;
  for (; b + 4 <= a.blocks; b += 4) {
#pragma unroll
    for (int u = 0; u < 4; ++u) s[u] += a.part[(long long)(b + u) * a.N4 + n];
  }
  for (; b < a.blocks; ++b) s[0] += a.part[(long long)b * a.N4 + n];
  using E = typename MmElem<KIND>::type;
  E* out = reinterpret_cast<E*>(a.db) + n;
  float v = (s[0] + s[1]) + (s[2] + s[3]);
  if (a.accumulate) v += (float)*out;
  *out = (E)v;
}

// The launches of one element type. Variants of the product kernel: see linear.hip.
struct LinLaunch {
  void (*tile)(const LinTileArgs&, int variant, hipStream_t);
  void (*join)(const LinTileArgs&, hipStream_t);
  void (*dz)(const LinDzArgs&, dim3 grid, hipStream_t);
  void (*colsum)(const LinColSumArgs&, hipStream_t);
};
const LinLaunch& lin_launch_f32();
const LinLaunch& lin_launch_bf16();
const LinLaunch& lin_launch_f16();

// The variants of the product kernel: tile, waves over it, stages in LDS, 128-byte pieces of k per stage.
enum LinVariant { LIN_REGS = 0, LIN_64 = 1, LIN_128 = 2, LIN_256 = 3 };
struct LinTile { int t, wgm, wgn, stages, subs; };
constexpr LinTile kLinTiles[] = {{128, 2, 2, 1, 1}, {64, 2, 2, 4, 1}, {128, 2, 4, 2, 2}, {256, 2, 4, 2, 1}};

template <MmKind KIND, bool KCA, bool KCB, int V>
struct LinLoopOf {
  static constexpr LinTile T = kLinTiles[V];
  using type = MmDirect<KIND, KCA, KCB, T.t, T.t, T.wgm, T.wgn, true, T.stages, T.subs>;
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
  launch("linear", linear_tile_kernel<KIND, Loop, T.t, T.t, T.wgm, T.wgn>, dim3((unsigned)((a.total + 7) / 8 * 8)), dim3(64 * WAVES), lin_lds<Loop, WAVES>(),
         stream, a);
}
template <MmKind KIND, bool KCA, bool KCB>
void lin_tile_launch(const LinTileArgs& a, int variant, hipStream_t stream) {
  switch (variant) {
    case LIN_REGS: return lin_tile_launch_as<KIND, KCA, KCB, LIN_REGS>(a, stream);
    case LIN_64: return lin_tile_launch_as<KIND, KCA, KCB, LIN_64>(a, stream);
    case LIN_128: return lin_tile_launch_as<KIND, KCA, KCB, LIN_128>(a, stream);
    case LIN_256: return lin_tile_launch_as<KIND, KCA, KCB, LIN_256>(a, stream);
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
  l.colsum = [](const LinColSumArgs& a, hipStream_t s) {
    launch("linear_colsum", linear_colsum_kernel<KIND>, dim3((unsigned)ceil_div(a.N, 256)), dim3(256), 0, s, a);
  };
  return l;
}

}  // namespace dtf
