// Tile products of the dense-layer (linear.hip) and matrix-optimizer (newton_schulz.hip) kernels.
//
// C[m][n] = sum_k A(m, k) B(k, n) for one BM x BN tile of C. An operand is either k-contiguous in memory
// (KC: element (row, k) at row * ld + k) or row-contiguous (element (row, k) at k * ld + row), where "row" is
// m for A and n for B; both are staged the way they are stored. One stage holds 128 bytes of k per row:
//   16-bit elements   64 k, two MFMA 16x16x32 steps
//   fp32              32 k, eight MFMA 16x16x4 steps (the exact-fp32 pipe)
//   pair              32 k of an fp32 value kept as h + l, two fp16 numbers: 32 h then 32 l, 64 bytes each.
//                     Three products h h + h l + l h on the fp16 pipe; what is left out is below 2^-22.
//
// LDS layout of a stage: KC [row][8 chunks of 16 bytes], chunk c of a row at c ^ (row & 7); row-contiguous
// [k][rows], segments swizzled by k (see Operand). With it the reads of a fragment are free of bank conflicts
// by the model of split_common.h (the 16 lanes served together hit 16 different 16-byte slots).
// Row-contiguous 16-bit fragments come out of LDS transposed (ds_read_b64_tr_b16).
#pragma once
#include "split_common.h"

namespace dtf {

typedef _Float16 halfx4 __attribute__((ext_vector_type(4)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef __bf16 bfx4 __attribute__((ext_vector_type(4)));

enum MmKind { MM_F32 = 0, MM_BF16 = 1, MM_F16 = 2, MM_PAIR = 3 };

template <MmKind KIND>
struct MmTraits {
  static constexpr int ES = (KIND == MM_F32 || KIND == MM_PAIR) ? 4 : 2;   // bytes per (row, k) element
  static constexpr int KB = 128 / ES;                                      // k per stage
  static constexpr int EPC = 16 / ES;                                      // elements per 16-byte chunk
  static constexpr int KS = KIND == MM_PAIR ? 1 : 2;                       // fragment steps per stage
};

// fp32, bf16 and fp16 values in memory
template <MmKind KIND> struct MmElem { using type = float; };
template <> struct MmElem<MM_BF16> { using type = __bf16; };
template <> struct MmElem<MM_F16> { using type = _Float16; };

struct Frag { uintx4 h, l; };   // l: pairs only

__device__ __forceinline__ void mm_mfma(std::integral_constant<MmKind, MM_BF16>, const Frag& x, const Frag& y, floatx4& acc) {
  acc = DTF_MFMA_BF16(__builtin_bit_cast(bf16x8, x.h), __builtin_bit_cast(bf16x8, y.h), acc);
}
__device__ __forceinline__ void mm_mfma(std::integral_constant<MmKind, MM_F16>, const Frag& x, const Frag& y, floatx4& acc) {
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, x.h), __builtin_bit_cast(halfx8, y.h), acc, 0, 0, 0);
}
__device__ __forceinline__ void mm_mfma(std::integral_constant<MmKind, MM_F32>, const Frag& x, const Frag& y, floatx4& acc) {
  const floatx4 xv = __builtin_bit_cast(floatx4, x.h), yv = __builtin_bit_cast(floatx4, y.h);
#pragma unroll
  for (int s = 0; s < 4; ++s) acc = DTF_MFMA16(xv[s], yv[s], acc);
}
__device__ __forceinline__ void mm_mfma(std::integral_constant<MmKind, MM_PAIR>, const Frag& x, const Frag& y, floatx4& acc) {
  const halfx8 xh = __builtin_bit_cast(halfx8, x.h), xl = __builtin_bit_cast(halfx8, x.l);
  const halfx8 yh = __builtin_bit_cast(halfx8, y.h), yl = __builtin_bit_cast(halfx8, y.l);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(xl, yh, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh, yl, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh, yh, acc, 0, 0, 0);
}

// One operand of a stage: ROWS rows x KB k, staged by NT threads.
template <MmKind KIND, bool KC, int ROWS, int NT>
struct Operand {
  using Tr = MmTraits<KIND>;
  static constexpr int BYTES = ROWS * 128;
  static constexpr int NV = ROWS * 8 / NT;           // 16-byte chunks per thread
  static constexpr int CPR = ROWS * Tr::ES / 16;     // row-contiguous: chunks per k
  static_assert(ROWS * 8 % NT == 0, "a stage is a whole number of chunks per thread");
  static constexpr int SEGS = CPR / 2;               // row-contiguous: 32-byte segments per k
  static_assert(KC || (ROWS >= 64 && (SEGS & (SEGS - 1)) == 0), "the swizzles permute the segments of a line");

  // Row-contiguous: where chunk c of line k lies. Transposed 16-bit reads fetch 32-byte segments (16 rows) of 16
  // values of k at once: the segment number is XORed with three bits of k that differ between the lanes served
  // together. fp32 reads fetch 64 bytes (16 rows) of four k that are 4 apart.
  __device__ static int rc_place(int k, int c) {
    if (KIND == MM_F32) return c ^ (((k >> 2) & 3) << 2);
    return c ^ ((((k & 3) | ((k >> 1) & 4)) & (SEGS - 1)) << 1);
  }

  // element offset from the tile's base, and how many of the chunk's elements exist
  struct Chunk { int row, k; };
  __device__ static Chunk chunk_of(int e) {   // chunk e of the stage in LDS order -> its (row, k) of the tile
    Chunk c;
    if (KC) {
      c.row = e >> 3;
      c.k = ((e & 7) ^ (c.row & 7)) * Tr::EPC;
    } else {
      c.k = e / CPR;
      c.row = rc_place(c.k, e % CPR) * Tr::EPC;
    }
    return c;
  }

  // Through registers, for any alignment and any edge: elements outside the matrix are zeros.
  __device__ static void fetch(const char* src, long long ld, int row0, int rows, int k0, int k_end, int tid, uintx4 (&r)[NV]) {
    typedef uintx4 __attribute__((aligned(2))) loose;   // only as aligned as its elements
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      const Chunk c = chunk_of(tid + it * NT);
      const int gr = row0 + c.row, gk = k0 + c.k;
      int have = KC ? (gr < rows ? k_end - gk : 0) : (gk < k_end ? rows - gr : 0);
      const char* p = src + (KC ? (long long)gr * ld + gk : (long long)gk * ld + gr) * Tr::ES;
      uintx4 v = {0, 0, 0, 0};
      if (have >= Tr::EPC) {
        v = *reinterpret_cast<const loose*>(p);
      } else if (have > 0) {
        if (Tr::ES == 4) {
#pragma unroll
          for (int i = 0; i < 3; ++i)
            if (i < have) v[i] = reinterpret_cast<const unsigned*>(p)[i];
        } else {
#pragma unroll
          for (int i = 0; i < 7; ++i)
            if (i < have) v[i >> 1] |= (unsigned)reinterpret_cast<const unsigned short*>(p)[i] << (16 * (i & 1));
        }
      }
      r[it] = v;
    }
  }
  __device__ static void commit(char* lds, int tid, const uintx4 (&r)[NV]) {
#pragma unroll
    for (int it = 0; it < NV; ++it) *reinterpret_cast<uintx4*>(lds + (tid + it * NT) * 16) = r[it];
  }

  // Fragment of 16 rows starting at row0 (a multiple of 16), step ks of the stage: lane (q, l15) gets row row0 + l15,
  // k = 32 ks + 8 q + (0..7) (16-bit, pair) or 16 ks + 4 q + (0..3) (fp32).
  __device__ static Frag frag(const char* lds, int row0, int ks, int q, int l15) {
    Frag f;
    if (KC) {
      const int row = row0 + l15;
      const char* p = lds + row * 128;
      f.h = *reinterpret_cast<const uintx4*>(p + (((ks * 4 + q) ^ (row & 7)) << 4));
      if (KIND == MM_PAIR) f.l = *reinterpret_cast<const uintx4*>(p + (((4 + q) ^ (row & 7)) << 4));
    } else if (KIND == MM_F32) {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int k = ks * 16 + 4 * q + s;
        f.h[s] = *reinterpret_cast<const unsigned*>(lds + (k * CPR + rc_place(k, (row0 + l15) >> 2)) * 16 + (l15 & 3) * 4);
      }
    } else {
      // lane i of a group of 16 supplies the address of 4 rows of line k + (i >> 2) and receives row i of four lines
      const int k = ks * 32 + 8 * q + (l15 >> 2);
      const int seg = KIND == MM_PAIR ? (row0 >> 5) * 4 + ((row0 >> 4) & 1) : row0 >> 4;   // 32-byte segment of the line
      auto read = [&](int kk, int sg) {
        return lds_read_tr(reinterpret_cast<const unsigned char*>(lds) + (kk * CPR + rc_place(kk, sg * 2 + ((l15 >> 1) & 1))) * 16 + (l15 & 1) * 8);
      };
      const uintx2 a = read(k, seg), b = read(k + 4, seg);
      f.h = uintx4{a[0], a[1], b[0], b[1]};
      if (KIND == MM_PAIR) {
        const uintx2 c = read(k, seg + 2), d = read(k + 4, seg + 2);
        f.l = uintx4{c[0], c[1], d[0], d[1]};
      }
    }
    return f;
  }
};

// acc[i][j] += the product of a wave's MI x NJ tiles of 16 x 16 over one stage. SWAP: lane (q, l15), register r holds
// C[m = l15][n = 4 q + r] of a tile (four consecutive n), else C[m = 4 q + r][n = l15].
template <MmKind KIND, class OpA, class OpB, int MI, int NJ, bool SWAP>
__device__ __forceinline__ void mm_stage(const char* As, const char* Bs, int wm, int wn, int q, int l15, floatx4 (&acc)[MI][NJ]) {
  constexpr std::integral_constant<MmKind, KIND> kind{};
#pragma unroll
  for (int ks = 0; ks < MmTraits<KIND>::KS; ++ks) {
    Frag a[MI], b[NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i) a[i] = OpA::frag(As, wm + i * 16, ks, q, l15);
#pragma unroll
    for (int j = 0; j < NJ; ++j) b[j] = OpB::frag(Bs, wn + j * 16, ks, q, l15);
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        if (SWAP) mm_mfma(kind, b[j], a[i], acc[i][j]);
        else mm_mfma(kind, a[i], b[j], acc[i][j]);
      }
  }
}

// What a product needs to know of its operands.
struct MmOperands {
  const char* a;
  const char* b;
  long long lda, ldb;   // elements
  int M, N;
};

// Through registers: the loads of stage s + 1 are in flight under the products of stage s. Any alignment.
template <MmKind KIND, bool KCA, bool KCB, int BM, int BN, int WGM, int WGN, bool SWAP>
struct MmRegs {
  static constexpr int NT = 64 * WGM * WGN, MI = BM / WGM / 16, NJ = BN / WGN / 16;
  using OpA = Operand<KIND, KCA, BM, NT>;
  using OpB = Operand<KIND, KCB, BN, NT>;
  static constexpr int LDS = OpA::BYTES + OpB::BYTES;
  __device__ static void run(const MmOperands& o, int m0, int n0, int k_begin, int k_end, char* smem, floatx4 (&acc)[MI][NJ]) {
    constexpr int KB = MmTraits<KIND>::KB;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q = lane >> 4, l15 = lane & 15;
    const int wm = (wave / WGN) * (BM / WGM), wn = (wave % WGN) * (BN / WGN);
    char *As = smem, *Bs = smem + OpA::BYTES;
    uintx4 ra[OpA::NV], rb[OpB::NV];
    if (k_begin < k_end) {
      OpA::fetch(o.a, o.lda, m0, o.M, k_begin, k_end, tid, ra);
      OpB::fetch(o.b, o.ldb, n0, o.N, k_begin, k_end, tid, rb);
    }
    for (int k0 = k_begin; k0 < k_end; k0 += KB) {
      OpA::commit(As, tid, ra);
      OpB::commit(Bs, tid, rb);
      __syncthreads();
      if (k0 + KB < k_end) {
        OpA::fetch(o.a, o.lda, m0, o.M, k0 + KB, k_end, tid, ra);
        OpB::fetch(o.b, o.ldb, n0, o.N, k0 + KB, k_end, tid, rb);
      }
      mm_stage<KIND, OpA, OpB, MI, NJ, SWAP>(As, Bs, wm, wn, q, l15, acc);
      __syncthreads();
    }
  }
};

// Work item of block `id` of `total`: every XCD (blocks go to the eight of them round-robin) takes one contiguous range.
__device__ __forceinline__ int mm_item(int id, int total) {
  const int per = (total + 7) >> 3;
  return (id & 7) * per + (id >> 3);
}
// Tile t of a gx x gy grid, in groups of eight rows of tiles walked column by column: the tiles that an XCD works on
// at a time share rows and columns of the operands in its L2.
__device__ __forceinline__ void mm_tile_of(int t, int gx, int gy, int& tx, int& ty) {
  const int g = t / (8 * gx), first = g * 8, h = min(8, gy - first), in = t - g * 8 * gx;
  ty = first + in % h;
  tx = in / h;
}

}  // namespace dtf
