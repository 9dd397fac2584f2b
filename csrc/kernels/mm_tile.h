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

// Step `step` of the product of two fragments, on the matrix pipe.
template <MmKind KIND>
struct MmSteps { static constexpr int N = KIND == MM_F32 ? 4 : KIND == MM_PAIR ? 3 : 1; };
template <MmKind KIND>
__device__ __forceinline__ void mm_mfma(int step, const Frag& x, const Frag& y, floatx4& acc) {
  if constexpr (KIND == MM_BF16) {
    acc = DTF_MFMA_BF16(__builtin_bit_cast(bf16x8, x.h), __builtin_bit_cast(bf16x8, y.h), acc);
  } else if constexpr (KIND == MM_F32) {
    acc = DTF_MFMA16(__builtin_bit_cast(floatx4, x.h)[step], __builtin_bit_cast(floatx4, y.h)[step], acc);
  } else {   // pairs: l h, h l, h h
    const uintx4 xv = KIND == MM_PAIR && step == 0 ? x.l : x.h, yv = KIND == MM_PAIR && step == 1 ? y.l : y.h;
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, xv), __builtin_bit_cast(halfx8, yv), acc, 0, 0, 0);
  }
}

template <MmKind KIND>
__device__ __forceinline__ void mm_mfma_all(const Frag& x, const Frag& y, floatx4& acc) {
#pragma unroll
  for (int s = 0; s < MmSteps<KIND>::N; ++s) mm_mfma<KIND>(s, x, y, acc);
}

// 16 bytes per lane from memory to LDS at lds + 16 lane, past the registers; done when vmcnt says so. Written in asm
// because the compiler, which cannot tell the two stages of a double buffer apart, would wait for every such load
// before the next read of LDS. There is no output register. M0 is written in the same block and named as lost: the compiler, which reserves the
// register for instructions of its own and sets it right in front of them, remarks on that (inline-asm).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void lds_load16(const char* base, unsigned off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void lds_load16_any(const char* p, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds), "v"(p) : "memory", "m0");
}
#pragma clang diagnostic pop
// All but the last PENDING loads of this wave have landed, every read of LDS has returned, and all waves are here.
template <int PENDING>
__device__ __forceinline__ void lds_stage_barrier() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(PENDING) : "memory"); }
__device__ __forceinline__ unsigned lds_address(const char* p) {
  return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) char*)(p);
}
__device__ const unsigned mm_zeros[4] = {0, 0, 0, 0};

// One operand of a stage: ROWS rows x KB k, staged by NT threads.
template <MmKind KIND, bool KC, int ROWS, int NT>
struct Operand {
  using Tr = MmTraits<KIND>;
  static constexpr int BYTES = ROWS * 128;
  static constexpr int NV = ROWS * 8 / NT;           // 16-byte chunks per thread
  static constexpr int CPR = ROWS * Tr::ES / 16;     // row-contiguous: chunks per k
  static_assert(ROWS * 8 % NT == 0, "a stage is a whole number of chunks per thread");
  static constexpr int SEGS = CPR / 2;               // row-contiguous: 32-byte segments per k
  static constexpr int XORS = SEGS % 8 == 0 ? 7 : 3;
  static_assert(KC || (ROWS % 64 == 0 && SEGS % (XORS + 1) == 0), "the swizzles permute the segments of a line");

  // Row-contiguous: where chunk c of line k lies. Transposed 16-bit reads fetch 32-byte segments (16 rows) of 16
  // values of k at once: the segment number is XORed with three bits of k that differ between the lanes served
  // together. fp32 reads fetch 64 bytes (16 rows) of four k that are 4 apart.
  __device__ static int rc_place(int k, int c) {
    if (KIND == MM_F32) return c ^ (((k >> 2) & 3) << 2);
    return c ^ ((((k & 3) | ((k >> 1) & 4)) & XORS) << 1);
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

  // Straight from memory into LDS (16 bytes a lane, no registers). Rows past the matrix repeat its last one: what they
  // give is not stored. `off`: byte offsets from the operand's first row of the tile and first k of the stage.
  __device__ static void offsets(long long ld, int row0, int rows, int tid, unsigned (&off)[NV]) {
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      const Chunk c = chunk_of(tid + it * NT);
      const int row = min(row0 + c.row, rows - (KC ? 1 : Tr::EPC)) - row0;
      off[it] = (unsigned)((KC ? (long long)row * ld + c.k : (long long)c.k * ld + row) * Tr::ES);
    }
  }
  __device__ static const char* first(const char* src, long long ld, int row0, int k0) {
    return src + (KC ? (long long)row0 * ld + k0 : (long long)k0 * ld + row0) * Tr::ES;
  }
  __device__ static void load_piece(int it, const char* base, const unsigned (&off)[NV], unsigned lds, int wave) {
    lds_load16(base, off[it], lds + (it * NT + wave * 64) * 16);
  }
  __device__ static void load(const char* base, const unsigned (&off)[NV], unsigned lds, int wave) {
#pragma unroll
    for (int it = 0; it < NV; ++it) load_piece(it, base, off, lds, wave);
  }
  // the last stage of a k that ends inside it: zeros from there on
  __device__ static void load_tail(const char* base, const unsigned (&off)[NV], unsigned lds, int wave, int tid, int k_left) {
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      const Chunk c = chunk_of(tid + it * NT);
      const char* p = c.k < k_left ? base + off[it] : reinterpret_cast<const char*>(mm_zeros);
      lds_load16_any(p, lds + (it * NT + wave * 64) * 16);
    }
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
// between(g) is called after each of the KS * MI groups of products.
template <MmKind KIND, class OpA, class OpB, int MI, int NJ, bool SWAP, class Between>
__device__ __forceinline__ void mm_stage(const char* As, const char* Bs, int wm, int wn, int q, int l15, floatx4 (&acc)[MI][NJ], Between&& between) {
  constexpr int KS = MmTraits<KIND>::KS, GROUPS = KS * MI, AHEAD = MI < 2 ? 1 : 2;
  Frag a[AHEAD + 1], b[KS][NJ];
  auto read_b = [&](int ks) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) b[ks][j] = OpB::frag(Bs, wn + j * 16, ks, q, l15);
  };
  auto read_a = [&](int g) { a[g % (AHEAD + 1)] = OpA::frag(As, wm + (g % MI) * 16, g / MI, q, l15); };
  read_b(0);
#pragma unroll
  for (int g = 0; g < AHEAD; ++g)
    if (g < GROUPS) read_a(g);
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const int ks = g / MI, i = g % MI;
    if (g + AHEAD < GROUPS) read_a(g + AHEAD);
    if (ks + 1 < KS && i == MI - AHEAD) read_b(ks + 1);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int s = 0; s < MmSteps<KIND>::N; ++s) {
        if (SWAP) mm_mfma<KIND>(s, b[ks][j], a[g % (AHEAD + 1)], acc[i][j]);
        else mm_mfma<KIND>(s, a[g % (AHEAD + 1)], b[ks][j], acc[i][j]);
      }
    between(g);
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
      mm_stage<KIND, OpA, OpB, MI, NJ, SWAP>(As, Bs, wm, wn, q, l15, acc, [](int) {});
      __syncthreads();
    }
  }
};

// Straight into LDS, a ring of STAGES: the loads of the next STAGES - 1 stages are in flight under the products of one,
// one barrier per stage. 16-byte aligned operands: bases and leading dimensions, and whole chunks along the contiguous dimension.
// Two stages are enough where a stage's products outlast a load's way (tiles of 128 and more; rings of three and four measured
// no faster, pairs 192 x 192, K 4096: 131 -> 152 us); a 64 x 64 tile has 0.1 us of products per stage and needs more.
// Measured and not kept: the fragments of a step read under the products of the step before (bf16 8192 x 4096 x 4096,
// 128 x 128: 239 -> 292 us; the second set of registers costs the second workgroup of a CU, or spills).
template <MmKind KIND, bool KCA, bool KCB, int BM, int BN, int WGM, int WGN, bool SWAP, int STAGES = 2, int SUBS = 1>
struct MmDirect {
  static constexpr int NT = 64 * WGM * WGN, MI = BM / WGM / 16, NJ = BN / WGN / 16;
  using OpA = Operand<KIND, KCA, BM, NT>;
  using OpB = Operand<KIND, KCB, BN, NT>;
  static constexpr int SUB = OpA::BYTES + OpB::BYTES, STAGE = SUBS * SUB, LDS = STAGES * STAGE;
  static constexpr int PENDING = (STAGES - 2) * SUBS * (OpA::NV + OpB::NV);   // loads of a wave that may be in flight behind the next stage's
  static_assert(LDS <= (int)kLdsBudget && PENDING < 64, "a ring of stages fits LDS and the load counter");
  __device__ static void run(const MmOperands& o, int m0, int n0, int k_begin, int k_end, char* smem, floatx4 (&acc)[MI][NJ]) {
    constexpr int KB = MmTraits<KIND>::KB, ES = MmTraits<KIND>::ES;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q = lane >> 4, l15 = lane & 15;
    const int wm = (wave / WGN) * (BM / WGM), wn = (wave % WGN) * (BN / WGN);
    unsigned oa[OpA::NV], ob[OpB::NV];
    OpA::offsets(o.lda, m0, o.M, tid, oa);
    OpB::offsets(o.ldb, n0, o.N, tid, ob);
    const char *pa = OpA::first(o.a, o.lda, m0, k_begin), *pb = OpB::first(o.b, o.ldb, n0, k_begin);
    const long long step_a = (KCA ? KB : KB * o.lda) * ES, step_b = (KCB ? KB : KB * o.ldb) * ES;
    const unsigned lds = __builtin_amdgcn_readfirstlane(lds_address(smem));
    int k_load = k_begin;
    unsigned slot_load = 0;   // byte offset of the slot that the next load fills
    auto load = [&]() {
#pragma unroll
      for (int u = 0; u < SUBS; ++u) {
        const unsigned at = lds + slot_load + u * SUB;
        if (k_load + KB <= k_end) {
          OpA::load(pa, oa, at, wave);
          OpB::load(pb, ob, at + OpA::BYTES, wave);
        } else if (k_load < k_end) {
          OpA::load_tail(pa, oa, at, wave, tid, k_end - k_load);
          OpB::load_tail(pb, ob, at + OpA::BYTES, wave, tid, k_end - k_load);
        }
        pa += step_a;
        pb += step_b;
        k_load += KB;
      }
      slot_load = slot_load + STAGE == LDS ? 0 : slot_load + STAGE;
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s)
      if (k_load < k_end) load();
    unsigned slot = 0;
    constexpr int GROUPS = MmTraits<KIND>::KS * MI, PIECES = OpA::NV + OpB::NV;
    constexpr int RATE = (PIECES + GROUPS - 1) / GROUPS;
    int k0 = k_begin;
    // This stage has landed once no more than the loads issued after it are pending; near the end there are fewer.
    auto enter = [&]() {
      if (STAGES > 2 && k0 + (STAGES - 1) * SUBS * KB <= k_end) lds_stage_barrier<PENDING>();
      else lds_stage_barrier<0>();
    };
    // The next loads go into the slot that every wave left before the barrier. A CU takes 16 cycles for each of them: all at
    // once they would hold up the reads and products behind them, so they are spread over the products.
    for (; k_load + SUBS * KB <= k_end; k0 += SUBS * KB) {
      enter();
#pragma unroll
      for (int u = 0; u < SUBS; ++u) {
        const char* As = smem + slot + u * SUB;
        const unsigned at = lds + slot_load + u * SUB;
        mm_stage<KIND, OpA, OpB, MI, NJ, SWAP>(As, As + OpA::BYTES, wm, wn, q, l15, acc, [&](int g) {
#pragma unroll
          for (int p = g * RATE; p < (g + 1) * RATE && p < PIECES; ++p) {
            if (p < OpA::NV) OpA::load_piece(p, pa, oa, at, wave);
            else OpB::load_piece(p - OpA::NV, pb, ob, at + OpA::BYTES, wave);
          }
        });
        pa += step_a;
        pb += step_b;
      }
      k_load += SUBS * KB;
      slot_load = slot_load + STAGE == LDS ? 0 : slot_load + STAGE;
      slot = slot + STAGE == LDS ? 0 : slot + STAGE;
    }
    for (; k0 < k_end; k0 += SUBS * KB) {   // the last stages: a partial load, or none
      enter();
      if (k_load < k_end) load();
#pragma unroll
      for (int u = 0; u < SUBS; ++u) {
        const char* As = smem + slot + u * SUB;
        if (u == 0 || k0 + u * KB < k_end) mm_stage<KIND, OpA, OpB, MI, NJ, SWAP>(As, As + OpA::BYTES, wm, wn, q, l15, acc, [](int) {});
      }
      slot = slot + STAGE == LDS ? 0 : slot + STAGE;
    }
    lds_stage_barrier<0>();   // the caller may use the memory
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
