// Newton-Schulz orthogonalisation on the fp16 matrix pipe with operands kept as pairs of fp16 numbers.
//
// Precision: five steps amplify a rounding error in a direction of a small singular value 485-fold. Single bf16 or fp16
// operands leave errors of 3 - 30 % / 0.4 - 4 % in the result; h + l with 22 bits and the three products hh + hl + lh (mm_tile.h)
// measures what fp32 products leave, in the norm of the whole (1e-6 - 1e-5 relative, 64x10 to 1024x2048). Everything is kept times the largest
// power of two that fits fp16: X by 2^13, A and P by 2^12. An element keeps its 22 bits down to 2^-16 (X) and 2^-15; below, the pair's smallest step is
// a floor: 2^-38 and 2^-37 at most. Rows or columns far below the others feel it, and fp32 products would not (64 x 256, one row scaled by 1e-2 / 1e-4 / 1e-6:
// its relative error 4e-7 / 3e-6 / 2e-4, by fp32 products 4e-7; 1024 x 4096 1e-6 / 4e-5 / 5e-3, by fp32 products 2e-6).
// A matrix whose norm is far below eps starts with tiny X_0; its part below one is carried apart in tau (a power of two per
// matrix, grown by `growth` per step up to 1), so that the fp16 numbers never see it: X = tau Xs,
//   Xs <- (tau / tau') (a I + b tau^2 As + c tau^4 As^2) Xs.
//
// A caller to whom such rows matter takes products of fp32 numbers (NsArgs::fp32) instead: the same kernels on the fp32 matrix pipe, by tiles for
// every size (us of a call by pairs / fp32 numbers: 6 x 576 x 64 68 / 125, 1024 x 1024 209 / 365, 4096 x 4096 3365 / 10974).
//
// A step is three products: A = X X^T and P = a I + b A + c A^2 are symmetric, so only the tiles on and below the diagonal are
// computed and each is stored twice; X' = P X. The last one writes the output (or updates the parameter) directly.
#include "newton_schulz.h"
#include "mm_tile.h"

namespace dtf {
namespace {

constexpr float kScaleX = 8192.f, kScaleA = 4096.f, kScaleP = 4096.f;   // |X| <= 3.8, |A| <= 3.8^2 and |P| <= 14 stay below fp16's 65504

struct NsDev {
  NsMat one;                   // table == nullptr: `batch` matrices of this shape
  const NsMat* table;
  const NsItem* items;
  int total, per_mat;          // items in all, and per matrix
  long long g_stride, out_stride, ws_stride;
  float* ws;
  const void* g;               // fp32 / bf16 / fp16
  void* out;
  int kind;
  float* m;                    // optimizer: momentum, updated in place; g is then the raw gradient
  float* v;                    // optimizer: second moments of the vectors
  const float* hyper;
  int nesterov;
  double eps;
  int step, last;
  float growth;
  NsCoeffs co;
  int fp32;                    // fp32 numbers in place of pairs
  int splits;                  // parts of a tile of X X^T, table == nullptr
  float* parts;                // their sums, as the accumulators lie in the registers of a workgroup
};

__device__ __forceinline__ void ns_find(const NsDev& a, int t, NsMat& m, int& tile) {
  if (a.table) {
    const NsItem it = a.items[t];
    m = a.table[it.mat];
    tile = it.tile;
  } else {
    const int b = t / a.per_mat;
    tile = t - b * a.per_mat;
    m = a.one;
    m.src += b * a.g_stride;
    m.out += b * a.out_stride;
    m.ws += b * a.ws_stride;
  }
}
__device__ __forceinline__ float ns_read(const void* g, int kind, long long i) {
  if (kind == MM_F32) return reinterpret_cast<const float*>(g)[i];
  if (kind == MM_BF16) return (float)reinterpret_cast<const __bf16*>(g)[i];
  return (float)reinterpret_cast<const _Float16*>(g)[i];
}

// Sum over a block of 256 in a fixed order; every thread gets it.
__device__ __forceinline__ double block_sum(double v, double* scratch) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  return (scratch[0] + scratch[1]) + (scratch[2] + scratch[3]);
}

__device__ __forceinline__ double squares(const uintx4& x, int kind) {
  double s = 0.0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (kind == MM_F32) {
      const double v = __uint_as_float(x[e]);
      s += v * v;
    } else {
      float lo, hi;
      if (kind == MM_BF16) {
        lo = pair_lo(x[e]);
        hi = pair_hi(x[e]);
      } else {
        const unsigned short a = (unsigned short)x[e], b = (unsigned short)(x[e] >> 16);
        lo = (float)__builtin_bit_cast(_Float16, a);
        hi = (float)__builtin_bit_cast(_Float16, b);
      }
      s += (double)lo * lo;
      s += (double)hi * hi;
    }
  }
  return s;
}

// Squares of one chunk of G, in 64 bits (squares of gradients leave fp32's range).
__global__ __launch_bounds__(256) void ns_norm_kernel(NsDev a) {
  __shared__ double scratch[4];
  NsMat m;
  int chunk;
  ns_find(a, blockIdx.x, m, chunk);
  const long long n = (long long)m.rows * m.cols;
  const long long lo = (long long)chunk * m.chunk, hi = min(n, lo + m.chunk);
  const int es = a.kind == MM_F32 ? 4 : 2;
  const char* base = reinterpret_cast<const char*>(a.g) + m.src * es;
  double s = 0.0;
  long long i = lo + threadIdx.x;
  if (m.ld == m.cols && !(reinterpret_cast<uintptr_t>(base) & 15)) {
    // whole rows back to back: 16 bytes a thread, four loads in flight (a chunk is a multiple of 64 elements)
    const int epv = 16 / es;
    const long long v0 = lo / epv, v1 = hi / epv;
    const uintx4* src = reinterpret_cast<const uintx4*>(base);
    for (long long v = v0 + threadIdx.x; v < v1; v += 1024) {
      uintx4 x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) x[u] = v + 256 * u < v1 ? src[v + 256 * u] : uintx4{0, 0, 0, 0};
#pragma unroll
      for (int u = 0; u < 4; ++u) s += squares(x[u], a.kind);
    }
    i = v1 * epv + threadIdx.x;
  }
  for (; i < hi; i += 256) {
    const long long row = i / m.cols;
    const float x = ns_read(a.g, a.kind, m.src + row * m.ld + (i - row * m.cols));
    s += (double)x * x;
  }
  s = block_sum(s, scratch);
  if (threadIdx.x == 0) reinterpret_cast<double*>(a.ws + m.ws)[chunk] = s;
}

// The optimizer's elementwise pass: momentum and the norm of the update for a chunk of a matrix, Adam for a piece of a vector.
__global__ __launch_bounds__(256) void muon_flat_kernel(NsDev a) {
  __shared__ double scratch[4];
  const NsItem it = a.items[blockIdx.x];
  const float mu = a.hyper[1], gs = a.hyper[2];
  const float* g = reinterpret_cast<const float*>(a.g);
  if (it.mat < 0) {
    const int n = -1 - it.mat;
    const float lr_t = a.hyper[4], c1 = a.hyper[5], c2 = a.hyper[6], eps = a.hyper[7];
    float* p = reinterpret_cast<float*>(a.out);
    for (int k = threadIdx.x; k < n; k += 256) {
      const long long i = (long long)it.tile * kMuonVecAlign + k;
      const float x = g[i] * gs;
      const float m = (1.f - c1) * a.m[i] + c1 * x;
      const float v = (1.f - c2) * a.v[i] + c2 * x * x;
      a.m[i] = m;
      a.v[i] = v;
      p[i] -= lr_t * m / (sqrtf(v) + eps);
    }
    return;
  }
  const NsMat m = a.table[it.mat];
  const long long n = (long long)m.rows * m.cols;
  const long long lo = (long long)it.tile * m.chunk, hi = min(n, lo + m.chunk);
  double s = 0.0;
  for (long long i = lo + threadIdx.x; i < hi; i += 256) {
    const float x = g[m.src + i] * gs;
    const float mom = mu * a.m[m.src + i] + x;
    a.m[m.src + i] = mom;
    const float u = a.nesterov ? x + mu * mom : mom;
    s += (double)u * u;
  }
  s = block_sum(s, scratch);
  if (threadIdx.x == 0) reinterpret_cast<double*>(a.ws + m.ws)[it.tile] = s;
}

__device__ __forceinline__ float tau_at(float tau0, float growth, int step) {
  float t = tau0;
  for (int k = 0; k < step; ++k) t = fminf(1.f, t * growth);
  return t;
}

// h and l of four values at (row, col..col+3), col a multiple of 4
__device__ __forceinline__ char* pair_at(float* base, int pitch, int row, int col) {
  return reinterpret_cast<char*>(base + (long long)row * pitch + (col & ~31)) + (col & 31) * 2;
}
__device__ __forceinline__ void pair_split(const floatx4& v, halfx4& h, halfx4& l) {
  h = __builtin_convertvector(v, halfx4);
  const floatx4 rest = v - __builtin_convertvector(h, floatx4);   // exact
  l = __builtin_convertvector(rest, halfx4);
}
__device__ __forceinline__ void pair_store4(float* base, int pitch, int row, int col, const floatx4& v) {
  halfx4 h, l;
  pair_split(v, h, l);
  char* p = pair_at(base, pitch, row, col);
  *reinterpret_cast<halfx4*>(p) = h;
  *reinterpret_cast<halfx4*>(p + 64) = l;
}
__device__ __forceinline__ floatx4 pair_load4(const float* base, int pitch, int row, int col) {
  const char* p = pair_at(const_cast<float*>(base), pitch, row, col);
  return __builtin_convertvector(*reinterpret_cast<const halfx4*>(p), floatx4) + __builtin_convertvector(*reinterpret_cast<const halfx4*>(p + 64), floatx4);
}

// Four values of X, A or P as the products read them: pairs, or fp32 numbers in their place
template <MmKind KIND>
__device__ __forceinline__ void ns_store4(float* base, int pitch, int row, int col, const floatx4& v) {
  if constexpr (KIND == MM_F32) *reinterpret_cast<floatx4*>(base + (long long)row * pitch + col) = v;
  else pair_store4(base, pitch, row, col, v);
}
template <MmKind KIND>
__device__ __forceinline__ floatx4 ns_load4(const float* base, int pitch, int row, int col) {
  if constexpr (KIND == MM_F32) return *reinterpret_cast<const floatx4*>(base + (long long)row * pitch + col);
  else return pair_load4(base, pitch, row, col);
}

// G / (|G| + eps) / tau as pairs, one 32 x 32 block of X per workgroup (transposed on the way where G is tall).
__global__ __launch_bounds__(256) void ns_split_kernel(NsDev a) {
  __shared__ double scratch[4];
  __shared__ float block[32][33];
  NsMat m;
  int tile;
  ns_find(a, blockIdx.x, m, tile);
  float* base = a.ws + m.ws;
  const double* parts = reinterpret_cast<const double*>(base);
  const double ss = block_sum(((int)threadIdx.x < m.parts ? parts[threadIdx.x] : 0.0) + ((int)threadIdx.x + 256 < m.parts ? parts[threadIdx.x + 256] : 0.0), scratch);
  const double norm = sqrt(ss), t = norm / (norm + a.eps);
  // tau: the power of two at or above t, 1 unless the norm is below eps (or is not a number)
  float tau = 1.f;
  if (t < 0.5) tau = t > 1e-37 ? ldexpf(1.f, ilogb(t) + 1) : 1.1754944e-38f;
  const double inv = (double)kScaleX / ((norm + a.eps) * (double)tau);
  const int bc = m.cp / 32, bi = tile / bc, bj = tile - bi * bc;   // block of X
  if (tile == 0 && threadIdx.x == 0) base[2 * kNsNormParts] = tau;
  const int r0 = (m.tall ? bj : bi) * 32, c0 = (m.tall ? bi : bj) * 32;   // block of G
  const float mu = a.m ? a.hyper[1] : 0.f, gs = a.m ? a.hyper[2] : 1.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int y = (threadIdx.x >> 5) + 8 * k, x = threadIdx.x & 31;
    float v = 0.f;
    if (r0 + y < m.rows && c0 + x < m.cols) {
      const long long i = m.src + (long long)(r0 + y) * m.ld + c0 + x;
      v = ns_read(a.g, a.kind, i);
      if (a.m) {
        const float mom = a.m[i];
        v = a.nesterov ? v * gs + mu * mom : mom;
      }
      v = (float)((double)v * inv);
    }
    if (m.tall) block[x][y] = v;
    else block[y][x] = v;
  }
  __syncthreads();
  const int y = threadIdx.x >> 3, x = (threadIdx.x & 7) * 4;
  const floatx4 v = {block[y][x], block[y][x + 1], block[y][x + 2], block[y][x + 3]};
  if (a.fp32) ns_store4<MM_F32>(a.ws + ns_x(m), m.cp, bi * 32 + y, bj * 32 + x, v);
  else ns_store4<MM_PAIR>(a.ws + ns_x(m), m.cp, bi * 32 + y, bj * 32 + x, v);
}

// Element (row, col) of the output, or of the parameter that it updates.
__device__ __forceinline__ void ns_write(const NsDev& a, const NsMat& m, int row, int col, float v, float lr, float decay) {
  const long long at = m.out + (long long)row * m.out_ld + col;
  if (a.m) {
    float* p = reinterpret_cast<float*>(a.out) + at;
    *p = decay * *p - lr * v;
  } else if (a.kind == MM_F32) {
    reinterpret_cast<float*>(a.out)[at] = v;
  } else if (a.kind == MM_BF16) {
    reinterpret_cast<__bf16*>(a.out)[at] = (__bf16)v;
  } else {
    reinterpret_cast<_Float16*>(a.out)[at] = (_Float16)v;
  }
}

enum NsOp { NS_GRAM, NS_POLY, NS_APPLY, NS_GRAM_PART, NS_GRAM_JOIN };

// Tiles: waves over T x T, stages in LDS, 128-byte pieces of k per stage; then what the choice between them goes by: workgroups
// that the card holds at a time, and us per 32 of k of one round of them with half the CUs busy and with all (measured on 576 x 64 to
// 4096 x 4096; us of a whole product by 64 / 128 / 192 / 256: X X^T of 1024 x 4096 36 / 73 / 133 / 216, of 4096 x 4096 322 / 246 / 175 / 221;
// P X of 1024 x 4096 36 / 31 / 47 / 73, of 4096 x 4096 420 / 322 / 337 / 276).
struct NsTileInfo { int t, wgm, wgn, stages, subs, slots; float us_some, us_full; };
constexpr NsTileInfo kNsTiles[] = {{64, 2, 2, 4, 1, 512, 0.26f, 0.5f}, {128, 2, 4, 2, 2, 256, 0.57f, 0.8f}, {192, 2, 4, 2, 1, 256, 1.1f, 1.36f}, {256, 2, 4, 2, 1, 256, 1.7f, 2.15f}};
template <int T>
struct NsTile {
  static constexpr NsTileInfo I = kNsTiles[T / 64 - 1];
  static constexpr int WGM = I.wgm, WGN = I.wgn, STAGES = I.stages, SUBS = I.subs, NT = 64 * WGM * WGN;
};
template <MmKind KIND, int T, bool KCB, bool SWAP>
using NsLoop = MmDirect<KIND, true, KCB, T, T, NsTile<T>::WGM, NsTile<T>::WGN, SWAP, NsTile<T>::STAGES, NsTile<T>::SUBS>;

// One T x T tile of one of the three products.
template <MmKind KIND, NsOp OP, int T>
__global__ __launch_bounds__(NsTile<T>::NT) void ns_product_kernel(NsDev a) {
  extern __shared__ __attribute__((aligned(16))) char ns_smem[];
  const int t = mm_item(blockIdx.x, a.total);
  if (t >= a.total) return;
  NsMat m;
  int tile, k0 = 0, kn = 0;
  long long slot = 0;
  if (OP == NS_GRAM_PART && !a.table) {   // the parts of one range of k together: they share rows of X in an XCD's L2
    const int tiles = a.total / a.splits, part = t / tiles, i = t - part * tiles;
    ns_find(a, i, m, tile);
    const int all = m.cp >> 5;
    k0 = all * part / a.splits;
    kn = all * (part + 1) / a.splits - k0;
    slot = (long long)i * a.splits + part;
  } else {
    ns_find(a, t, m, tile);
    if (a.table) {
      k0 = a.items[t].k0;
      kn = a.items[t].kn;
      slot = a.items[t].slot;
    } else {
      kn = a.splits;
      slot = (long long)t * a.splits;
    }
  }
  int tx, ty;
  if (OP == NS_APPLY) {
    mm_tile_of(tile, (m.cp + T - 1) / T, (m.rp + T - 1) / T, tx, ty);
  } else {   // lower triangle, row by row
    ty = (int)((sqrtf(8.f * tile + 1.f) - 1.f) * 0.5f);
    while ((ty + 1) * (ty + 2) / 2 <= tile) ++ty;
    while (ty * (ty + 1) / 2 > tile) --ty;
    tx = tile - ty * (ty + 1) / 2;
  }
  const int m0 = ty * T, n0 = tx * T;
  float *xa = a.ws + ns_x(m), *xb = xa + ns_x_floats(m);
  if (a.step & 1) { float* s = xa; xa = xb; xb = s; }
  float *A = a.ws + ns_a(m), *P = a.ws + ns_p(m);

  constexpr int WGM = NsTile<T>::WGM, WGN = NsTile<T>::WGN, MI = T / WGM / 16, NJ = T / WGN / 16;
  floatx4 acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, l15 = lane & 15;
  const int wm = (wave / WGN) * (T / WGM), wn = (wave % WGN) * (T / WGN);

  if (OP != NS_APPLY) {
    constexpr bool GRAM = OP != NS_POLY;
    if constexpr (OP == NS_GRAM_JOIN) {
      const floatx4* s = reinterpret_cast<const floatx4*>(a.parts) + slot * (MI * NJ * NsTile<T>::NT) + threadIdx.x;
      for (int p = 0; p < kn; ++p)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j) acc[i][j] += s[((p * MI + i) * NJ + j) * NsTile<T>::NT];
    } else {
      const int pitch = GRAM ? m.cp : m.rp;
      const char* s = reinterpret_cast<const char*>(GRAM ? xa : A);
      const int kb = OP == NS_GRAM_PART ? k0 * 32 : 0, ke = OP == NS_GRAM_PART ? (k0 + kn) * 32 : pitch;
      NsLoop<KIND, T, true, true>::run(MmOperands{s, s, pitch, pitch, m.rp, m.rp}, m0, n0, kb, ke, ns_smem, acc);
    }
    if constexpr (OP == NS_GRAM_PART) {
      floatx4* d = reinterpret_cast<floatx4*>(a.parts) + slot * (MI * NJ * NsTile<T>::NT) + threadIdx.x;
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) d[(i * NJ + j) * NsTile<T>::NT] = acc[i][j];
      return;
    }
    float* dst = GRAM ? A : P;
    float ca = 0.f, cb = 0.f, cc;   // value = ca I + cb A + cc acc
    if (GRAM) {
      cc = kScaleA / (kScaleX * kScaleX);
    } else {
      const float tau = tau_at(a.ws[m.ws + 2 * kNsNormParts], a.growth, a.step), next = fminf(1.f, tau * a.growth);
      const float s1 = kScaleP * (tau / next), t2 = tau * tau;
      ca = s1 * a.co.a;
      cb = s1 * a.co.b * t2 * (1.f / kScaleA);
      cc = s1 * a.co.c * t2 * t2 * (1.f / (kScaleA * kScaleA));
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int mm = m0 + wm + i * 16 + l15;
      if (mm >= m.rp) continue;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int nn = n0 + wn + j * 16 + 4 * q;
        if (nn >= m.rp) continue;
        floatx4 v = acc[i][j] * cc;
        if (OP == NS_POLY) {
          v += ns_load4<KIND>(A, m.rp, mm, nn) * cb;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (mm == nn + e && mm < m.r) v[e] += ca;
        }
        ns_store4<KIND>(dst, m.rp, mm, nn, v);
        if (m0 == n0) continue;
        // the mirrored tile
        if constexpr (KIND == MM_F32) {
#pragma unroll
          for (int e = 0; e < 4; ++e) dst[(long long)(nn + e) * m.rp + mm] = v[e];
        } else {
          halfx4 h, l;
          pair_split(v, h, l);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            _Float16* p = reinterpret_cast<_Float16*>(dst + (long long)(nn + e) * m.rp + (mm & ~31)) + (mm & 31);
            p[0] = h[e];
            p[32] = l[e];
          }
        }
      }
    }
    return;
  }

  const MmOperands o{reinterpret_cast<const char*>(P), reinterpret_cast<const char*>(xa), m.rp, m.cp, m.rp, m.cp};
  if (!a.last || !m.tall) NsLoop<KIND, T, false, true>::run(o, m0, n0, 0, m.rp, ns_smem, acc);
  else NsLoop<KIND, T, false, false>::run(o, m0, n0, 0, m.rp, ns_smem, acc);
  if (!a.last) {
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int mm = m0 + wm + i * 16 + l15;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int nn = n0 + wn + j * 16 + 4 * q;
        if (mm < m.rp && nn < m.cp) ns_store4<KIND>(xb, m.cp, mm, nn, acc[i][j] * (1.f / kScaleP));
      }
    }
    return;
  }
  // The output, in G's orientation: a lane holds four consecutive elements of a row of it.
  const float tau = tau_at(a.ws[m.ws + 2 * kNsNormParts], a.growth, a.step + 1);
  const float f = 1.f / (kScaleP * kScaleX);   // tau apart: their product can leave fp32's normal range
  const float lr = a.m ? a.hyper[0] * m.scale : 0.f, decay = a.m ? a.hyper[3] : 0.f;
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int row = m.tall ? n0 + wn + j * 16 + l15 : m0 + wm + i * 16 + l15;
      const int col = (m.tall ? m0 + wm + i * 16 : n0 + wn + j * 16) + 4 * q;
      if (row >= m.rows) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < m.cols) ns_write(a, m, row, col + e, acc[i][j][e] * f * tau, lr, decay);
    }
}

// ---- Small matrices: all steps in one workgroup of eight waves, X in registers.
//
// A wave owns up to four blocks of 32 columns of X, as the fragments that X X^T needs: lane (q, l15) has row 16 i + l15 and, of block b, the
// columns 32 b + {4 q .. 4 q + 3, 16 + 4 q .. 16 + 4 q + 3} (any order of k serves a product whose operands share it, and this is the
// order in which P X leaves the matrix pipe). A step: the waves' parts of X X^T are added in wave order in LDS, P is formed there, and
// each wave turns its blocks round through LDS (transposed reads), multiplies them by P and has the next X. The kernel starts from
// the pairs that ns_split_kernel wrote and leaves pairs for ns_out_kernel: reading and writing the matrices themselves here ran as slowly as
// one CU can (35 us of a 6 x 576 x 64 call).
constexpr int kSmallWaves = 8, kSmallPitch = 272, kTurnPitch = 144;   // bytes per row of A and P, and of a block being turned
constexpr int kSmallPart = 10 * 1024;                                 // bytes of a wave's part of X X^T
constexpr int kSmallLds = kSmallWaves * kSmallPart + 2 * 64 * kSmallPitch;
static_assert(64 * kTurnPitch <= kSmallPart && kSmallLds <= (int)kLdsBudget, "LDS of the small-matrix kernel");

// h and l of four values of row `row` of A or P, columns col .. col + 3
__device__ __forceinline__ void small_store4(char* mat, int row, int col, const floatx4& v) {
  halfx4 h, l;
  pair_split(v, h, l);
  char* p = mat + row * kSmallPitch + (col >> 5) * 128 + (col & 31) * 2;
  *reinterpret_cast<halfx4*>(p) = h;
  *reinterpret_cast<halfx4*>(p + 64) = l;
}
// four values of a symmetric matrix in both places
__device__ __forceinline__ void small_store_sym(char* mat, int row, int col, const floatx4& v, bool mirror) {
  small_store4(mat, row, col, v);
  if (!mirror) return;
  halfx4 h, l;
  pair_split(v, h, l);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    _Float16* p = reinterpret_cast<_Float16*>(mat + (col + e) * kSmallPitch + (row >> 5) * 128) + (row & 31);
    p[0] = h[e];
    p[32] = l[e];
  }
}

template <int RT, int NB>   // 16-row tiles of X, blocks of a wave (those past X's columns are zeros)
__device__ __forceinline__ void ns_small_run(const NsDev& a, const NsMat& m, const NsCoeffs* co, int steps, char* smem) {
  constexpr int KBS = (RT + 1) / 2, TILES = RT * (RT + 1) / 2;   // 32-row blocks of X, tiles on and below the diagonal
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, l15 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  char *parts = smem, *A = smem + kSmallWaves * kSmallPart, *P = A + 64 * kSmallPitch;
  char* mine = parts + wave * kSmallPart;
  for (int e = tid; e < 2 * 64 * kSmallPitch / 16; e += 64 * kSmallWaves) reinterpret_cast<uintx4*>(A)[e] = uintx4{0, 0, 0, 0};

  float* X = a.ws + ns_x(m);
  Frag F[RT][NB];
#pragma unroll
  for (int kb = 0; kb < NB; ++kb)
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int row = 16 * i + l15, col = 32 * (kb * kSmallWaves + wave);
      uintx2 v[4] = {};
      if (row < m.rp && col < m.cp) {
        const char* p = reinterpret_cast<const char*>(X + (long long)row * m.cp + col) + q * 8;
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = *reinterpret_cast<const uintx2*>(p + 32 * u);   // h, h, l, l
      }
      F[i][kb].h = uintx4{v[0][0], v[0][1], v[1][0], v[1][1]};
      F[i][kb].l = uintx4{v[2][0], v[2][1], v[3][0], v[3][1]};
    }
  float tau = a.ws[m.ws + 2 * kNsNormParts];
  __syncthreads();

#pragma unroll 1
  for (int step = 0; step < steps; ++step) {
    // the wave's part of X X^T: lane (q, l15) of a tile has row 16 i + l15, columns 16 j + 4 q ..
    {
      floatx4 acc[TILES];
#pragma unroll
      for (int k = 0; k < TILES; ++k) acc[k] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int s = 0; s < 3; ++s)
#pragma unroll
          for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j <= i; ++j) mm_mfma<MM_PAIR>(s, F[j][kb], F[i][kb], acc[i * (i + 1) / 2 + j]);
#pragma unroll
      for (int k = 0; k < TILES; ++k) *reinterpret_cast<floatx4*>(mine + k * 1024 + lane * 16) = acc[k];
    }
    __syncthreads();
    for (int e = tid; e < TILES * 64; e += 64 * kSmallWaves) {
      floatx4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kSmallWaves; ++w) s += *reinterpret_cast<const floatx4*>(parts + w * kSmallPart + e * 16);
      const int k = e >> 6, i = k >= 6 ? 3 : k >= 3 ? 2 : k >= 1 ? 1 : 0, j = k - i * (i + 1) / 2;
      small_store_sym(A, 16 * i + (e & 15), 16 * j + 4 * ((e >> 4) & 3), s * (kScaleA / (kScaleX * kScaleX)), i != j);
    }
    __syncthreads();
    const float next = fminf(1.f, tau * a.growth);
    {
      const float s1 = kScaleP * (tau / next), t2 = tau * tau;
      const float ca = s1 * co[step].a, cb = s1 * co[step].b * t2 * (1.f / kScaleA), cc = s1 * co[step].c * t2 * t2 * (1.f / (kScaleA * kScaleA));
      for (int k = wave; k < TILES; k += kSmallWaves) {
        const int i = k >= 6 ? 3 : k >= 3 ? 2 : k >= 1 ? 1 : 0, j = k - i * (i + 1) / 2;
        floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kb = 0; kb < KBS; ++kb) {
          auto frag = [&](int tile) {
            const char* p = A + (16 * tile + l15) * kSmallPitch + kb * 128 + q * 16;
            Frag f;
            f.h = *reinterpret_cast<const uintx4*>(p);
            f.l = *reinterpret_cast<const uintx4*>(p + 64);
            return f;
          };
          mm_mfma_all<MM_PAIR>(frag(j), frag(i), acc);
        }
        const int row = 16 * i + l15, col = 16 * j + 4 * q;
        const char* p = A + row * kSmallPitch + (col >> 5) * 128 + (col & 31) * 2;
        floatx4 x = acc * cc + (__builtin_convertvector(*reinterpret_cast<const halfx4*>(p), floatx4) +
                                __builtin_convertvector(*reinterpret_cast<const halfx4*>(p + 64), floatx4)) * cb;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (row == col + e && row < m.r) x[e] += ca;
        small_store_sym(P, row, col, x, i != j);
      }
    }
    // The blocks, rows as lines, into the wave's own memory (free since the barrier behind the sums) and back with columns as lanes.
    Frag G[NB][KBS][2];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        char* p = mine + (16 * i + l15) * kTurnPitch + q * 8;
        *reinterpret_cast<uintx2*>(p) = uintx2{F[i][kb].h[0], F[i][kb].h[1]};
        *reinterpret_cast<uintx2*>(p + 32) = uintx2{F[i][kb].h[2], F[i][kb].h[3]};
        *reinterpret_cast<uintx2*>(p + 64) = uintx2{F[i][kb].l[0], F[i][kb].l[1]};
        *reinterpret_cast<uintx2*>(p + 96) = uintx2{F[i][kb].l[2], F[i][kb].l[3]};
      }
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");   // this wave's lines are there; the reads stay behind them
#pragma unroll
      for (int kk = 0; kk < KBS; ++kk)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const unsigned char* p = reinterpret_cast<const unsigned char*>(mine) + (32 * kk + 4 * q + (l15 >> 2)) * kTurnPitch + c * 32 + (l15 & 3) * 8;
          const uintx2 h0 = lds_read_tr(p), l0 = lds_read_tr(p + 64);
          uintx2 h1 = {0, 0}, l1 = {0, 0};
          if (RT > 1) {
            h1 = lds_read_tr(p + 16 * kTurnPitch);
            l1 = lds_read_tr(p + 16 * kTurnPitch + 64);
          }
          G[kb][kk][c].h = uintx4{h0[0], h0[1], h1[0], h1[1]};
          G[kb][kk][c].l = uintx4{l0[0], l0[1], l1[0], l1[1]};
        }
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");   // read before the next block's lines are written
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      Frag w[KBS];
#pragma unroll
      for (int kk = 0; kk < KBS; ++kk) {
        const char* p = P + (16 * i + l15) * kSmallPitch + kk * 128 + q * 8;
        const uintx2 h0 = *reinterpret_cast<const uintx2*>(p), h1 = *reinterpret_cast<const uintx2*>(p + 32);
        const uintx2 l0 = *reinterpret_cast<const uintx2*>(p + 64), l1 = *reinterpret_cast<const uintx2*>(p + 96);
        w[kk].h = uintx4{h0[0], h0[1], h1[0], h1[1]};
        w[kk].l = uintx4{l0[0], l0[1], l1[0], l1[1]};
      }
      floatx4 acc[NB][2];
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) acc[kb][0] = acc[kb][1] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KBS; ++kk)
#pragma unroll
        for (int s = 0; s < 3; ++s)
#pragma unroll
          for (int kb = 0; kb < NB; ++kb)
#pragma unroll
            for (int c = 0; c < 2; ++c) mm_mfma<MM_PAIR>(s, G[kb][kk][c], w[kk], acc[kb][c]);
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) {
        halfx4 h[2], l[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) pair_split(acc[kb][c] * (1.f / kScaleP), h[c], l[c]);
        F[i][kb].h = __builtin_bit_cast(uintx4, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
        F[i][kb].l = __builtin_bit_cast(uintx4, __builtin_shufflevector(l[0], l[1], 0, 1, 2, 3, 4, 5, 6, 7));
      }
    }
    tau = next;
    __syncthreads();   // the waves' memory, A and P are free
  }
#pragma unroll
  for (int kb = 0; kb < NB; ++kb)
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int row = 16 * i + l15, col = 32 * (kb * kSmallWaves + wave);
      if (row < m.rp && col < m.cp) {
        char* p = reinterpret_cast<char*>(X + (long long)row * m.cp + col) + q * 8;
        *reinterpret_cast<uintx2*>(p) = uintx2{F[i][kb].h[0], F[i][kb].h[1]};
        *reinterpret_cast<uintx2*>(p + 32) = uintx2{F[i][kb].h[2], F[i][kb].h[3]};
        *reinterpret_cast<uintx2*>(p + 64) = uintx2{F[i][kb].l[0], F[i][kb].l[1]};
        *reinterpret_cast<uintx2*>(p + 96) = uintx2{F[i][kb].l[2], F[i][kb].l[3]};
      }
    }
  if (tid == 0) a.ws[m.ws + 2 * kNsNormParts] = tau;
}
struct NsSmallArgs { NsDev d; int steps; NsCoeffs co[kNsMaxSteps]; };
__global__ __launch_bounds__(64 * kSmallWaves) void ns_small_kernel(NsSmallArgs a) {
  extern __shared__ __attribute__((aligned(16))) char ns_smem[];
  NsMat m;
  int tile;
  ns_find(a.d, blockIdx.x, m, tile);
  const int nb = (m.c + 32 * kSmallWaves - 1) / (32 * kSmallWaves);
#define NS_SMALL(RT, NB) ns_small_run<RT, NB>(a.d, m, a.co, a.steps, ns_smem)
  if (m.r <= 16) {
    if (nb == 1) NS_SMALL(1, 1);
    else if (nb <= 4) NS_SMALL(1, 4);
    else NS_SMALL(1, 8);
  } else if (m.r <= 32) {
    if (nb <= 2) NS_SMALL(2, 2);
    else NS_SMALL(2, 4);
  } else if (nb == 1) {
    NS_SMALL(4, 1);
  } else {
    NS_SMALL(4, 3);
  }
#undef NS_SMALL
}
// What ns_small_kernel left, into the output or the parameter: one 32 x 32 block of X per workgroup.
__global__ __launch_bounds__(256) void ns_out_kernel(NsDev a) {
  __shared__ float block[32][33];
  NsMat m;
  int tile;
  ns_find(a, blockIdx.x, m, tile);
  const int bc = m.cp / 32, bi = tile / bc, bj = tile - bi * bc;
  {
    const int y = threadIdx.x >> 3, x = (threadIdx.x & 7) * 4;
    const floatx4 v = pair_load4(a.ws + ns_x(m), m.cp, bi * 32 + y, bj * 32 + x);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (m.tall) block[x + e][y] = v[e];
      else block[y][x + e] = v[e];
    }
  }
  __syncthreads();
  const float f = 1.f / kScaleX, tau = a.ws[m.ws + 2 * kNsNormParts];
  const float lr = a.m ? a.hyper[0] * m.scale : 0.f, decay = a.m ? a.hyper[3] : 0.f;
  const int r0 = (m.tall ? bj : bi) * 32, c0 = (m.tall ? bi : bj) * 32;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int y = (threadIdx.x >> 5) + 8 * k, x = threadIdx.x & 31;
    if (r0 + y < m.rows && c0 + x < m.cols) ns_write(a, m, r0 + y, c0 + x, block[y][x] * f * tau, lr, decay);
  }
}

template <MmKind KIND>
void gram_in_parts_as(const char* part, const char* join, const NsDev& p, const NsDev& j, hipStream_t stream) {
  constexpr int T = kNsSplitTile;
  const size_t lds = NsLoop<KIND, T, true, true>::LDS;
  launch(part, ns_product_kernel<KIND, NS_GRAM_PART, T>, dim3((unsigned)((p.total + 7) / 8 * 8)), dim3(NsTile<T>::NT), lds, stream, p);
  launch(join, ns_product_kernel<KIND, NS_GRAM_JOIN, T>, dim3((unsigned)((j.total + 7) / 8 * 8)), dim3(NsTile<T>::NT), 0, stream, j);
}
void gram_in_parts(const char* part, const char* join, const NsDev& p, const NsDev& j, hipStream_t stream) {
  if (p.fp32) gram_in_parts_as<MM_F32>(part, join, p, j, stream);
  else gram_in_parts_as<MM_PAIR>(part, join, p, j, stream);
}
template <NsOp OP>
void product(const char* name, NsDev d, int tile, hipStream_t stream) {
  auto as = [&](auto kernel, int threads, size_t lds) { launch(name, kernel, dim3((unsigned)((d.total + 7) / 8 * 8)), dim3(threads), lds, stream, d); };
  if (d.fp32) as(ns_product_kernel<MM_F32, OP, 64>, NsTile<64>::NT, NsLoop<MM_F32, 64, true, true>::LDS);
  else if (tile == 256) as(ns_product_kernel<MM_PAIR, OP, 256>, 512, NsLoop<MM_PAIR, 256, true, true>::LDS);
  else if (tile == 192) as(ns_product_kernel<MM_PAIR, OP, 192>, 512, NsLoop<MM_PAIR, 192, true, true>::LDS);
  else if (tile == 128) as(ns_product_kernel<MM_PAIR, OP, 128>, NsTile<128>::NT, NsLoop<MM_PAIR, 128, true, true>::LDS);
  else as(ns_product_kernel<MM_PAIR, OP, 64>, NsTile<64>::NT, NsLoop<MM_PAIR, 64, true, true>::LDS);
}

int sym_tiles(const NsMat& m, int T) { const int t = ceil_div(m.rp, T); return t * (t + 1) / 2; }
// The tile with the least estimated time: rounds of workgroups times k.
template <class Count>
int pick_tile(Count&& count, int k_stages, int fp32) {
  // fp32 numbers: 64 x 64 for every size (us of a call of five steps by 64 / 128: 512 x 512 214 / 537, 1024 x 4096 745 / 1858, 2048 x 2048 1717 / 1878,
  // 4096 x 4096 10974 / 11984; 128 for P X of the last two alone would gain 0 and 4 %)
  if (fp32) return 64;
  int best = 64;
  float least = 0.f;
  for (const NsTileInfo& i : kNsTiles) {
    const long long n = count(i.t);
    const float us = (float)k_stages * (float)((n + i.slots - 1) / i.slots) * (n <= 160 ? i.us_some : i.us_full);
    if (i.t == 64 || us < least) { best = i.t; least = us; }
  }
  return best;
}
int apply_tiles(const NsMat& m, int T) { return ceil_div(m.rp, T) * ceil_div(m.cp, T); }

}  // namespace

void ns_shape(NsMat& m, int rows, int cols) {
  m.rows = rows; m.cols = cols;
  m.tall = rows > cols;
  if (rows > (1 << 30) || cols > (1 << 30)) throw std::runtime_error("newton_schulz: a dimension passes 2^30");
  m.r = rows < cols ? rows : cols;
  m.c = rows < cols ? cols : rows;
  m.rp = ceil_div(m.r, 32) * 32;
  m.cp = ceil_div(m.c, 32) * 32;
  // the rows of a tile are found by 32-bit byte offsets from its first
  if ((long long)(m.rp < 256 ? m.rp : 256) * m.cp > 1ll << 30) throw std::runtime_error("newton_schulz: the rows are too long");
  const long long n = (long long)rows * cols;
  const long long chunk = (n + kNsNormParts - 1) / kNsNormParts;
  m.chunk = (int)(((chunk < 2048 ? 2048 : chunk) + 63) / 64 * 64);
  m.parts = (int)((n + m.chunk - 1) / m.chunk);
}

namespace {
// parts of X X^T of a uniform call, 1 where a tile kernel does it alone
int gram_splits(const NsMat& m, int batch, int fp32) {
  const long long tiles = (long long)sym_tiles(m, kNsSplitTile) * batch;
  if ((ns_small(m) && !fp32) || pick_tile([&](int T) { return (long long)sym_tiles(m, T) * batch; }, m.cp / 32, fp32) != kNsSplitTile) return 1;
  return ns_splits(m, tiles);
}
}  // namespace

size_t ns_workspace(const NsArgs& a) {
  NsMat m{};
  ns_shape(m, a.rows, a.cols);
  const int s = gram_splits(m, a.batch, a.fp32);
  const long long parts = s > 1 ? (long long)sym_tiles(m, kNsSplitTile) * a.batch * s * kNsSplitTile * kNsSplitTile : 0;
  return (size_t)(ns_floats(m) * a.batch + parts) * sizeof(float);
}

void newton_schulz(const NsArgs& a, void* ws, size_t ws_bytes, hipStream_t stream) {
  if (a.batch <= 0 || a.rows <= 0 || a.cols <= 0) return;
  if (a.steps < 1 || a.steps > kNsMaxSteps) throw std::runtime_error("newton_schulz: 1..16 steps");
  if (ns_workspace(a) > ws_bytes || !ws || (reinterpret_cast<uintptr_t>(ws) & 15)) throw std::runtime_error("newton_schulz: workspace too small or unaligned");
  NsDev d{};
  ns_shape(d.one, a.rows, a.cols);
  d.one.ld = a.ld; d.one.out_ld = a.out_ld;
  d.g = a.g; d.out = a.out; d.kind = a.kind;
  d.g_stride = a.g_stride; d.out_stride = a.out_stride; d.ws_stride = ns_floats(d.one);
  d.ws = reinterpret_cast<float*>(ws);
  d.eps = a.eps; d.growth = a.growth; d.fp32 = a.fp32;
  const NsMat& m = d.one;
  auto with = [&](int per) {
    if ((long long)per * a.batch > 0x7ffff8) throw std::runtime_error("newton_schulz: too many tiles");   // x 512 threads: below 2^32
    NsDev x = d;
    x.per_mat = per;
    x.total = per * a.batch;
    return x;
  };
  const NsDev n = with(m.parts);
  launch("ns_norm", ns_norm_kernel, dim3(n.total), dim3(256), 0, stream, n);
  const NsDev s = with((m.rp / 32) * (m.cp / 32));
  launch("ns_split", ns_split_kernel, dim3(s.total), dim3(256), 0, stream, s);
  if (ns_small(m) && !a.fp32) {
    NsSmallArgs k{};
    k.d = with(1);
    k.steps = a.steps;
    for (int i = 0; i < a.steps; ++i) k.co[i] = a.coeffs[i];
    launch("ns_small", ns_small_kernel, dim3(k.d.total), dim3(64 * kSmallWaves), kSmallLds, stream, k);
    launch("ns_out", ns_out_kernel, dim3(s.total), dim3(256), 0, stream, s);
    return;
  }
  // X X^T of few rows and many columns: in parts, which are added in order (us of 512 x 3136 26 -> 15, of 1024 x 4096 36 -> 26)
  const int splits = gram_splits(m, a.batch, a.fp32);
  d.splits = splits;
  d.parts = d.ws + ns_floats(m) * a.batch;
  const int tg = pick_tile([&](int T) { return (long long)sym_tiles(m, T) * a.batch; }, m.cp / 32, a.fp32);
  const int tp = pick_tile([&](int T) { return (long long)sym_tiles(m, T) * a.batch; }, m.rp / 32, a.fp32);
  const int ta = pick_tile([&](int T) { return (long long)apply_tiles(m, T) * a.batch; }, m.rp / 32, a.fp32);
  for (int k = 0; k < a.steps; ++k) {
    d.step = k;
    d.last = k == a.steps - 1;
    d.co = a.coeffs[k];
    if (splits > 1) {
      NsDev p = with(sym_tiles(m, kNsSplitTile)), j = p;
      p.total *= splits;
      gram_in_parts("ns_gram_part", "ns_gram_join", p, j, stream);
    } else {
      product<NS_GRAM>("ns_gram", with(sym_tiles(m, tg)), tg, stream);
    }
    product<NS_POLY>("ns_poly", with(sym_tiles(m, tp)), tp, stream);
    product<NS_APPLY>("ns_apply", with(apply_tiles(m, ta)), ta, stream);
  }
}

void muon_step(const MuonArgs& a, void* ws, hipStream_t stream) {
  if (a.steps < 1 || a.steps > kNsMaxSteps) throw std::runtime_error("muon_step: 1..16 steps");
  NsDev d{};
  d.table = a.mats;
  d.ws = reinterpret_cast<float*>(ws);
  d.g = a.g; d.out = a.p; d.m = a.m; d.v = a.v; d.hyper = a.hyper; d.kind = MM_F32;
  d.nesterov = a.nesterov; d.eps = a.eps; d.growth = a.growth; d.parts = a.parts; d.fp32 = a.fp32;
  auto with = [&](const NsItem* items, int total) {
    NsDev x = d;
    x.items = items;
    x.total = total;
    return x;
  };
  if (a.n_flat > 0) launch("muon_flat", muon_flat_kernel, dim3(a.n_flat), dim3(256), 0, stream, with(a.items_flat, a.n_flat));
  if (a.n_split <= 0) return;
  launch("muon_split", ns_split_kernel, dim3(a.n_split), dim3(256), 0, stream, with(a.items_split, a.n_split));
  if (a.n_small > 0) {
    NsSmallArgs s{};
    s.d = with(a.items_small, a.n_small);
    s.steps = a.steps;
    for (int k = 0; k < a.steps; ++k) s.co[k] = a.coeffs[k];
    launch("muon_small", ns_small_kernel, dim3(a.n_small), dim3(64 * kSmallWaves), kSmallLds, stream, s);
    launch("muon_out", ns_out_kernel, dim3(a.n_out), dim3(256), 0, stream, with(a.items_split, a.n_out));
  }
  if (a.n_sym <= 0) return;
  for (int k = 0; k < a.steps; ++k) {
    d.step = k;
    d.last = k == a.steps - 1;
    d.co = a.coeffs[k];
    gram_in_parts("muon_gram_part", "muon_gram_join", with(a.items_gram, a.n_gram), with(a.items_join, a.n_sym), stream);
    product<NS_POLY>("muon_poly", with(a.items_sym, a.n_sym), kMuonTile, stream);
    product<NS_APPLY>("muon_apply", with(a.items_apply, a.n_apply), kMuonTile, stream);
  }
}

}  // namespace dtf
