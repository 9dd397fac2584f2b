// Orthogonalised updates of matrices by Newton-Schulz products, and the optimizer step built on them
// (newton_schulz.hip).
//
//   X_0 = G / (|G|_F + eps),   X_{k+1} = (a I + b A + c A^2) X_k  with  A = X_k X_k^T
//
// on the orientation with the fewer rows (r x c, r <= c). Singular values of X go through sigma (a + b sigma^2 +
// c sigma^4) per step and are driven towards one; small ones grow by a per step (485-fold over five steps with the
// usual a = 3.4445), and with them every rounding error of the early steps.
#pragma once
#include "common.h"

namespace dtf {

constexpr int kNsMaxSteps = 16;
constexpr int kNsNormParts = 512;   // partial sums of a squared norm

// One matrix. Its workspace (base `ws`, in floats from the call's workspace) holds
//   [kNsNormParts doubles][tau, 63 spare][X, X': rp x cp pairs][A, P: rp x rp pairs]
// with sides padded to multiples of 32 by zeros. A pair is two fp16 numbers h + l in 4 bytes, laid out per row in
// blocks of 32: 32 h, then 32 l. Products in fp32 keep fp32 numbers there instead, in the same 4 bytes.
struct NsMat {
  long long src, out;   // element offset of G, and of the output / parameter
  long long ld, out_ld; // row strides
  long long ws;
  int rows, cols;       // as stored
  int r, c, rp, cp;     // r = min, c = max side; padded
  int tall;             // rows > cols: X = G^T
  int parts, chunk;     // pieces of the norm, elements each
  float scale;          // optimizer: W <- decay W - lr scale O
};
__host__ __device__ inline long long ns_x_floats(const NsMat& m) { return (long long)m.rp * m.cp; }
__host__ __device__ inline long long ns_x(const NsMat& m) { return m.ws + 2 * kNsNormParts + 64; }
__host__ __device__ inline long long ns_a(const NsMat& m) { return ns_x(m) + 2 * ns_x_floats(m); }
__host__ __device__ inline long long ns_p(const NsMat& m) { return ns_a(m) + (long long)m.rp * m.rp; }
__host__ __device__ inline long long ns_floats(const NsMat& m) { return 2 * kNsNormParts + 64 + 2 * ns_x_floats(m) + 2ll * m.rp * m.rp; }
// Fills in everything but the offsets.
void ns_shape(NsMat& m, int rows, int cols);

// Matrices whose steps all run in one workgroup (us that way / by tiles: 10 x 1039 36 / 90, 16 x 2048 43 / 92; what does not fit its registers
// takes 95 - 105 by tiles: 32 x 2048, 64 x 1024).
inline bool ns_small(const NsMat& m) { return m.r <= 16 ? m.c <= 2048 : m.r <= 32 ? m.c <= 1024 : m.r <= 64 && m.c <= 768; }

// A work item. Split X X^T: kn blocks of 32 columns of X from k0 on, its sums into slot `slot`; joining it: kn slots from `slot` on.
struct NsItem { int mat, tile, k0, kn, slot, pad; };
constexpr int kNsSplitTile = 64;
constexpr int kNsSplitMax = 8;
// Parts that X X^T is computed in where `tiles` 64 x 64 tiles in all leave CUs idle: twelve blocks of k each at least.
inline int ns_splits(const NsMat& m, long long tiles) {
  long long s = tiles > 0 ? 512 / tiles : 1;
  if (s > kNsSplitMax) s = kNsSplitMax;
  if (s > m.cp / (12 * 32)) s = m.cp / (12 * 32);
  return s < 1 ? 1 : (int)s;
}

struct NsCoeffs { float a, b, c; };

// Orthogonalises `batch` matrices of one shape: kind (MmKind) fp32, bf16 or fp16.
struct NsArgs {
  int kind, batch, rows, cols, steps;
  const void* g; long long ld, g_stride;       // elements
  void* out; long long out_ld, out_stride;
  double eps;
  NsCoeffs coeffs[kNsMaxSteps];
  float growth;         // a power of two that bounds |a + b s + c s^2| over the values that s takes
  int fp32;             // products of fp32 numbers instead of pairs
};
size_t ns_workspace(const NsArgs& a);
void newton_schulz(const NsArgs& a, void* ws, size_t ws_bytes, hipStream_t stream);

// One step over a flat fp32 parameter buffer. `mats` / `items_*` are device tables that live as long as the optimizer;
// hyper: {lr, momentum, grad_scale, decay, vector lr_t, 1 - beta1, 1 - beta2,
// vector eps} (the differences: 1 - beta2 formed from an fp32 beta2 is off by 1e-5). Matrices: m = momentum m + g, u = g + momentum m (nesterov)
// or m, W = decay W - lr scale NS(u), with g scaled by grad_scale. Vectors (mat < 0 in items_flat): Adam.
struct MuonArgs {
  float* p; const float* g; float* m; float* v;
  const float* hyper;
  const NsMat* mats;
  const NsItem* items_flat; int n_flat;     // (matrix, chunk of it), or (-1 - count, first element / kMuonVecAlign)
  const NsItem* items_small; int n_small;   // matrices that ns_small covers, in none of the lists of tiles
  const NsItem* items_split; int n_split;   // 32 x 32 blocks of every matrix, those of the small ones first:
  int n_out;                                // this many
  const NsItem* items_gram; int n_gram;     // parts of the tiles of X X^T, and their joining (tiles as items_sym)
  const NsItem* items_join;
  const NsItem* items_sym; int n_sym;       // tiles of the r x r products, lower triangle
  const NsItem* items_apply; int n_apply;   // tiles of the r x c products
  int nesterov, steps;
  float* parts;                             // 4096 floats per item of items_gram
  double eps;
  NsCoeffs coeffs[kNsMaxSteps];
  float growth;
  int fp32;                                 // products of fp32 numbers; the tables then hold no small matrices
};
constexpr int kMuonTile = 64;
constexpr int kMuonVecChunk = 1024;   // vector elements per item
constexpr int kMuonVecAlign = 64;     // tensors of a parameter buffer start on multiples of this
void muon_step(const MuonArgs& a, void* ws, hipStream_t stream);

}  // namespace dtf
