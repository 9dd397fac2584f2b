// Dense layers y = act(x W + b) + residual in fp32, bf16 and fp16, and their gradients: the host side, which
// picks a product kernel (linear_tile.h) and lays out the workspace.
//
// Per output element the forward pass costs 2 K flops and the epilogue rides in the product's registers: bias, the
// stored pre-activation, the activation and the residual cost their own bytes and no launch. The backward pass
// is one pass over dy and the pre-activation (dz and the column sums) and two products.
#include "linear_tile.h"
#include <math.h>

namespace dtf {
namespace {

// Rows that the few-rows kernels take; more go through 32 x 64 tiles. 4096 x 4096, us by rows kernel / tiles: bf16 W [K,N] 1 row 10.6 / 9.7 (1024 x 1024
// 5.2 / 6.5), 2 rows 12.0 / 9.9; W [N,K] 2 rows 8.6 / 9.9, 3 rows 10.6 / 9.9; fp32 W [K,N] 4 rows 16.6 / 20.1, 5 rows 18.7 / 20.2 (1024 x 1024 10.8 / 8.5).
// One 16-bit row over W [K,N] thus goes by the small weight: the large one would be 0.9 us sooner by tiles.
int lin_rows_max(const MmProduct& p) { return p.kind == MM_F32 ? 4 : p.kc_b ? 2 : 1; }
constexpr size_t kMaxPartialBytes = 256ull << 20;   // partial sums of a split product

const LinLaunch& lin_launch(int kind) {
  switch (kind) {
    case MM_F32: return lin_launch_f32();
    case MM_BF16: return lin_launch_bf16();
    case MM_F16: return lin_launch_f16();
    default: throw std::runtime_error("linear: unknown element type");
  }
}
int elem_bytes(int kind) { return kind == MM_F32 ? 4 : 2; }
bool aligned_to(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
size_t round_up(size_t v) { return (v + 255) & ~(size_t)255; }

struct Plan {
  int variant, splits, k_per_split, gx, gy;
  long long N4;
  int copy_a, copy_b;            // the operand goes through a padded copy
  long long ld_a, ld_b;          // leading dimension of the copy
  size_t bytes, bytes_a, bytes_b;   // partial sums, copies
};
// The larger the tile the less is loaded per product, but it takes about a tile per CU to use the card; and k in parts fills it with fewer
// tiles, for the price of the parts' way through memory and a second launch. The choice goes by an estimate of the time: what a
// workgroup takes for a stage of 128 bytes of k, alone on its CU and with as many as fit, and what a launch takes besides, in us: a fit to times of every
// tile and number of parts over sizes of 9 to 8192 (bench/linear_sweep.py times what it picks against the library's product: 0.84 of its time
// in the geometric mean over 110 sizes, 0.78 of aligned ones).
struct TileCost { int variant, per_cu; float alone, full, launch; };
constexpr TileCost kTileCosts[2][4] = {
    {{LIN_64, 2, 0.58f, 1.11f, 4.7f}, {LIN_128, 1, 1.8f, 1.87f, 5.9f}, {LIN_256, 1, 7.0f, 7.0f, 11.3f}, {LIN_32, 3, 0.33f, 0.89f, 4.4f}},   // fp32
    {{LIN_64, 2, 0.24f, 0.5f, 4.3f}, {LIN_128, 1, 0.45f, 0.7f, 5.1f}, {LIN_256, 1, 1.22f, 1.32f, 9.7f}, {LIN_32, 3, 0.16f, 0.53f, 4.0f}}};  // 16 bits
// Through registers, 128 x 128: fp32 and 16 bits
constexpr TileCost kRegsCost[2] = {{LIN_REGS, 1, 2.6f, 3.f, 5.f}, {LIN_REGS, 1, 1.8f, 2.f, 5.f}};
constexpr int kSplitChoices[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128, 256};
struct TilePick { int variant, splits; float us; };
void pick_splits(const MmProduct& p, const TileCost& c, TilePick& best) {
  const int stages = ceil_div(p.K, 128 / elem_bytes(p.kind));
  const long long tiles = (long long)ceil_div(p.M, kLinTiles[c.variant].tm) * ceil_div(p.N, kLinTiles[c.variant].tn);
  const float plane = (float)p.M * (float)p.N * 4.f;   // bytes of a part
  for (int splits : kSplitChoices) {
    if (splits > 1 && (stages < 2 * splits || tiles * splits > 2048 || plane * splits > (float)kMaxPartialBytes)) break;
    const int per = ceil_div(stages, splits);
    const float n = (float)((tiles * splits + 255) / 256);   // workgroups of the busiest CU
    const float stage = c.per_cu > 1 ? fmaxf(c.alone, c.full * n / c.per_cu) : tiles * splits <= 154 ? c.alone : c.full * n;
    const float us = c.launch + stage * per + (splits > 1 ? 0.8f + 0.25f * splits + splits * plane * 4e-7f : 0.f);
    if (us < best.us) best = TilePick{c.variant, splits, us};
  }
}
TilePick pick_tile(const MmProduct& p) {
  TilePick best{LIN_64, 1, 3e38f};
  for (const TileCost& c : kTileCosts[p.kind != MM_F32])
    if (c.variant != LIN_32 || (p.kc_a && p.M <= 256)) pick_splits(p, c, best);
  return best;
}
// Sizes and indices of a tile or a stage past a dimension's end are 32 bits.
void check_sizes(long long M, long long N, long long K) {
  constexpr long long most = (1ll << 31) - 65536;
  if (M > most || N > most || K > most) throw std::runtime_error("linear: a dimension passes 2^31 - 65536");
}
// A launch has fewer than 2^32 threads.
void check_blocks(long long blocks, int threads) {
  if (blocks * threads > 0xffffffffll) throw std::runtime_error("linear: the product has too many tiles");
}
Plan plan_of(const MmProduct& p) {
  Plan l{};
  check_sizes(p.M, p.N, p.K);
  const int es = elem_bytes(p.kind), epc = 16 / es;
  // An operand can be loaded 16 bytes at a time if its lines start and end on multiples of them
  auto direct = [&](const void* base, long long ld, int contiguous, int padded) {
    return aligned_to(base, 16) && !(ld * es & 15) && (padded || !((long long)contiguous * es & 15)) && ld * es < (1 << 23);
  };
  const int line_a = p.kc_a ? p.K : p.M, line_b = p.kc_b ? p.K : p.N;
  const bool ok_a = direct(p.a, p.lda, line_a, p.pad_a), ok_b = direct(p.b, p.ldb, line_b, p.pad_b);
  bool whole = ok_a && ok_b;
  // One that is not is copied, unless its lines or the whole are very long: 128 x 128 tiles that load it as it is take a third longer at
  // 1000 cubed (fp16 gradients of 777 x 1001 x 1300 97 us, 45 with copies), and 4 to 8 times as long for few rows (bf16 21 x 5904 x 225 19.5 and
  // 13.4 us, fp32 1 x 973 x 628 14.7 and 11.8, the former in the best number of parts).
  const int rows_a = p.kc_a ? p.M : p.K, rows_b = p.kc_b ? p.N : p.K;
  auto copied = [&](int line, int rows) { return line < (1 << 20) && ((long long)line / epc + 1) * rows < (1 << 30); };
  if (!whole && (ok_a || copied(line_a, rows_a)) && (ok_b || copied(line_b, rows_b))) {
    if (!ok_a) { l.copy_a = 1; l.ld_a = (line_a + epc - 1) / epc * epc; l.bytes_a = round_up((size_t)l.ld_a * rows_a * es); }
    if (!ok_b) { l.copy_b = 1; l.ld_b = (line_b + epc - 1) / epc * epc; l.bytes_b = round_up((size_t)l.ld_b * rows_b * es); }
    whole = true;
  }
  const int kb = 128 / es;
  // A few rows: no tile is worth filling. x has to fit LDS where W's rows are along k.
  if (whole && p.kc_a && p.M <= lin_rows_max(p) && !(p.K & 7) && p.K > 0 && (!p.kc_b || (long long)4 * p.K * es <= 128 * 1024)) {
    l.variant = LIN_ROWS;
    l.N4 = ((long long)p.N + 3) / 4 * 4;
    l.gx = p.kc_b ? ceil_div(p.N, kRowWaves) : ceil_div(p.N, lin_row_lanes(p.N, 16 / es) * (16 / es));
    l.gy = 1;
    // W [K,N] with few columns: workgroups along k, where one would read more than 256 KB (a second launch costs what it reads in that time)
    int splits = 1;
    if (!p.kc_b) while (l.gx * splits * 2 <= 256 && (long long)p.K * 64 / splits >= 256 * 1024) splits *= 2;
    l.k_per_split = ceil_div(ceil_div(p.K, splits), 8) * 8;
    l.splits = ceil_div(p.K, l.k_per_split);
    l.bytes = l.splits > 1 ? round_up((size_t)l.splits * p.M * l.N4 * sizeof(float)) : 0;
    check_blocks((long long)l.gx * l.splits + 7, 64 * kRowWaves);
    return l;
  }
  TilePick pick{LIN_REGS, 1, 3e38f};
  if (whole) pick = pick_tile(p);
  else pick_splits(p, kRegsCost[p.kind != MM_F32], pick);
  l.variant = pick.variant;
  l.gx = ceil_div(p.N, kLinTiles[l.variant].tn);
  l.gy = ceil_div(p.M, kLinTiles[l.variant].tm);
  l.N4 = ((long long)p.N + 3) / 4 * 4;
  const long long tiles = (long long)l.gx * l.gy;
  const int per = ceil_div(ceil_div(p.K, kb), pick.splits) * kb;
  l.splits = p.K > 0 ? ceil_div(p.K, per) : 1;
  l.k_per_split = p.K > 0 ? per : kb;
  l.bytes = l.splits > 1 ? round_up((size_t)l.splits * p.M * l.N4 * sizeof(float)) : 0;
  check_blocks(tiles * l.splits + 7, 64 * kLinTiles[l.variant].wgm * kLinTiles[l.variant].wgn);
  return l;
}

void check_ws(const char* what, size_t need, const void* ws, size_t have) {
  if (need > have || (need && (!ws || !aligned_to(ws, 16)))) throw std::runtime_error(std::string(what) + ": workspace too small or unaligned");
}

// rows of a dz block: enough blocks to fill the card, at least 16 rows each
int dz_rows(int M, int N) {
  if (M <= 0 || N <= 0) return 16;
  const int col_blocks = ceil_div(N, 256);
  int blocks = ceil_div(2048, col_blocks);
  if (blocks > 128) blocks = 128;
  int rows = ceil_div(M, blocks);
  return rows < 16 ? 16 : rows;
}

}  // namespace

size_t mm_product_workspace(const MmProduct& p) {
  if (p.M <= 0 || p.N <= 0) return 0;
  const Plan l = plan_of(p);
  return l.bytes + l.bytes_a + l.bytes_b;
}

void mm_product(const MmProduct& p, void* ws, size_t ws_bytes, hipStream_t stream) {
  if (p.M <= 0 || p.N <= 0) return;
  const Plan l = plan_of(p);
  check_ws("linear", l.bytes + l.bytes_a + l.bytes_b, ws, ws_bytes);
  LinTileArgs a{};
  a.p = p;
  a.partial = reinterpret_cast<float*>(ws);
  a.N4 = l.N4;
  a.k_per_split = l.k_per_split;
  a.gx = l.gx; a.gy = l.gy; a.splits = l.splits; a.total = l.gx * l.gy * l.splits;
  const int es = elem_bytes(p.kind), epc = 16 / es, v4 = 4 * es;
  auto up = [&](int n) { return (n + epc - 1) / epc * epc; };
  if ((l.copy_a || l.copy_b) && p.K > 0) {
    LinPadArgs c{};
    char* at = reinterpret_cast<char*>(ws) + l.bytes;
    if (l.copy_a) {
      c.src[0] = p.a; c.ld[0] = p.lda; c.dst[0] = at; c.ld_dst[0] = l.ld_a;
      c.rows[0] = p.kc_a ? p.M : p.K; c.cols[0] = p.kc_a ? p.K : p.M;
      a.p.a = at; a.p.lda = l.ld_a; a.p.pad_a = 1;
    }
    if (l.copy_b) {
      c.src[1] = p.b; c.ld[1] = p.ldb; c.dst[1] = at + l.bytes_a; c.ld_dst[1] = l.ld_b;
      c.rows[1] = p.kc_b ? p.N : p.K; c.cols[1] = p.kc_b ? p.K : p.N;
      a.p.b = at + l.bytes_a; a.p.ldb = l.ld_b; a.p.pad_b = 1;
    }
    lin_launch(p.kind).pad(c, stream);
  }
  a.rows_a = !p.kc_a && a.p.pad_a ? up(p.M) : p.M;
  a.rows_b = !p.kc_b && a.p.pad_b ? up(p.N) : p.N;
  a.vec = !(p.N & 3) && !(p.ldc & 3) && aligned_to(p.c, v4) && (!p.bias || aligned_to(p.bias, v4)) &&
          (!p.res || (!(p.ldr & 3) && aligned_to(p.res, v4))) && (!p.pre || (!(p.ldp & 3) && aligned_to(p.pre, v4)));
  const LinLaunch& f = lin_launch(p.kind);
  f.tile(a, l.variant, stream);
  if (l.splits > 1) f.join(a, stream);
}

namespace {
MmProduct forward_of(const LinearArgs& a) {
  MmProduct p{};
  p.kind = a.kind;
  p.kc_a = 1; p.kc_b = a.trans_w;
  p.M = a.M; p.N = a.N; p.K = a.K;
  p.a = a.x; p.lda = a.ldx;
  p.b = a.w; p.ldb = a.ldw;
  p.c = a.y; p.ldc = a.ldy;
  p.bias = a.bias; p.res = a.res; p.ldr = a.ldr; p.pre = a.pre; p.ldp = a.ldp;
  p.act = a.act;
  p.scale = 1.f;
  return p;
}
struct BwdPlan {
  MmProduct dx, dw;
  int rows, blocks;
  long long N4, lddz;
  float dz_scale;
  size_t dz_bytes, part_bytes, prod_bytes;
};
BwdPlan bwd_plan(const LinearBwdArgs& a, void* dz) {
  BwdPlan b{};
  check_sizes(a.M, a.N, a.K);
  if (a.db) check_blocks(ceil_div(a.N, 64), 256);
  const bool own_dz = a.act != ACT_NONE && (a.dx || a.dw);
  b.N4 = ((long long)a.N + 3) / 4 * 4;
  b.lddz = ((long long)a.N + 7) / 8 * 8;
  // Slopes reach 1.13 (gelu, gelu_tanh) and 1.10 (silu): times an fp16 dy near 65504 they leave the type's range, where the sums of dx and dw need
  // not. There dz is kept halved and the products doubled, exactly but below 2^-13, where a value keeps one bit less (multiples of 2^-23).
  b.dz_scale = own_dz && a.kind == MM_F16 && a.act != ACT_RELU ? 0.5f : 1.f;
  b.dx.scale = b.dw.scale = 1.f / b.dz_scale;
  b.rows = dz_rows(a.M, a.N);
  b.blocks = ceil_div(a.M, b.rows);
  b.dz_bytes = own_dz ? round_up((size_t)a.M * b.lddz * elem_bytes(a.kind)) : 0;
  b.part_bytes = a.db ? round_up((size_t)b.blocks * b.N4 * sizeof(float)) : 0;
  const void* src = own_dz ? dz : a.dy;
  const long long ld = own_dz ? b.lddz : a.lddy;
  // dx[M,K] = dz[M,N] W^T: W^T(n, k) is n-contiguous where W is [K,N]
  b.dx.kind = a.kind;
  b.dx.kc_a = 1; b.dx.kc_b = !a.trans_w;
  b.dx.M = a.M; b.dx.N = a.K; b.dx.K = a.N;
  b.dx.pad_a = own_dz;
  (a.trans_w ? b.dw.pad_a : b.dw.pad_b) = own_dz;
  b.dx.a = src; b.dx.lda = ld; b.dx.b = a.w; b.dx.ldb = a.ldw;
  b.dx.c = a.dx; b.dx.ldc = a.lddx;
  // dw[K,N] = x^T dz, or [N,K] = dz^T x
  b.dw.kind = a.kind;
  b.dw.K = a.M;
  b.dw.M = a.trans_w ? a.N : a.K; b.dw.N = a.trans_w ? a.K : a.N;
  b.dw.a = a.trans_w ? src : a.x; b.dw.lda = a.trans_w ? ld : a.ldx;
  b.dw.b = a.trans_w ? a.x : src; b.dw.ldb = a.trans_w ? a.ldx : ld;
  b.dw.c = a.dw; b.dw.ldc = a.lddw;
  b.dw.accumulate = a.accumulate;
  const size_t x = a.dx ? mm_product_workspace(b.dx) : 0, w = a.dw ? mm_product_workspace(b.dw) : 0;
  b.prod_bytes = x > w ? x : w;
  return b;
}
}  // namespace

size_t linear_workspace(const LinearArgs& a) { return mm_product_workspace(forward_of(a)); }
void linear(const LinearArgs& a, void* ws, size_t ws_bytes, hipStream_t stream) { mm_product(forward_of(a), ws, ws_bytes, stream); }

size_t linear_bwd_workspace(const LinearBwdArgs& a) {
  const BwdPlan b = bwd_plan(a, nullptr);
  return b.dz_bytes + b.part_bytes + b.prod_bytes;
}

void linear_bwd(const LinearBwdArgs& a, void* ws, size_t ws_bytes, hipStream_t stream) {
  char* at = reinterpret_cast<char*>(ws);
  const BwdPlan b = bwd_plan(a, at);
  check_ws("linear_bwd", b.dz_bytes + b.part_bytes + b.prod_bytes, ws, ws_bytes);
  float* part = reinterpret_cast<float*>(at + b.dz_bytes);
  char* prod = at + b.dz_bytes + b.part_bytes;
  const LinLaunch& f = lin_launch(a.kind);
  if ((b.dz_bytes || a.db) && a.N > 0) {
    if (a.M > 0) {
      LinDzArgs d{};
      d.dy = a.dy; d.lddy = a.lddy; d.pre = a.pre; d.ldp = a.ldp;
      d.dz = b.dz_bytes ? at : nullptr; d.lddz = b.lddz;
      d.part = a.db ? part : nullptr; d.N4 = b.N4;
      d.M = a.M; d.N = a.N; d.act = a.act; d.rows_per_block = b.rows; d.dz_scale = b.dz_scale;
      const int v4 = 4 * elem_bytes(a.kind);
      d.vec = !(a.N & 3) && !(a.lddy & 3) && aligned_to(a.dy, v4) && (a.act == ACT_NONE || (!(a.ldp & 3) && aligned_to(a.pre, v4)));
      f.dz(d, dim3((unsigned)ceil_div(a.N, 256), (unsigned)b.blocks), stream);
    }
    if (a.db) {
      LinColSumArgs c{};
      c.part = part; c.N4 = b.N4; c.blocks = b.blocks; c.N = a.N; c.accumulate = a.accumulate; c.db = a.db;
      f.colsum(c, stream);
    }
  }
  if (a.dx) mm_product(b.dx, prod, b.prod_bytes, stream);
  if (a.dw) mm_product(b.dw, prod, b.prod_bytes, stream);
}

}  // namespace dtf
