// Dense layers y = act(x W + b) + residual in fp32, bf16 and fp16, and their gradients: the host side, which
// picks a product kernel (linear_tile.h) and lays out the workspace.
//
// Per output element the forward pass costs 2 K flops and the epilogue rides in the product's registers: bias, the
// stored pre-activation, the activation and the residual cost their own bytes and no launch. The backward pass
// is one pass over dy and the pre-activation (dz and the column sums) and two products.
#include "linear_tile.h"

namespace dtf {
namespace {

// Rows that the few-rows kernels take. More go through 64 x 64 tiles: 4096 x 4096, us by rows kernel / tiles, bf16 W [K,N] 1 row
// 10.3 / 17, 4 rows 13.3 / 13.7, 8 rows (spills) 37 / 13.7; fp32 8 rows 18.3 / 25.9.
constexpr int lin_rows_max(int kind) { return kind == MM_F32 ? 8 : 4; }
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
// The larger the tile the less is loaded per product, but it takes about a tile per CU to use the card. The choice goes by an
// estimate: rounds of workgroups times stages of k, with the us of a round's stage measured with half the CUs busy and with all
// (whole products, us by 64 / 128 / 256: bf16 8192 x 4096 x 4096 383 / 298 / 216, 2048 cubed 28 / 22 / 39, 1024 x 1536 x 2048 12.6 / 14.7 / -;
// fp32 2048 cubed 132 / 125 / 148).
struct TileCost { int variant, slots; float some16, full16, some32, full32; };
constexpr TileCost kTileCosts[] = {{LIN_64, 512, 0.22f, 0.39f, 0.6f, 1.0f}, {LIN_128, 256, 0.55f, 0.6f, 1.8f, 1.92f}, {LIN_256, 256, 1.5f, 1.63f, 7.0f, 7.2f}};
int pick_tile(const MmProduct& p) {
  int best = LIN_64;
  float least = 0.f;
  for (const TileCost& c : kTileCosts) {
    const int t = kLinTiles[c.variant].t;
    const float n = (float)((long long)ceil_div(p.M, t) * ceil_div(p.N, t)) / (float)c.slots;
    // two workgroups share a CU with 64 x 64 tiles: a round need not be full; else every round begun takes its time
    const float rounds = n <= 1.f ? 1.f : c.slots > 256 ? n + 0.25f : ceilf(n);
    const float us = rounds * (n <= 0.6f ? (p.kind == MM_F32 ? c.some32 : c.some16) : (p.kind == MM_F32 ? c.full32 : c.full16));
    if (c.variant == LIN_64 || us < least) { best = c.variant; least = us; }
  }
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
  // One that is not is copied where the product reads it often enough (fp16 gradients of 777 x 1001 x 1300: 97 -> 45 us)
  if (!whole && p.M >= 64 && p.N >= 64 && p.K >= 64 && line_a < (1 << 20) && line_b < (1 << 20)) {
    if (!ok_a) { l.copy_a = 1; l.ld_a = (line_a + epc - 1) / epc * epc; l.bytes_a = round_up((size_t)l.ld_a * (p.kc_a ? p.M : p.K) * es); }
    if (!ok_b) { l.copy_b = 1; l.ld_b = (line_b + epc - 1) / epc * epc; l.bytes_b = round_up((size_t)l.ld_b * (p.kc_b ? p.N : p.K) * es); }
    whole = true;
  }
  l.variant = whole ? pick_tile(p) : LIN_REGS;
  const int kb = 128 / es;
  // A few rows: no tile is worth filling. x has to fit LDS where W's rows are along k.
  if (whole && p.kc_a && p.M <= lin_rows_max(p.kind) && !(p.K & 7) && p.K > 0 && (!p.kc_b || (long long)8 * p.K * es <= 128 * 1024)) {
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
  const int tile = kLinTiles[l.variant].t;
  l.gx = ceil_div(p.N, tile);
  l.gy = ceil_div(p.M, tile);
  l.N4 = ((long long)p.N + 3) / 4 * 4;
  // Few tiles and a long k: several workgroups share a tile's k, twelve stages each at least, until two stand on every CU
  // (fp32 128 x 3136 x 512, 64 x 64 tiles, us in 1 / 4 / 8 / 16 parts: 40 / 22.4 / 19.0 / 18.8, the host's time).
  const long long tiles = (long long)l.gx * l.gy;
  const int stages = ceil_div(p.K, kb);
  const int slots = l.variant == LIN_REGS || l.variant == LIN_64 ? 512 : 256;
  int splits = 1;
  while (tiles * splits * 2 <= slots && stages >= splits * 24 && (size_t)p.M * l.N4 * splits * 8 <= kMaxPartialBytes) splits *= 2;
  const int per = ceil_div(stages, splits) * kb;
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
  if (l.copy_a || l.copy_b) {
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
  return p;
}
struct BwdPlan {
  MmProduct dx, dw;
  int rows, blocks;
  long long N4, lddz;
  size_t dz_bytes, part_bytes, prod_bytes;
};
BwdPlan bwd_plan(const LinearBwdArgs& a, void* dz) {
  BwdPlan b{};
  check_sizes(a.M, a.N, a.K);
  if (a.db) check_blocks(ceil_div(a.N, 64), 256);
  const bool own_dz = a.act != ACT_NONE && (a.dx || a.dw);
  b.N4 = ((long long)a.N + 3) / 4 * 4;
  b.lddz = ((long long)a.N + 7) / 8 * 8;
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
      d.M = a.M; d.N = a.N; d.act = a.act; d.rows_per_block = b.rows;
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
