// Dense layers: y = act(x W + b) + residual and its gradients, in fp32, bf16 or fp16 (linear.hip).
#pragma once
#include "common.h"

namespace dtf {

enum LinearAct { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_GELU_TANH = 3, ACT_SILU = 4 };

// One product C[M,N] = A B with a fused epilogue; operands as in mm_tile.h. Leading dimensions in elements.
struct MmProduct {
  int kind;                 // MmKind of every tensor (not MM_PAIR)
  int kc_a, kc_b;           // k-contiguous operands
  int M, N, K;
  const void* a; long long lda;
  const void* b; long long ldb;
  int pad_a, pad_b;         // the operand's lines end in zeros up to a multiple of 16 bytes
  void* c; long long ldc;
  const void* bias;         // nullable, [N]
  const void* res;          // nullable, [M,N]: added after the activation
  long long ldr;
  void* pre;                // nullable, [M,N]: receives the value before the activation
  long long ldp;
  int act;
  float scale;              // a power of two: C = act(scale A B + bias) + res
  int accumulate;           // C += result
};
size_t mm_product_workspace(const MmProduct& p);
void mm_product(const MmProduct& p, void* ws, size_t ws_bytes, hipStream_t stream);

// y[M,N] = act(x[M,K] W + bias) + res; W is [K,N], or [N,K] with trans_w.
struct LinearArgs {
  int kind, M, N, K, trans_w, act;
  const void* x; long long ldx;
  const void* w; long long ldw;
  const void* bias;
  const void* res; long long ldr;
  void* y; long long ldy;
  void* pre; long long ldp;
};
size_t linear_workspace(const LinearArgs& a);
void linear(const LinearArgs& a, void* ws, size_t ws_bytes, hipStream_t stream);

// dz = dy * act'(pre); dx = dz W^T, dw = x^T dz (laid out like W), db = column sums of dz; null outputs are left out.
struct LinearBwdArgs {
  int kind, M, N, K, trans_w, act;
  const void* dy; long long lddy;
  const void* pre; long long ldp;      // not read for ACT_NONE
  const void* x; long long ldx;
  const void* w; long long ldw;
  void* dx; long long lddx;
  void* dw; long long lddw;
  void* db;
  int accumulate;                      // dw and db are added to
};
size_t linear_bwd_workspace(const LinearBwdArgs& a);
void linear_bwd(const LinearBwdArgs& a, void* ws, size_t ws_bytes, hipStream_t stream);

}  // namespace dtf
