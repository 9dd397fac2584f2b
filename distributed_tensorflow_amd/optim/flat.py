"""Optimizers over a flat parameter arena, usable without the training driver.

`FlatAdam` is tf.train.AdamOptimizer as the reference configures it (beta1 0.9, beta2 0.999,
epsilon 1e-8, bias correction folded into the step size; reference:
DistributedLeNet/src/distributed_train.py:164), `FlatMomentumSGD` is momentum SGD with L2 weight
decay (the `weight_decay` hyper-parameter of DistributedResNet/src/hyper_parameters.py:29). `FlatMuon`
orthogonalises the momentum of every weight matrix by Newton-Schulz products and uses Adam for the vectors.

One `step()` of the first two is ONE kernel launch over the whole arena on a GPU (csrc/kernels/optim.hip); the
averaging of an aggregated gradient (`grad_scale` = 1 / contributors) happens inside that launch,
so a summed gradient never needs a separate scaling pass. On a CPU arena the same arithmetic runs
in PyTorch (ops/reference.py), which is also what the kernels are tested against.
"""
from __future__ import annotations

import math
from typing import Iterable, List, Optional, Tuple

import torch

from ..ops import reference as ref
from ..runtime.arena import ParamArena


class _FlatOptimizer:
    slots: Tuple[str, ...] = ()

    def __init__(self, arena: ParamArena):
        for s in self.slots:
            if s not in arena.slots:
                raise ValueError(f"arena was built without optimizer slot '{s}' (pass slots={self.slots})")
        self.arena = arena
        self.steps = 0
        self._gpu = arena.params.is_cuda
        if self._gpu:
            from ..ops import native as nv

            self._nv = nv
            self._hyper = torch.zeros(nv.HYPER_SLOTS, device=arena.params.device, dtype=torch.float32)

    def _stage(self, lr_t, beta1, beta2, eps, grad_scale, momentum, weight_decay) -> None:
        # by value with the launch: steps queued without a host synchronisation keep their own values
        self._nv.set_scalars(self._hyper, (lr_t, beta1, beta2, eps, grad_scale, momentum, weight_decay))

    def _range(self, lo: Optional[int], hi: Optional[int]) -> Tuple[int, int]:
        lo = 0 if lo is None else lo
        hi = self.arena.total if hi is None else hi
        if not (0 <= lo <= hi <= self.arena.total):
            raise ValueError(f"range [{lo}, {hi}) outside the arena of {self.arena.total} elements")
        return lo, hi

    def zero_grad(self) -> None:
        self.arena.grads.zero_()


class FlatAdam(_FlatOptimizer):
    slots = ("m", "v")

    def __init__(self, arena: ParamArena, beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8):
        super().__init__(arena)
        self.beta1, self.beta2, self.eps = beta1, beta2, eps

    def step(self, lr: float, grad_scale: float = 1.0, lo: Optional[int] = None, hi: Optional[int] = None) -> None:
        """Updates params[lo:hi] (default: everything) from grads[lo:hi] * grad_scale."""
        lo, hi = self._range(lo, hi)
        a = self.arena
        t = self.steps + 1
        lr_t = lr * (1.0 - self.beta2 ** t) ** 0.5 / (1.0 - self.beta1 ** t)
        if hi > lo:
            if self._gpu:
                self._stage(lr_t, self.beta1, self.beta2, self.eps, grad_scale, 0.0, 0.0)
                self._nv.fused_adam(a.params[lo:hi], a.grads[lo:hi], a.slots["m"][lo:hi], a.slots["v"][lo:hi], self._hyper)
            else:
                g = a.grads[lo:hi] * grad_scale if grad_scale != 1.0 else a.grads[lo:hi]
                ref.adam_update(a.params[lo:hi], g, a.slots["m"][lo:hi], a.slots["v"][lo:hi], lr_t,
                                self.beta1, self.beta2, self.eps)
        self.steps = t


class FlatMomentumSGD(_FlatOptimizer):
    slots = ("m",)

    def __init__(self, arena: ParamArena, momentum: float = 0.9, weight_decay: float = 0.0):
        super().__init__(arena)
        self.momentum, self.weight_decay = momentum, weight_decay

    def step(self, lr: float, grad_scale: float = 1.0, lo: Optional[int] = None, hi: Optional[int] = None) -> None:
        lo, hi = self._range(lo, hi)
        a = self.arena
        if hi > lo:
            if self._gpu:
                self._stage(lr, 0.0, 0.0, 0.0, grad_scale, self.momentum, self.weight_decay)
                self._nv.fused_momentum_sgd(a.params[lo:hi], a.grads[lo:hi], a.slots["m"][lo:hi], self._hyper)
            else:
                g = a.grads[lo:hi] * grad_scale if grad_scale != 1.0 else a.grads[lo:hi]
                ref.momentum_update(a.params[lo:hi], g, a.slots["m"][lo:hi], lr, self.momentum, self.weight_decay)
        self.steps += 1


class FlatMuon(_FlatOptimizer):
    """Momentum whose update is orthogonalised, matrix by matrix (ops/reference.py::muon_update): a parameter of two or
    more dimensions is the matrix [product of the leading dimensions, last dimension], so an HWIO filter is
    [kh kw in, out]; its step is lr * sqrt(max(1, out / in)) times an update whose singular values are near one, after a
    decoupled weight decay. Everything else (biases, normalisation parameters, and matrices not named in `matrices`)
    is updated by Adam with `vector_lr`. Slot "m" holds the momentum of either kind, "v" the vectors' second moments.

    ns_products: what the orthogonalisation multiplies, "pairs" or "fp32" as in ops/native.py::newton_schulz; a CPU arena is
    updated in fp32 either way.

    On a GPU the launches of a step do not grow with the number of parameters, since every one works on all matrices at once from tables
    built here: three (the scalars, momentum with the vectors' Adam, the matrices' split), two more for matrices of up to 64 x 768,
    32 x 1024 or 16 x 2048, which one workgroup takes, and 4 * ns_steps for larger ones. The tables' workspace holds the iterates of all matrices
    at once: 8 bytes per element of a long matrix, 18 of a square one (a whole ResNet-20 10, the MNIST network 12), next to
    parameter, gradient and slots."""

    slots = ("m", "v")

    def __init__(self, arena: ParamArena, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0, ns_steps: int = 5,
                 ns_coeffs=ref.NS_COEFFS, ns_eps: float = 1e-7, beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8,
                 matrices: Optional[Iterable[str]] = None, ns_products: str = "pairs"):
        super().__init__(arena)
        if not ns_eps > 0:
            raise ValueError("FlatMuon: ns_eps must be positive")   # a matrix without a gradient would be 0 / 0
        from ..ops import native as nv   # the same refusals on any device, and here rather than in the first step

        nv._ns_steps(nv._ns_key(ns_coeffs), ns_steps)
        nv._ns_fp32(ns_products)
        self.momentum, self.nesterov, self.weight_decay = momentum, nesterov, weight_decay
        self.ns_steps, self.ns_coeffs, self.ns_eps = ns_steps, ns_coeffs, ns_eps
        self.beta1, self.beta2, self.eps = beta1, beta2, eps
        named = None if matrices is None else set(matrices)
        if named is not None and named - set(arena.names()):
            raise ValueError(f"no parameter is named {sorted(named - set(arena.names()))}")
        if named is not None and any(len(arena.spec(n).shape) < 2 for n in named):
            raise ValueError("a matrix has at least two dimensions")
        self._matrices: List[Tuple[int, int, int]] = []
        self._vectors: List[Tuple[int, int]] = []
        for s in arena.specs:
            off = arena.offsets[s.name]
            if s.numel == 0:
                continue
            if len(s.shape) >= 2 and (named is None or s.name in named):
                self._matrices.append((off, s.numel // s.shape[-1], s.shape[-1]))
            else:
                self._vectors.append((off, s.numel))
        if self._gpu:
            self._tables = self._nv.MuonTables(self._matrices, self._vectors, arena.params.device, ns_products)

    def step(self, lr: float, grad_scale: float = 1.0, vector_lr: Optional[float] = None) -> None:
        """Updates every parameter from grads * grad_scale. `vector_lr` is the vectors' Adam step size; it defaults to lr, which suits the
        matrices (0.02 or so) and is ten times what Adam usually takes."""
        a, t = self.arena, self.steps + 1
        lr_t = (lr if vector_lr is None else vector_lr) * math.sqrt(1.0 - self.beta2 ** t) / (1.0 - self.beta1 ** t)
        if self._gpu:
            self._nv.check_current_device("FlatMuon", a.params, self._hyper, self._tables.workspace)   # the scalars are a launch already
            self._nv.set_scalars(self._hyper, (lr, self.momentum, grad_scale, 1.0 - lr * self.weight_decay, lr_t, 1.0 - self.beta1,
                                               1.0 - self.beta2, self.eps))
            self._nv.muon_step(a.params, a.grads, a.slots["m"], a.slots["v"], self._hyper, self._tables, nesterov=self.nesterov,
                               steps=self.ns_steps, coeffs=self.ns_coeffs, eps=self.ns_eps)
        else:
            for off, rows, cols in self._matrices:
                p, g, m = (b[off:off + rows * cols].view(rows, cols) for b in (a.params, a.grads, a.slots["m"]))
                ref.muon_update(p, g * grad_scale, m, lr, self.momentum, self.nesterov, self.weight_decay, self.ns_steps, self.ns_coeffs, self.ns_eps)
            for off, n in self._vectors:
                p, g, m, v = (b[off:off + n] for b in (a.params, a.grads, a.slots["m"], a.slots["v"]))
                ref.adam_update(p, g * grad_scale, m, v, lr_t, self.beta1, self.beta2, self.eps)
        self.steps = t
