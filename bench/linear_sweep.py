"""nv.linear against the library's product of the same operands, over random sizes.

Sizes are drawn over their logarithm, 9 to 8192 rows and 64 to 8192 columns, three types, both weight layouts; 7 of 10 with 16-byte rows. Each call
is captured into a graph and replayed, so the figure is GPU time. The library multiplies into a given output; nv.linear has a bias in its epilogue.

    python bench/linear_sweep.py [number of sizes] [seed]
"""
import math
import os
import random
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from distributed_tensorflow_amd.ops import native as nv  # noqa: E402


def timed(fn):
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        fn()
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record(s)
        fn()
        e1.record(s)
        s.synchronize()
        rep = max(2, min(40, int(2 / max(e0.elapsed_time(e1), 1e-3))))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            for _ in range(rep):
                fn()
        best = math.inf
        for _ in range(4):
            e0.record(s)
            g.replay()
            e1.record(s)
            s.synchronize()
            best = min(best, e0.elapsed_time(e1) * 1e3 / rep)
    return best


def main():
    count = int(sys.argv[1]) if len(sys.argv) > 1 else 60
    rng = random.Random(int(sys.argv[2]) if len(sys.argv) > 2 else 1)

    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    rows = []
    for _ in range(count):
        dt = rng.choice((torch.float32, torch.bfloat16, torch.float16))
        m, k, n, aligned, trans_w = size(9, 8192), size(64, 8192), size(64, 8192), rng.random() < 0.7, rng.random() < 0.4
        if aligned:
            k, n = (k + 7) // 8 * 8, (n + 7) // 8 * 8
        while 2 * m * k * n * (4 if dt == torch.float32 else 1) > 3e11:
            m //= 2
        x = torch.randn(m, k, device="cuda").to(dt)
        w = torch.randn(*((n, k) if trans_w else (k, n)), device="cuda").to(dt)
        b, y = torch.randn(n, device="cuda").to(dt), torch.empty(m, n, device="cuda", dtype=dt)
        ws = torch.empty(max(16, nv.linear_workspace(m, n, k, dt, trans_w)), device="cuda", dtype=torch.uint8)
        wm = w.t() if trans_w else w
        own = timed(lambda: nv.linear(x, w, b, trans_w=trans_w, out=y, workspace=ws))
        lib = timed(lambda: torch.mm(x, wm, out=y))
        rows.append((own / lib, aligned))
        print(f"{str(dt)[6:]:9s} {m:5d} x {k:5d} x {n:5d} {'[N,K]' if trans_w else '[K,N]'} {'aligned  ' if aligned else 'unaligned'} "
              f"{own:8.1f} us, library {lib:8.1f} us: {own / lib:.2f}", flush=True)
    for name, pick in (("all", rows), ("aligned", [r for r in rows if r[1]]), ("unaligned", [r for r in rows if not r[1]])):
        if pick:
            ratios = sorted(r[0] for r in pick)
            print(f"{name}: {len(pick)} sizes, geometric mean {math.exp(sum(math.log(r) for r in ratios) / len(ratios)):.2f}, {ratios[0]:.2f} to {ratios[-1]:.2f}")


if __name__ == "__main__":
    main()
