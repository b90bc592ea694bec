#!/usr/bin/env python
"""The two forms of the linear softmax cross entropy (csrc/dimn_xent.h for many rows, csrc/dimn_xent_thin.h for few), timed at the same shapes,
and the time models by which XentPlan::prefers_thin chooses between them.

    make -C deepimpute_amd/csrc variant_rowops OUT=libdimn_few.so DEFS=-DDIMN_XENT_FORM=1     # always the form for few rows
    make -C deepimpute_amd/csrc variant_rowops OUT=libdimn_many.so DEFS=-DDIMN_XENT_FORM=0    # always the other one
    DIMN_LIB_PATH=.../libdimn_few.so python tools/xent_forms.py time > few.txt                # on a GPU; likewise many.txt, and chosen.txt of libdimn.so
    python tools/xent_forms.py table few.txt many.txt chosen.txt > profiles/xent_forms.txt
    python tools/xent_forms.py fit profiles/xent_forms.txt                                    # coefficients, and what choosing by them costs

A line of the table: type, width, classes, memory order, rows, microseconds of a forward call in either form and as chosen, of a backward call
likewise.  `fit` is a non-negative least-squares fit of relative errors to the terms named in prefers_thin."""
import math
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
SHAPES = [(1344, 28165), (300, 20011), (256, 20000), (64, 18000), (2048, 8000), (3000, 50000), (512, 3000)]
ROWS = [40, 100, 150, 200, 300, 500, 800]


def time_all():
    import torch
    from deepimpute_amd import ops

    def timed(call, passes=8):
        for _ in range(3):
            call()
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        a.record()
        for _ in range(passes):
            call()
        b.record()
        torch.cuda.synchronize()
        return a.elapsed_time(b) / passes * 1e3
    for name, dtype in (("float32", torch.float32), ("bfloat16", torch.bfloat16)):
        for width, classes in SHAPES:
            for order in ("out_in", "in_out"):
                kernel = (torch.randn(classes, width, device="cuda") / math.sqrt(width)).to(dtype).t()
                kernel = kernel if order == "out_in" else kernel.contiguous()
                bias = torch.zeros(classes, device="cuda")
                for rows in ROWS:
                    x = torch.randn(rows, width, device="cuda").to(dtype)
                    y = torch.randint(0, classes, (rows,), device="cuda", dtype=torch.int32)
                    d = torch.ones(rows, device="cuda") / rows
                    _, lse = ops.linear_cross_entropy(x, kernel, y, bias)
                    forward = timed(lambda: ops.linear_cross_entropy(x, kernel, y, bias))
                    backward = timed(lambda: ops.linear_cross_entropy_grad(d, x, kernel, y, lse, bias))
                    print(name, width, classes, order, rows, "%.1f %.1f" % (forward, backward), flush=True)


def table(paths):
    files = []
    for path in paths:
        with open(path) as f:
            files.append([l.split() for l in f if l.startswith(("float32", "bfloat16"))])
    print("# us of a call: type width classes order rows | forward: few-rows form, many-rows form, chosen | backward: likewise (tools/xent_forms.py)")
    for few, many, chosen in zip(*files):
        assert few[:5] == many[:5] == chosen[:5]
        print(" ".join(few[:5]), few[5], many[5], chosen[5], few[6], many[6], chosen[6])


def fit(path):
    import numpy as np
    from scipy.optimize import nnls
    with open(path) as f:
        lines = [l.split() for l in f if not l.startswith("#")]
    up = lambda a, b: -(-a // b) * b  # noqa: E731
    for which, direction in ((0, "forward"), (1, "backward")):
        for name in ("float32", "bfloat16"):
            cases = [l for l in lines if l[0] == name]
            few, many = [], []
            for _, width, classes, order, rows, *_ in cases:
                H, V, N = int(width), int(classes), int(rows)
                hv, nv = H * V * 1e-6, N * V * 1e-6
                few.append([1, H * V * up(N, 32 if name == "float32" else 64) * 1e-9, hv, nv])
                laid = 0 if which == 0 and name == "bfloat16" and order == "out_in" and H % 64 == 0 else hv
                many.append([1, up(H, 64) * V * up(N, 128) * 1e-9, laid, nv, up(H, 64)])
            t = np.array([[float(v) for v in l[5 + 3 * which:8 + 3 * which]] for l in cases])

            def model(terms, times):
                a = np.array(terms)
                c, _ = nnls(a / times[:, None], np.ones(len(times)))
                return c, a @ c
            cf, pf = model(few, t[:, 0])
            cm, pm = model(many, t[:, 1])
            best, by_fit = t[:, :2].min(1), np.where(pf < pm, t[:, 0], t[:, 1])
            now = np.where(np.abs(t[:, 2] - t[:, 0]) < np.abs(t[:, 2] - t[:, 1]), t[:, 0], t[:, 1])
            print("%s %s, %d shapes: few rows %s, many rows %s" % (direction, name, len(cases), cf.round(4), cm.round(4)))
            print("    over the better form: by this fit %.1f %% (at worst %.0f %%), as the library chooses %.1f %% (%.0f %%)"
                  % (*(100 * f(v / best - 1) for v in (by_fit, now) for f in (np.mean, np.max)),))


if __name__ == "__main__":
    {"time": lambda a: time_all(), "table": table, "fit": lambda a: fit(a[0])}[sys.argv[1]](sys.argv[2:])
