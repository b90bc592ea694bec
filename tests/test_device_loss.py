"""Softmax cross entropy of a linear output layer on device tensors (deepimpute_amd.ops.linear_cross_entropy / _grad, include/dimn.h
dimn_linear_cross_entropy*) against the formulas in float64.

Tolerances, all propagated element by element in float64 (u = 2^-24, half a float32 step):
  * a product of bfloat16 numbers is exact in float32; a float32 operand is three bfloat16 terms and the products left out are below 4 u of
    a product; a sum over K in steps of 32 accumulates at most K / 16 + 32 roundings of partial sums bounded by sum |a b|:
    E(A B) = 2 u (K / 16 + 32) |A| |B|
  * exp(z - c) is off by the error of z, by 2 u |z - c| from the scaled argument and by 8 u of its own; sums of them by 64 u
  * a bfloat16 G (the operand of two more products) is rounded by half a step, as is a bfloat16 result."""
import ctypes as C
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from deepimpute_amd import _cabi, _lib  # noqa: E402

U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _products(K):
    return 2 * U * (K / 16 + 32)


def _problem(rows, width, classes, dtype, order="out_in", target="labels", seed=0, bias=True, ignored=True):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1000 * seed + rows + 7 * width + 13 * classes)
    n = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    x = n(rows, width).to(dtype)
    kernel = (n(classes, width) * (2.0 / math.sqrt(width))).to(dtype)
    kernel = kernel.t() if order == "out_in" else kernel.t().contiguous()
    b = n(classes) * 0.5 if bias else None
    u = torch.rand((rows,), generator=gen, device="cuda")
    if target in ("labels", "labels64"):
        t = (u * classes).long().clamp(max=classes - 1)
        if ignored and rows > 2:
            t[::5] = -1
        t = t if target == "labels64" else t.int()
    else:
        t = torch.log1p(torch.floor(torch.exp(1.5 * n(rows, classes)))) / classes
        t[:: 4] = 0 if rows > 2 else t[:: 4]                         # some rows without any target
        t = t.to(torch.float32 if target == "profile" else torch.bfloat16)
    dloss = (0.5 + torch.rand((rows,), generator=gen, device="cuda")) / rows
    return x, kernel, t, b, dloss


def _target64(t, classes):
    if t.dim() == 2:
        return t.double()
    hot = torch.zeros((t.numel(), classes), dtype=torch.float64, device=t.device)
    at = torch.nonzero(t >= 0).squeeze(1)
    hot[at, t[at].long()] = 1.0
    return hot


def _reference(x, kernel, t, b, dloss=None):
    """Everything in float64, with the room each result gets."""
    X, W = x.double(), kernel.double()
    H, V, N = W.shape[0], W.shape[1], X.shape[0]
    z = X @ W + (0 if b is None else b.double())
    ez = (_products(H) + 4 * U) * (X.abs() @ W.abs()) + 2 * U * z.abs()
    lse = torch.logsumexp(z, 1)
    T = _target64(t, V)
    ts = T.sum(1)
    masked = torch.where(T > 0, z, torch.zeros_like(z))
    loss = ts * lse - (T * masked).sum(1)
    fin = torch.where(torch.isfinite(ez), ez, torch.zeros_like(ez))
    elog = fin.amax(1) + 2 * U * (72 + 2 * math.log(V) + lse.abs())
    eloss = ts * elog + (T * fin).sum(1) + 2 * U * (V / 16 + 32 if t.dim() == 2 else 4) * (ts * lse.abs() + (T * masked).abs().sum(1))
    out = dict(lse=(lse, elog), loss=(loss, eloss))
    if dloss is None:
        return out
    d = dloss.double()[:, None]
    p = torch.exp(z - lse[:, None])
    G = d * (ts[:, None] * p - T)
    eG = d * (ts[:, None] * p * (fin + elog[:, None] + 2 * U * (torch.where(torch.isfinite(z), (z - lse[:, None]).abs(), torch.zeros_like(z)) + 40 + (V / 64 + 8 if t.dim() == 2 else 0))) + 4 * U * T)
    rounded = eG + (_half(torch.bfloat16) * G.abs() if x.dtype == torch.bfloat16 else 4 * U * G.abs())
    h = _half(x.dtype)
    dx, dW, db = G @ W.t(), X.t() @ G, G.sum(0)
    out["dx"] = (dx, rounded @ W.abs().t() + (_products(V) + 4 * U) * (G.abs() @ W.abs().t()) + h * dx.abs())
    out["dkernel"] = (dW, X.abs().t() @ rounded + (_products(N) + 4 * U) * (X.abs().t() @ G.abs()) + h * dW.abs())
    out["dbias"] = (db, eG.sum(0) + 2 * U * (N / 2 + 32) * G.abs().sum(0))
    return out


def _close(name, got, want, room):
    off = (got.double() - want).abs()
    bad = ~(off <= room + 1e-30)
    assert not bool(bad.any()), "%s: %d of %d off, by up to %.3g times the room" % (name, int(bad.sum()), bad.numel(), float((off / (room + 1e-30)).max()))


def _check(rows, width, classes, dtype, order="out_in", target="labels", **kw):
    from deepimpute_amd import ops
    x, kernel, t, b, dloss = _problem(rows, width, classes, DTYPES[dtype], order, target, **kw)
    loss, lse = ops.linear_cross_entropy(x, kernel, t, b)
    ref = _reference(x, kernel, t, b, dloss)
    _close("lse", lse, *ref["lse"])
    _close("loss", loss, *ref["loss"])
    dx, dk, db = ops.linear_cross_entropy_grad(dloss, x, kernel, t, lse, b)
    assert dx.shape == x.shape and dx.dtype == x.dtype and dk.shape == kernel.shape and dk.dtype == kernel.dtype and db.dtype == torch.float32
    assert dk.stride() == kernel.stride() or min(kernel.shape) == 1
    for name, got in (("dx", dx), ("dkernel", dk), ("dbias", db)):
        _close(name, got, *ref[name])
    if t.dim() == 1:
        assert not bool(dx[t < 0].any()) and not bool(loss[t < 0].any())


SIZES = [
    (1, 1, 1), (1, 64, 2), (2, 3, 5), (3, 64, 100), (5, 65, 127), (16, 63, 128), (17, 128, 129), (63, 100, 255), (64, 256, 512), (65, 64, 257),
    (127, 200, 300), (128, 192, 640), (130, 301, 1001), (256, 128, 256), (257, 64, 4097), (300, 1000, 77), (1000, 40, 3001),
]


@pytest.mark.gpu
@pytest.mark.parametrize("target", ["labels", "profile"])
@pytest.mark.parametrize("order", ["out_in", "in_out"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sizes(dtype, order, target):
    """One row, one class, one input; everything around the tiles' 64 / 128 / 256 and the steps of 64; both memory orders of the kernel."""
    for rows, width, classes in SIZES:
        print(dtype, order, target, rows, width, classes, flush=True)
        _check(rows, width, classes, dtype, order, target, bias=classes % 3 != 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,width,classes,order,target", [
    ("bf16", 1, 1024, 32000, "out_in", "labels"),
    ("bf16", 1100, 512, 20011, "out_in", "labels64"),
    ("bf16", 2048, 256, 50000, "in_out", "labels"),
    ("f32", 64, 256, 20000, "in_out", "profile"),
    ("f32", 700, 300, 9001, "out_in", "labels64"),
    ("bf16", 999, 300, 20011, "in_out", "profile16"),
    ("f32", 33, 2048, 5000, "out_in", "profile16"),
])
def test_large(dtype, rows, width, classes, order, target):
    _check(rows, width, classes, dtype, order, target)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,width,classes,order", [
    ("f32", 12, 1480, 20011, "out_in"), ("f32", 30, 1537, 18004, "out_in"), ("f32", 60, 1100, 20011, "out_in"), ("f32", 12, 1480, 20011, "in_out"),
    ("f32", 30, 1537, 18004, "in_out"), ("f32", 101, 700, 20011, "in_out"), ("bf16", 12, 2300, 20011, "out_in"), ("bf16", 30, 2061, 18004, "out_in"),
    ("bf16", 60, 2432, 20011, "out_in"), ("bf16", 12, 2061, 20011, "in_out"), ("bf16", 60, 1300, 40001, "in_out"),
])
def test_few_rows_of_wide_layers(dtype, rows, width, classes, order):
    """Few rows of long inner dimensions: whole rounds of chunks, leftovers of every kind behind them, blocks of 16 / 32 / 64 rows."""
    _check(rows, width, classes, dtype, order, "labels")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,width,classes,order,target", [
    ("f32", 3001, 64, 40007, "out_in", "labels"),
    ("f32", 300, 4000, 47001, "in_out", "labels64"),
    ("bf16", 8200, 70, 40011, "in_out", "profile16"),
    ("bf16", 8200, 64, 70003, "out_in", "labels"),
])
def test_several_pieces(dtype, rows, width, classes, order, target):
    """More classes than one piece of the workspace holds: the last piece is an odd one, dx adds up over all of them."""
    _check(rows, width, classes, dtype, order, target)


@pytest.mark.gpu
def test_rows_far_apart():
    """Strides of 2^24 elements and more, where an offset inside a tile passes 32 bits: x's rows, then the rows of a kernel in either order."""
    from deepimpute_amd import ops
    far = (1 << 24) + 4

    def check(x, kernel, t, b, dloss):
        loss, lse = ops.linear_cross_entropy(x, kernel, t, b)
        ref = _reference(x, kernel, t, b, dloss)
        _close("lse", lse, *ref["lse"])
        _close("loss", loss, *ref["loss"])
        for name, got in zip(("dx", "dkernel", "dbias"), ops.linear_cross_entropy_grad(dloss, x, kernel, t, lse, b)):
            _close(name, got, *ref[name])

    def spread(a):
        wide = torch.empty((a.shape[0], far), dtype=a.dtype, device="cuda")
        wide[:, :a.shape[1]] = a
        return wide[:, :a.shape[1]]
    for order in ("out_in", "in_out"):
        x, kernel, t, b, dloss = _problem(20, 1500, 20011, torch.float32, order)
        check(spread(x), kernel, t, b, dloss)
        x, kernel, t, b, dloss = _problem(300, 200, 500, torch.bfloat16, order)
        check(spread(x), kernel, t, b, dloss)
    x, kernel, t, b, dloss = _problem(3, 8, 600001, torch.float32, "in_out")
    check(x, spread(kernel), t, b, dloss)
    x, kernel, t, b, dloss = _problem(3, 2100, 8, torch.bfloat16, "out_in")
    check(x, spread(kernel.t()).t(), t, b, dloss)
    x, kernel, t, b, dloss = _problem(200, 300, 40, torch.bfloat16, "out_in")
    check(x, spread(kernel.t()).t(), t, b, dloss)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,width,classes", [("f32", 20, 1500, 3001), ("f32", 300, 200, 500), ("f32", 20, 700, 20011), ("bf16", 20, 2304, 3001), ("bf16", 300, 256, 512)])
@pytest.mark.parametrize("order", ["out_in", "in_out"])
def test_rows_in_descending_order(dtype, rows, width, classes, order):
    """Negative strides, which tensors cannot have, through the C entries: x, the kernel and its gradient walked from their last row, few rows and many:
    the bits of the same rows in ascending order up to the order of a sum (which test_sizes bounds)."""
    from deepimpute_amd import ops
    fns = _lib.load()
    x, kernel, t, b, dloss = _problem(rows, width, classes, DTYPES[dtype], order)
    k = kernel if order == "in_out" else kernel.t()                  # rows in memory
    size = x.element_size()
    ref = _reference(x, kernel, t, b, dloss)
    xd, kd = x.flip(0).contiguous(), k.flip(0).contiguous()
    ld = kd.shape[1]
    strides = (-ld, 1) if order == "in_out" else (1, -ld)
    last = lambda a: a.data_ptr() + (a.shape[0] - 1) * a.shape[1] * size  # noqa: E731
    stream = torch.cuda.current_stream().cuda_stream
    d = _cabi.OutputLoss(0, 0 if dtype == "f32" else 1, rows, width, classes, last(xd), -width, last(kd), strides[0], strides[1], b.data_ptr(), t.data_ptr(), 0, 0)
    out = torch.empty((2, rows), device="cuda")

    def space(grad):
        n = C.c_int64()
        assert fns["linear_cross_entropy_workspace"](d, grad, n) == 0
        return torch.empty(n.value, dtype=torch.uint8, device="cuda")
    work = space(0)
    assert fns["linear_cross_entropy"](d, stream, out[0].data_ptr(), out[1].data_ptr(), work.data_ptr(), work.numel()) == 0, fns["last_error"]()
    _close("loss", out[0], *ref["loss"])
    _close("lse", out[1], *ref["lse"])
    work, dx, dk, db = space(1), torch.empty_like(xd), torch.empty_like(kd), torch.empty(classes, device="cuda")
    assert fns["linear_cross_entropy_grad"](d, stream, dloss.data_ptr(), out[1].data_ptr(), last(dx), -width, last(dk), strides[0], strides[1], db.data_ptr(), work.data_ptr(), work.numel()) == 0, fns["last_error"]()
    dk = dk.flip(0)
    for name, got in (("dx", dx.flip(0)), ("dkernel", dk if order == "in_out" else dk.t()), ("dbias", db)):
        _close(name, got, *ref[name])


@pytest.mark.gpu
@pytest.mark.parametrize("target", ["labels", "profile"])
@pytest.mark.parametrize("rows,width,classes", [(1, 40, 33), (20, 70, 90), (150, 66, 1001), (4000, 130, 2001), (300, 1000, 77), (7698, 22, 900)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_outputs_of_the_c_entries(dtype, rows, width, classes, target):
    """Gradients into padded planes, dkernel in the kernel's order and in the other one, dbias wanted or not: the bits of the tensors' call where the
    order is the kernel's, and nothing written behind a row, behind the last row, or behind the workspace."""
    from deepimpute_amd import ops
    fns = _lib.load()
    stream = torch.cuda.current_stream().cuda_stream
    dt = DTYPES[dtype]
    for order in ("out_in", "in_out"):
        x, kernel, t, b, dloss = _problem(rows, width, classes, dt, order, target)
        _, lse = ops.linear_cross_entropy(x, kernel, t, b)
        want = ops.linear_cross_entropy_grad(dloss, x, kernel, t, lse, b)
        ref = _reference(x, kernel, t, b, dloss)
        d, keep = ops._output_loss("test", x, kernel, t, b)
        n = C.c_int64()
        assert fns["linear_cross_entropy_workspace"](d, 1, n) == 0
        for dk_order in ("out_in", "in_out"):
            for bias in (True, False):
                dx = torch.full((rows + 1, width + 3), 7.0, dtype=dt, device="cuda")
                flat = (classes, width) if dk_order == "out_in" else (width, classes)
                dk = torch.full((flat[0] + 1, flat[1] + 5), 7.0, dtype=dt, device="cuda")
                db = torch.full((classes + 1,), 7.0, device="cuda")
                work = torch.full((n.value + 512,), 77, dtype=torch.uint8, device="cuda")
                at = -work.data_ptr() % 256
                ld = flat[1] + 5
                strides = (1, ld) if dk_order == "out_in" else (ld, 1)
                assert fns["linear_cross_entropy_grad"](d, stream, dloss.data_ptr(), lse.data_ptr(), dx.data_ptr(), width + 3, dk.data_ptr(), strides[0], strides[1],
                                                        db.data_ptr() if bias else None, work.data_ptr() + at, n.value) == 0, fns["last_error"]()
                assert bool((work[at + n.value:] == 77).all()) and bool((work[:at] == 77).all())
                assert bool((dx[:, width:] == 7).all()) and bool((dx[rows:] == 7).all())
                assert bool((dk[:, flat[1]:] == 7).all()) and bool((dk[flat[0]:] == 7).all())
                assert bool((db[classes:] == 7).all()) and (bias or bool((db == 7).all()))
                got = dk[:flat[0], :flat[1]]
                got = got.t() if dk_order == "out_in" else got
                if dk_order == order:
                    assert torch.equal(got, want[1]) and torch.equal(dx[:rows, :width], want[0]) and (not bias or torch.equal(db[:classes], want[2]))
                _close("dkernel", got, *ref["dkernel"])
                _close("dx", dx[:rows, :width], *ref["dx"])


@pytest.mark.gpu
def test_broadcast_inputs():
    """Axes of stride 0: the same row for every sample, one profile for all of them, a kernel of equal rows or columns."""
    from deepimpute_amd import ops
    for dtype in (torch.float32, torch.bfloat16):
        for rows in (9, 200):
            x, kernel, t, b, dloss = _problem(rows, 70, 90, dtype, "in_out", "profile")
            for X, K, T in ((x[1:2].expand(rows, 70), kernel, t[1:2].expand(rows, 90)), (x, kernel[:1].expand(70, 90), t), (x, kernel[:, :1].expand(70, 90), t),
                            (x, kernel, t[:, :1].expand(rows, 90)), (x[:, :1].expand(rows, 70), kernel, t)):
                got = ops.linear_cross_entropy(X, K, T, b)
                ref = _reference(X, K, T, b, dloss)
                _close("loss", got[0], *ref["loss"])
                for name, g in zip(("dx", "dkernel", "dbias"), ops.linear_cross_entropy_grad(dloss, X, K, T, got[1], b)):
                    _close(name, g, *ref[name])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,width,classes", [("f32", 4, 5), ("bf16", 64, 40)])
def test_most_rows(dtype, width, classes):
    """2^22 rows of a profile, the most a call takes: the losses and dx of the first and the last rows, and the sums over all of them."""
    from deepimpute_amd import ops
    rows = 1 << 22
    x, kernel, t, b, dloss = _problem(rows, width, classes, DTYPES[dtype], "in_out", "profile")
    loss, lse = ops.linear_cross_entropy(x, kernel, t, b)
    dx, dk, db = ops.linear_cross_entropy_grad(dloss, x, kernel, t, lse, b)
    for part in (slice(0, 300), slice(rows - 300, rows)):
        ref = _reference(x[part], kernel, t[part], b, dloss[part])
        _close("lse", lse[part], *ref["lse"])
        _close("loss", loss[part], *ref["loss"])
        _close("dx", dx[part], *ref["dx"])
    ref = _reference(x, kernel, t, b, dloss)
    _close("dkernel", dk, *ref["dkernel"])
    _close("dbias", db, *ref["dbias"])


@pytest.mark.gpu
def test_workspaces_are_far_smaller_than_the_logits():
    """Many rows and classes, narrow layers among them: one piece of the classes at a time, whatever form a call takes (the query only)."""
    fns = _lib.load()

    def space(grad, kind, rows, width, classes, order, target_kind):
        n = C.c_int64()
        k_in, k_out = (1, width) if order == "out_in" else (classes, 1)
        d = _describe(type=kind, rows=rows, width=width, classes=classes, x_row=width, kernel_in=k_in, kernel_out=k_out, target_kind=target_kind, target_row=classes)
        assert fns["linear_cross_entropy_workspace"](d, grad, n) == 0, fns["last_error"]()
        return n.value
    for kind in (0, 1):
        for order in ("out_in", "in_out"):
            for target_kind in (0, 2):
                for rows, width, classes in ((65536, 32, 100000), (65536, 72, 100000), (1 << 20, 32, 1 << 15), (1 << 20, 64, 262144), (1 << 22, 64, 65536), (1 << 22, 16, 30000)):
                    for grad in (0, 1):
                        operands = 12 * rows * ((width + 63) // 64 * 64) * 2 + 4 * rows * width
                        # a piece of 256 classes at least: G in two orders and three terms, 12 bytes for each of its elements
                        piece = max(1 << 30, 256 * 12 * rows if grad else 0)
                        got = space(grad, kind, rows, width, classes, order, target_kind)
                        assert got <= 1.1 * (piece + operands) + (64 << 20), (kind, order, target_kind, rows, width, classes, grad, got)
                        assert got < rows * classes * (4 if kind == 0 else 2)


@pytest.mark.gpu
def test_most_threads():
    """Calls whose products, layouts and last sums have 2^32 threads or more in all, which one launch cannot hold: 2^22 rows x 65536 classes forward
    (float32), 2^22 rows of 4096 inputs backward (all rows of x the same row: what is expected is a product of vectors)."""
    from deepimpute_amd import ops
    rows = 1 << 22
    x, kernel, t, b, dloss = _problem(rows, 64, 65536, torch.float32, "in_out")
    loss, lse = ops.linear_cross_entropy(x, kernel, t, b)
    for part in (slice(0, 300), slice(rows - 300, rows)):
        ref = _reference(x[part], kernel, t[part], b)
        _close("lse", lse[part], *ref["lse"])
        _close("loss", loss[part], *ref["loss"])
    del x, kernel, t, b, dloss, loss, lse
    torch.cuda.empty_cache()
    width, classes = 4096, 200
    one, kernel, _, b, _ = _problem(1, width, classes, torch.bfloat16, "in_out")
    t = torch.arange(rows, device="cuda", dtype=torch.int32) % classes
    dloss = (0.5 + (torch.arange(rows, device="cuda") % 7) / 8).float() / rows
    x = one.expand(rows, width)
    _, lse1 = ops.linear_cross_entropy(one, kernel, t[:1], b)
    dx, dk, db = ops.linear_cross_entropy_grad(dloss, x, kernel, t, lse1.expand(rows).contiguous(), b)
    for part in (slice(0, 300), slice(rows - 300, rows)):
        ref = _reference(x[part], kernel, t[part], b, dloss[part])
        _close("dx", dx[part], *ref["dx"])
    del dx
    ref = _reference(one, kernel, t[:1], b, torch.ones(1, device="cuda"))
    p = torch.exp((one.double() @ kernel.double() + b.double() - lse1.double()[:, None]))[0]
    at = torch.zeros(classes, dtype=torch.float64, device="cuda").index_add_(0, t.long(), dloss.double())
    G = dloss.double().sum() * p - at                                # per class, over all rows
    size = dloss.double().sum() * p + at                             # of its terms
    room = (_products(width) * 64 * 10 + _half(torch.bfloat16)) * size + 2 * U * (rows / 2 + 32) * size
    _close("dbias", db, G, room)
    X = one.double()[0]
    _close("dkernel", dk, X[:, None] * G[None], X.abs()[:, None] * (room + _products(rows) * size)[None] + _half(torch.bfloat16) * (X[:, None] * G[None]).abs())
    del x, dk, db
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [50, 150])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides(dtype, rows):
    """Row strides and base addresses of every remainder, a kernel that is a slice of a larger one in either order, a strided profile: the
    bits of contiguous copies in the same memory order (the two orders may add in another order: test_sizes bounds both)."""
    from deepimpute_amd import ops
    dt = DTYPES[dtype]
    x, kernel, t, b, dloss = _problem(rows, 72, 333, dt, "in_out", "profile")
    wants = []
    for k in (kernel, kernel.t().contiguous().t()):
        want = ops.linear_cross_entropy(x, k, t, b)
        wants.append(want + ops.linear_cross_entropy_grad(dloss, x, k, t, want[1], b))
    for pad, first in ((1, 0), (3, 1), (8, 5), (56, 8)):
        xs = torch.full((rows, 72 + pad + first), float("nan"), dtype=dt, device="cuda")
        xs[:, first:first + 72] = x
        ks = torch.full((72 + 2, 333 + pad + first), float("nan"), dtype=dt, device="cuda")
        ks[1:73, first:first + 333] = kernel
        kt = torch.full((333 + 1, 72 + pad + first), float("nan"), dtype=dt, device="cuda")
        kt[1:, first:first + 72] = kernel.t()
        ts = torch.full((rows, 333 + pad + first), float("nan"), device="cuda")
        ts[:, first:first + 333] = t
        for k, want in zip((ks[1:73, first:first + 333], kt[1:, first:first + 72].t()), wants):
            a, tt = xs[:, first:first + 72], ts[:, first:first + 333]
            got = ops.linear_cross_entropy(a, k, tt, b)
            grad = ops.linear_cross_entropy_grad(dloss, a, k, tt, got[1], b)
            for u, v in zip(got + grad, want):
                assert torch.equal(u, v)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_masks_and_odd_labels(dtype):
    """Classes masked by a bias of -infinity or of the lowest float32, a masked label, rows with no class left, labels past the classes, huge logits."""
    from deepimpute_amd import ops
    dt = DTYPES[dtype]
    inf = float("inf")
    for classes in (40, 700):
        x, kernel, t, _, dloss = _problem(70, 64, classes, dt, ignored=False)
        b = torch.zeros(classes, device="cuda")
        b[1::2] = -inf
        t = t // 2 * 2                                               # labels that are there
        t = t.clamp(max=classes - 2 if classes % 2 == 0 else classes - 1)
        loss, lse = ops.linear_cross_entropy(x, kernel, t, b)
        keep = list(range(0, classes, 2))
        sub = kernel[:, keep].contiguous()
        ref = _reference(x, sub, t // 2, None, dloss)
        _close("lse", lse, *ref["lse"])
        _close("loss", loss, *ref["loss"])
        dx, dk, db = ops.linear_cross_entropy_grad(dloss, x, kernel, t, lse, b)
        _close("dx", dx, *ref["dx"])
        _close("dkernel", dk[:, keep], *ref["dkernel"])
        assert not bool(dk[:, 1::2].any()) and not bool(db[1::2].any())
        low = torch.where(torch.isinf(b), torch.full_like(b, torch.finfo(torch.float32).min), b)
        loss2, lse2 = ops.linear_cross_entropy(x, kernel, t, low)
        assert torch.equal(loss2, loss) and torch.equal(lse2, lse)
        # a masked label: probability 0
        odd = torch.full_like(t, 1)
        loss3, lse3 = ops.linear_cross_entropy(x, kernel, odd, b)
        assert bool((loss3 == inf).all()) and torch.equal(lse3, lse)
        g = ops.linear_cross_entropy_grad(dloss, x, kernel, odd, lse3, b)
        assert all(bool(torch.isfinite(v).all()) for v in g)
        # nothing left at all
        none = torch.full_like(b, -inf)
        loss4, lse4 = ops.linear_cross_entropy(x, kernel, t, none)
        assert bool((lse4 == -inf).all()) and bool((loss4 == inf).all())
        g = ops.linear_cross_entropy_grad(dloss, x, kernel, t, lse4, none)
        assert all(bool(torch.isfinite(v).all()) for v in g)
        # every class masked by the lowest float32: all of them equally likely, not none
        loss6, lse6 = ops.linear_cross_entropy(x, kernel, t, torch.full_like(b, torch.finfo(torch.float32).min))
        assert bool((lse6 == torch.finfo(torch.float32).min).all()) and bool((loss6 == 0).all())
        loss7, _ = ops.linear_cross_entropy(x, kernel, odd, low)
        assert bool(torch.isfinite(loss7).all()) and float(loss7.min()) > 3.4e38
        # labels that are no classes: a loss that says so, no gradient, nothing out of bounds
        bad = t.clone()
        bad[3], bad[7], bad[9] = classes, 2 ** 31 - 1, -(2 ** 31)
        loss5, lse5 = ops.linear_cross_entropy(x, kernel, bad, None)
        assert bool(loss5[3].isnan()) and bool(loss5[7].isnan()) and float(loss5[9]) == 0 and int(loss5.isnan().sum()) == 2
        dx, _, _ = ops.linear_cross_entropy_grad(dloss, x, kernel, bad, lse5, None)
        assert not bool(dx[[3, 7, 9]].any())
    x, kernel, t, b, dloss = _problem(20, 64, 300, dt, ignored=False)
    loss, lse = ops.linear_cross_entropy(x * 1000, kernel, t, b)     # far over exp's range
    ref = _reference(x * 1000, kernel, t, b)
    _close("lse", lse, *ref["lse"])
    _close("loss", loss, *ref["loss"])
    x[5, 3] = float("nan")                                           # stays in its row
    l2, s2 = ops.linear_cross_entropy(x, kernel, t, b)
    assert bool(s2[5].isnan()) and int(s2.isnan().sum()) == 1
    clean, _ = ops.linear_cross_entropy(torch.where(x.isnan(), torch.zeros_like(x), x), kernel, t, b)
    rest = [r for r in range(20) if r != 5]
    assert torch.equal(l2[rest], clean[rest])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,classes", [(9, 64, 40), (4000, 128, 2001)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_profiles_of_masked_classes(dtype, rows, width, classes):
    """Weight on classes that a bias of -infinity masks: the loss of a label there, +infinity, also where no class is left at all; finite gradients."""
    from deepimpute_amd import ops
    inf = float("inf")
    x, kernel, t, _, dloss = _problem(rows, width, classes, DTYPES[dtype], target="profile")
    t[:: 4] = 0
    weighted = (t != 0).any(1)
    some = torch.zeros(classes, device="cuda")
    some[1::2] = -inf
    for b in (some, torch.full_like(some, -inf)):
        hit = ((t != 0) & torch.isinf(b)).any(1)
        loss, lse = ops.linear_cross_entropy(x, kernel, t, b)
        assert bool((loss[hit] == inf).all()) and bool(torch.isfinite(loss[~hit]).all()) and not bool(loss[~weighted].any())
        assert bool((lse == -inf).all() if b is not some else torch.isfinite(lse).all())
        assert all(bool(torch.isfinite(g).all()) for g in ops.linear_cross_entropy_grad(dloss, x, kernel, t, lse, b))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,classes", [(9, 128, 300), (4000, 128, 2001)])
@pytest.mark.parametrize("order", ["out_in", "in_out"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_masks_in_the_operands(dtype, order, rows, width, classes):
    """The lowest value and infinities in the kernel and in x, few rows and many: a class they mask is not there, a product with 0 is 0 (lowest value),
    and nothing spreads to other classes or rows."""
    from deepimpute_amd import ops
    dt = DTYPES[dtype]
    low, inf = torch.finfo(dt).min, float("inf")
    x, kernel, t, b, dloss = _problem(rows, width, classes, dt, order)
    x[:, 5] = 0
    x[:, 7] = x[:, 7].abs() + 0.25
    x[2, 9], x[3, 9] = low, -low
    kernel[9] = 0                                                    # (x's lowest and largest value meet zeros only)
    kernel[5], kernel[7] = 0, 0
    masked = torch.zeros(classes, dtype=torch.bool, device="cuda")
    masked[1::3] = True
    t = torch.where((t >= 0) & masked[t.clamp(min=0).long()], t - 1, t)              # labels that are there
    keep = torch.nonzero(~masked).squeeze(1)
    place = torch.cumsum(~masked, 0) - 1
    sub_t = torch.where(t >= 0, place[t.clamp(min=0).long()].to(t.dtype), t)
    ref = _reference(x, kernel[:, keep], sub_t, b[keep], dloss)
    for at_zero, mask in ((0.0, low), (low, low), (-low, low), (0.0, -inf), (low, -inf)):
        k = kernel.clone()
        k[5, ::2] = at_zero                                          # meets x = 0
        k[7, masked] = mask                                          # meets x >= 0.25
        loss, lse = ops.linear_cross_entropy(x, k, t, b)
        _close("lse", lse, *ref["lse"])
        _close("loss", loss, *ref["loss"])
        dx, dk, db = ops.linear_cross_entropy_grad(dloss, x, k, t, lse, b)
        assert not bool(dk[:, masked].any()) and not bool(db[masked].any())
        rest = [i for i in range(width) if i not in (5, 7)]          # (there dx multiplies the masks themselves)
        _close("dx", dx[:, rest], *(v[:, rest] for v in ref["dx"]))
        _close("dkernel", dk[:, keep], *ref["dkernel"])
        _close("dbias", db[keep], *(v for v in ref["dbias"]))
        if mask == low and at_zero == 0.0:
            assert bool(torch.isfinite(dx).all())
    # an infinite input: a logit of -infinity, or a row without a softmax, never another row
    y = x.clone()
    y[4, 9] = -inf
    k = kernel.clone()
    k[9] = 0.5
    k[9, ~masked] = -0.5
    y[2, 9], y[3, 9] = 0, inf
    loss, lse = ops.linear_cross_entropy(y, k, t, b)
    assert bool(lse[4].isnan()) and not bool(lse[[0, 1, 2] + list(range(5, rows))].isnan().any())
    k[9] = 0.5
    k[9, keep[1]] = 1e-3 if dtype == "bf16" else 1.000001e-3         # one of them with terms of either sign
    y[4, 9], y[3, 9] = -inf, 0
    _, lse = ops.linear_cross_entropy(y, k, t, b)
    assert float(lse[4]) == -inf                                     # every logit is -infinity: no class left
    for a, c in ((inf, -inf), (-inf, inf), (inf, low), (low, inf)):
        y[4, 9], k[9] = a, c
        y[[r for r in range(rows) if r != 4], 9] = 1
        _, lse = ops.linear_cross_entropy(y, k, t, b)
        assert float(lse[4]) == -inf
    # values within half a bfloat16 step of the largest float32, times small ones
    if dtype == "f32":
        k = kernel.clone()
        k[11] = 3.4e38
        y = x.clone()
        y[:, 11] = torch.linspace(-1e-30, 1e-30, rows, device="cuda")
        loss, lse = ops.linear_cross_entropy(y, k, t, b)
        ref = _reference(y, k, t, b)
        _close("lse", lse, *ref["lse"])
        y[:, 11] = 0
        loss, lse = ops.linear_cross_entropy(y, k, t, b)
        k[11] = 0
        ref = _reference(y, k, t, b)
        _close("lse", lse, *ref["lse"])
        _close("loss", loss, *ref["loss"])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,classes", [(9, 70, 90), (70, 64, 2001), (300, 70, 40), (4000, 128, 2001)])
@pytest.mark.parametrize("target", ["labels", "labels64", "profile", "profile16"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_without_a_gradient_hold_anything(dtype, target, rows, width, classes):
    """Padding rows (no label, a label that is no class, a profile of zeros, dloss = 0) full of NaN and infinities: the gradients of the same call with
    zeros there, bit by bit."""
    from deepimpute_amd import ops
    x, kernel, t, b, dloss = _problem(rows, width, classes, DTYPES[dtype], "in_out" if rows % 2 else "out_in", target)
    dead = torch.zeros(rows, dtype=torch.bool, device="cuda")
    dead[1::3] = True
    dead[-1] = True
    if t.dim() == 1:
        t[dead] = -1
        t[4] = classes
        dead = dead | (t < 0) | (t >= classes)
    else:
        t[dead] = 0
        dead = dead | ~(t != 0).any(1)
        t[6], t[6, 2], t[6, 5] = 0, 1, -1                            # a sum of 0 that is a target all the same
        dead[6] = False
    dloss[7] = 0
    dead[7] = True
    clean = torch.where(dead[:, None], torch.zeros_like(x), x)
    dirty = clean.clone()
    at = torch.nonzero(dead).squeeze(1)
    dirty[at] = float("nan")
    dirty[at[::2], ::2] = float("inf")
    _, lse = ops.linear_cross_entropy(clean, kernel, t, b)
    want = ops.linear_cross_entropy_grad(dloss, clean, kernel, t, lse, b)
    loss, bad = ops.linear_cross_entropy(dirty, kernel, t, b)
    assert torch.equal(bad[~dead], lse[~dead]) and not bool(loss[dead & (t < 0 if t.dim() == 1 else ~(t != 0).any(1))].any())
    got = ops.linear_cross_entropy_grad(dloss, dirty, kernel, t, bad, b)
    assert not bool(got[0][dead].any()) and all(bool(torch.isfinite(g).all()) for g in want)
    for g, w in zip(got, want):
        assert torch.equal(g, w)


@pytest.mark.gpu
@pytest.mark.parametrize("target", ["labels", "profile"])
def test_gradient_against_differences(target):
    """Central differences of sum(dloss * loss) of the float64 formula at the float32 point."""
    from deepimpute_amd import ops
    x, kernel, t, b, dloss = _problem(5, 6, 9, torch.float32, "in_out", target)
    _, lse = ops.linear_cross_entropy(x, kernel, t, b)
    grads = ops.linear_cross_entropy_grad(dloss, x, kernel, t, lse, b)
    T = _target64(t, 9)

    def f(X, W, B):
        z = X @ W + B
        return float((dloss.double() * (T.sum(1) * torch.logsumexp(z, 1) - (T * z).sum(1))).sum())
    point = [x.double(), kernel.double(), b.double()]
    h = 1e-5
    for i, g in enumerate(grads):
        for at in np.ndindex(*point[i].shape):
            v = []
            for s in (h, -h):
                q = [p.clone() for p in point]
                q[i][at] += s
                v.append(f(*q))
            assert abs(float(g[at]) - (v[0] - v[1]) / (2 * h)) < 2e-6


@pytest.mark.gpu
def test_streams_graphs_and_repeats():
    """On a side stream, two calls at once on two streams, captured and replayed with new inputs and eager work between: the same bits."""
    from deepimpute_amd import ops
    for target, dtype in (("labels", torch.bfloat16), ("profile", torch.float32)):
        def both(x, kernel, t, b, dloss):
            loss, lse = ops.linear_cross_entropy(x, kernel, t, b)
            return (loss, lse) + ops.linear_cross_entropy_grad(dloss, x, kernel, t, lse, b)
        args = _problem(200, 100, 1500, dtype, "in_out", target)
        other = _problem(200, 100, 1500, dtype, "in_out", target, seed=3)
        want, want2 = both(*args), both(*other)
        for u, v in zip(both(*args), want):
            assert torch.equal(u, v)
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        got = []
        for s, a in zip(streams, (args, other)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(both(*a))
        torch.cuda.synchronize()
        for g, w in zip(got, (want, want2)):
            for u, v in zip(g, w):
                assert torch.equal(u, v)
        held = [a.clone() for a in args]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both(*held)
        for k in range(4):
            new = _problem(200, 100, 1500, dtype, "in_out", target, seed=10 + k)
            for a, v in zip(held, new):
                a.copy_(v)
            graph.replay()
            torch.cuda.synchronize()
            for u, v in zip(out, both(*new)):
                assert torch.equal(u, v)


@pytest.mark.gpu
def test_norm_and_loss_together():
    """A normalised hidden layer in front of the output layer, forward and back through both operators, against autograd in float64."""
    from deepimpute_amd import ops
    x, kernel, t, b, dloss = _problem(150, 96, 777, torch.float32, "in_out", "labels")
    x = 3 * x + 1
    gamma, beta = torch.linspace(0.5, 1.5, 96, device="cuda"), torch.linspace(-1, 1, 96, device="cuda")
    y, mean, rstd = ops.layer_norm(x, gamma, beta)
    loss, lse = ops.linear_cross_entropy(y, kernel, t, b)
    dy, dk, db = ops.linear_cross_entropy_grad(dloss, y, kernel, t, lse, b)
    dx, dgamma, dbeta = ops.layer_norm_grad(dy, x, mean, rstd, gamma)
    leaves = [v.double().cpu().requires_grad_() for v in (x, gamma, beta, kernel, b)]
    X, g, c, K, B = leaves
    m = X.mean(1, keepdim=True)
    hat = (X - m) / torch.sqrt(((X - m) ** 2).mean(1, keepdim=True) + 1e-3)
    z = (hat * g + c) @ K + B
    T = _target64(t, 777).cpu()
    total = (dloss.double().cpu() * (T.sum(1) * torch.logsumexp(z, 1) - (T * z).sum(1))).sum()
    total.backward()
    for got, leaf in zip((dx, dgamma, dbeta, dk, db), leaves):
        w = leaf.grad
        assert float((got.double().cpu() - w).norm()) <= 2e-5 * float(w.norm())      # 1e-6 of the operands' errors, amplified by at most 10 on either way


def _describe(**kw):
    base = dict(device_id=0, type=0, rows=4, width=8, classes=16, x=4096, x_row=8, kernel=4096, kernel_in=16, kernel_out=1, bias=None, target=4096,
                target_row=0, target_kind=0)
    base.update(kw)
    return _cabi.OutputLoss(**base)


def test_refusals_on_the_host():
    """Refused before anything reaches a GPU (no GPU needed)."""
    fns = _lib.load()
    n = C.c_int64()

    def refused(what, **kw):
        d = _describe(**kw)
        assert fns["linear_cross_entropy"](d, None, 4096, 4096, 4096, 1 << 40) < 0
        assert what in fns["last_error"]().decode()
        assert fns["linear_cross_entropy_grad"](d, None, 4096, 4096, 4096, 8, 4096, 16, 1, None, 4096, 1 << 40) < 0
        assert what in fns["last_error"]().decode()
        assert fns["linear_cross_entropy_workspace"](d, 1, n) < 0
    refused("element type", type=5)
    refused("target kind", target_kind=9)
    refused("width 0", width=0)
    refused("0 classes", classes=0)
    refused("rows", rows=-1)
    refused("rows", rows=1 << 30)
    refused("strides", kernel_in=16, kernel_out=2)
    refused("null", x=None)
    refused("null", kernel=None)
    refused("null", target=None)
    refused("tiles", rows=1 << 22, classes=1 << 22)
    assert fns["linear_cross_entropy"](None, None, 4096, 4096, 4096, 1) < 0
    assert fns["linear_cross_entropy"](_describe(), None, None, 4096, 4096, 1) < 0 and b"null" in fns["last_error"]()
    assert fns["linear_cross_entropy_grad"](_describe(), None, None, 4096, 4096, 8, 4096, 16, 1, None, 4096, 1) < 0 and b"null" in fns["last_error"]()
    assert fns["linear_cross_entropy_grad"](_describe(), None, 4096, 4096, 4096, 8, 4096, 16, 3, None, 4096, 1) < 0 and b"dkernel" in fns["last_error"]()
    assert fns["linear_cross_entropy"](_describe(rows=0), None, 4096, 4096, None, 0) == 0


@pytest.mark.parametrize("target_kind", [0, 3])
@pytest.mark.parametrize("kind", [0, 1])
def test_no_rows_at_the_c_entries(kind, target_kind):
    """rows = 0: no workspace for either direction, nothing to do forward, refused backward -- before a plan is made (no GPU needed)."""
    fns = _lib.load()
    for width, classes in ((8, 16), (2048, 32000), (3, 2)):
        d = _describe(type=kind, rows=0, width=width, classes=classes, kernel_in=classes, target_kind=target_kind, x=None, kernel=None, target=None)
        for grad in (0, 1):
            n = C.c_int64(-1)
            assert fns["linear_cross_entropy_workspace"](d, grad, n) == 0 and n.value == 0
        assert fns["linear_cross_entropy"](d, None, None, None, None, 0) == 0
        assert fns["linear_cross_entropy_grad"](d, None, None, None, None, width, 4096, classes, 1, None, None, 0) == -1
        assert b"no rows" in fns["last_error"]()


def test_refusals_of_tensors():
    from deepimpute_amd import ops
    x, k, t = torch.zeros((4, 8)), torch.zeros((8, 16)), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        ops.linear_cross_entropy(x, k, t)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        ops.linear_cross_entropy(x.half(), k.half(), t)
    with pytest.raises(ValueError, match="the kernel"):
        ops.linear_cross_entropy(x, k.bfloat16(), t)
    with pytest.raises(ValueError, match="expected, got"):
        ops.linear_cross_entropy(x, k.t(), t)
    with pytest.raises(ValueError, match="bias has shape"):
        ops.linear_cross_entropy(x, k, t, torch.zeros(15))
    for bad in (torch.zeros(3, dtype=torch.int32), torch.zeros(4), torch.zeros((4, 15)), torch.zeros(4, dtype=torch.int16), torch.zeros((4, 16), dtype=torch.int32)):
        with pytest.raises(ValueError, match="target must be"):
            ops.linear_cross_entropy(x, k, bad)


def test_tensors_that_require_a_gradient_are_refused():
    """While gradients are recorded (a result would silently be a constant of the graph); not under no_grad (no GPU needed)."""
    from deepimpute_amd import ops
    x, k, t, v, b = torch.zeros((4, 8)), torch.zeros((8, 16)), torch.zeros(4, dtype=torch.int32), torch.zeros(4), torch.zeros(16)
    g = torch.ones(8)
    calls = [(ops.layer_norm, (x, g, g), (0, 1, 2)), (ops.layer_norm_grad, (x, x, v, v, g), (0, 1, 2, 3, 4)),
             (ops.linear_cross_entropy, (x, k, t, b), (0, 1, 3)), (ops.linear_cross_entropy_grad, (v, x, k, t, v, b), (0, 1, 2, 4, 5))]
    for call, args, which in calls:
        with pytest.raises(ValueError, match="GPU"):
            call(*args)
        for i in which:
            leaf = args[:i] + (args[i].clone().requires_grad_(),) + args[i + 1:]
            with pytest.raises(ValueError, match="requires a gradient"):
                call(*leaf)
            with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
                call(*leaf)


@pytest.mark.gpu
def test_refusals_on_the_device():
    from deepimpute_amd import ops
    fns = _lib.load()
    x, kernel, t, b, dloss = _problem(8, 16, 20, torch.float32, "in_out")
    out = torch.zeros((2, 8), device="cuda")
    d, keep = ops._output_loss("test", x, kernel, t, b)
    n = C.c_int64()
    assert fns["linear_cross_entropy_workspace"](d, 0, n) == 0
    work = torch.empty(n.value + 512, dtype=torch.uint8, device="cuda")
    assert fns["linear_cross_entropy"](d, None, out[0].data_ptr(), out[1].data_ptr(), work.data_ptr(), n.value - 1) == -1 and b"workspace" in fns["last_error"]()
    assert fns["linear_cross_entropy"](d, None, out[0].data_ptr(), out[1].data_ptr(), work.data_ptr() + 16, n.value) == -1
    with pytest.raises(ValueError, match="lse has shape"):
        ops.linear_cross_entropy_grad(dloss, x, kernel, t, dloss[:5], b)
    with pytest.raises(ValueError, match="dloss must be float32"):
        ops.linear_cross_entropy_grad(dloss.double(), x, kernel, t, dloss, b)
    empty = ops.linear_cross_entropy(x[:0], kernel, t[:0], b)
    assert empty[0].shape == (0,)
    g = ops.linear_cross_entropy_grad(dloss[:0], x[:0], kernel, t[:0], dloss[:0], b)
    assert g[0].shape == (0, 16) and not bool(g[1].any()) and not bool(g[2].any())
