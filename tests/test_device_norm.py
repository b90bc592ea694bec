"""Layer normalisation on device tensors (deepimpute_amd.ops.layer_norm / layer_norm_grad, include/dimn.h dimn_layer_norm*) against
the formulas in float64.

Tolerances.  A float32 row sum of n terms in any order the kernels use is off by at most (log2(n) + 32) half steps of the sum of the
terms' sizes (a thread adds at most 32 terms one after the other, the rest is a tree); with the few roundings of the formula itself every
float32 result is within 64 half steps = 64 * 2^-24 of the size of what is added, measured here per row as the largest |term|.  A bfloat16
result adds half a step of its own, 2^-8 relative... torch.finfo(bfloat16).eps / 2.  Sums over rows: a thread adds its rows one after the
other (their number over the number of sets), the sets' partial rows are added in strands of 16: bounded by (rows + 64) half steps."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
from deepimpute_amd import _cabi, _lib  # noqa: E402

F32 = 2.0 ** -24


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _make(shape, dtype, seed, offset=0.0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    x = torch.randn(shape, generator=gen, device="cuda") * 1.7 + offset
    return x.to(dtype)


def _formula(x, gamma, beta, eps):
    x = x.double()
    mean = x.mean(-1)
    d = x - mean[..., None]
    rstd = 1.0 / torch.sqrt((d * d).mean(-1) + eps)
    per = (lambda p: p.double()[:, None, :]) if gamma is not None and gamma.dim() == 2 else (lambda p: p.double())
    y = d * rstd[..., None]
    if gamma is not None:
        y = y * per(gamma)
    if beta is not None:
        y = y + per(beta)
    return y, mean, rstd


def _formula_grad(dy, x, mean, rstd, gamma):
    dy, x, mean, rstd = dy.double(), x.double(), mean.double(), rstd.double()
    xh = (x - mean[..., None]) * rstd[..., None]
    g = dy if gamma is None else dy * (gamma.double()[:, None, :] if gamma.dim() == 2 else gamma.double())
    dx = rstd[..., None] * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    over = tuple(range(1, x.dim() - 1)) if gamma is not None and gamma.dim() == 2 else tuple(range(x.dim() - 1))
    return dx, (dy * xh).sum(over), dy.sum(over), xh


def _close(got, want, room):
    bad = (got.double() - want).abs() > room
    assert not bool(bad.any()), "off by up to %.3g of the room" % float(((got.double() - want).abs() / room.clamp(min=1e-300)).max())


def _check_forward(x, gamma, beta, eps):
    from deepimpute_amd import ops
    y, mean, rstd = ops.layer_norm(x, gamma, beta, eps)
    assert y.shape == x.shape and y.dtype == x.dtype and mean.shape == x.shape[:-1] and rstd.dtype == torch.float32
    want, wmean, wrstd = _formula(x, gamma, beta, eps)
    if x.numel() == 0:
        return y, mean, rstd
    top = x.double().abs().amax(-1)
    _close(mean, wmean, 64 * F32 * top + 1e-30)
    # the mean's error moves every centred value; relative to the spread 1 / rstd
    shift = 64 * F32 * top * wrstd
    _close(rstd, wrstd, wrstd * (64 * F32 + shift))
    size = (want if gamma is None else _formula(x, None, None, eps)[0] * (gamma.double()[:, None, :] if gamma.dim() == 2 else gamma.double())).abs()
    gmax = 1.0 if gamma is None else float(gamma.abs().max())
    bmax = 0.0 if beta is None else float(beta.abs().max())
    room = size * (64 * F32 + shift[..., None]) + gmax * shift[..., None] + bmax * 2 * F32 + _half(x.dtype) * want.abs() + 1e-30
    _close(y, want, room)
    return y, mean, rstd


def _check_backward(x, gamma, eps, seed):
    from deepimpute_amd import ops
    dy = _make(tuple(x.shape), x.dtype, seed + 1)
    _, mean, rstd = ops.layer_norm(x, gamma, None, eps)
    dx, dgamma, dbeta = ops.layer_norm_grad(dy, x, mean, rstd, gamma)
    assert dx.shape == x.shape and dx.dtype == x.dtype and dgamma.dtype == torch.float32
    want, wg, wb, xh = _formula_grad(dy, x, mean, rstd, gamma)
    assert dgamma.shape == wg.shape and dbeta.shape == wb.shape
    if x.numel() == 0:
        assert not bool(dgamma.any()) and not bool(dbeta.any())
        return
    gmax = 1.0 if gamma is None else float(gamma.abs().max())
    dmax, hmax = float(dy.double().abs().max()), float(xh.abs().max())
    # xh itself carries three roundings of (x - mean) rstd
    room = rstd.double()[..., None] * gmax * dmax * (1 + hmax + hmax * hmax) * 64 * F32 + _half(x.dtype) * want.abs() + 1e-30
    _close(dx, want, room)
    rows = x.numel() // x.shape[-1] // (gamma.shape[0] if gamma is not None and gamma.dim() == 2 else 1)
    steps = (min(rows, 400) + 64) * F32
    over = tuple(range(1, x.dim() - 1)) if gamma is not None and gamma.dim() == 2 else tuple(range(x.dim() - 1))
    _close(dgamma, wg, (dy.double() * xh).abs().sum(over) * steps + dmax * hmax * 8 * F32 * rows ** 0.5 + 1e-30)
    _close(dbeta, wb, dy.double().abs().sum(over) * steps + 1e-30)


WIDTHS = [1, 2, 3, 7, 8, 64, 127, 128, 129, 255, 256, 257, 301, 1024, 1025, 2047, 2400, 2401]
LONG = [4096, 8191, 8193, 12289, 16384, 16385, 24577, 40000]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("width", WIDTHS + LONG)
def test_widths(width, dtype):
    """Every form of the kernels (16, 64, 256, 1024 threads per row, the register piece counts, rows past the registers), one row and ragged
    numbers of rows, forward and backward."""
    for rows in ([1, 5, 67] if width < 4096 else [1, 3]):
        x = _make((rows, width), dtype, 10 * width + rows, offset=0.5)
        gamma, beta = 1 + 0.3 * _make((width,), torch.float32, 3), _make((width,), torch.float32, 4)
        _check_forward(x, gamma, beta, 1e-3)
        _check_backward(x, gamma, 1e-3, 5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_many_rows_and_groups(dtype):
    """More rows than sets of threads (the loop over rows with the next row in flight), groups with parameters of their own, no parameters."""
    x = _make((9001, 300), dtype, 1)
    _check_forward(x, None, None, 1e-5)
    _check_backward(x, None, 1e-5, 2)
    x = _make((3, 2, 131, 72), dtype, 3, offset=-2.0)
    gamma, beta = 1 + 0.2 * _make((3, 72), torch.float32, 4), _make((3, 72), torch.float32, 5)
    grouped = x.reshape(3, 262, 72)
    _check_forward(grouped, gamma, beta, 1e-3)
    _check_backward(grouped, gamma, 1e-3, 6)
    from deepimpute_amd import ops
    y4, _, _ = ops.layer_norm(x, gamma, beta)
    y3, _, _ = ops.layer_norm(grouped, gamma, beta)
    assert torch.equal(y4.reshape(3, 262, 72), y3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_strides_and_alignment(dtype):
    """Row strides of every remainder, odd base addresses, transposed and broadcast rows: the same values as of a contiguous copy, and nothing
    around the rows is written."""
    from deepimpute_amd import ops
    gamma, beta = 1 + 0.3 * _make((77,), torch.float32, 3), _make((77,), torch.float32, 4)
    for pitch, first in [(77, 0), (78, 1), (79, 3), (80, 2), (85, 5)]:
        store = _make((40 * pitch + 16,), dtype, pitch)
        x = store[first:first + 33 * pitch].view(33, pitch)[:, :77]
        a, am, ar = ops.layer_norm(x, gamma, beta)
        b, bm, br = ops.layer_norm(x.contiguous(), gamma, beta)
        assert torch.equal(a, b) and torch.equal(am, bm) and torch.equal(ar, br)
        dy = _make((33, 77), dtype, 9)
        for u, v in zip(ops.layer_norm_grad(dy, x, am, ar, gamma), ops.layer_norm_grad(dy, x.contiguous(), am, ar, gamma)):
            assert torch.equal(u, v)
    x = _make((77, 33), dtype, 7).t()                                # the last axis is not contiguous: copied
    assert torch.equal(ops.layer_norm(x, gamma, beta)[0], ops.layer_norm(x.contiguous(), gamma, beta)[0])
    x = _make((1, 77), dtype, 8).expand(20, 77)                      # broadcast rows
    y, _, _ = ops.layer_norm(x, gamma, beta)
    assert torch.equal(y, ops.layer_norm(x.contiguous(), gamma, beta)[0])
    x = _make((6, 40, 77), dtype, 12).transpose(0, 1)                # [40, 6, 77], strided in both leading axes
    g2 = 1 + 0.3 * _make((40, 77), torch.float32, 13)
    assert torch.equal(ops.layer_norm(x, g2)[0], ops.layer_norm(x.contiguous(), g2)[0])


@pytest.mark.gpu
def test_only_the_rows_are_written():
    """Through the C entry: a result with a row stride and rows behind the last one keeps every byte outside the rows."""
    fns = _lib.load()
    x = _make((10, 19), torch.float32, 1)
    y = torch.full((14, 24), 7.0, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    assert fns["layer_norm"](0, s, 0, 1, 10, 19, x.data_ptr(), 0, 19, None, None, 1e-3, y.data_ptr(), 0, 24, None, None) == 0
    want = _formula(x, None, None, 1e-3)[0]
    assert float((y[:10, :19].double() - want).abs().max()) < 1e-5
    assert bool((y[10:] == 7).all()) and bool((y[:, 19:] == 7).all())


@pytest.mark.gpu
def test_no_rows_and_in_place():
    from deepimpute_amd import ops
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.empty((0, 50), dtype=dtype, device="cuda")
        _check_forward(x, None, None, 1e-3)
        _check_backward(x, 1 + torch.zeros(50, device="cuda"), 1e-3, 1)
        x = torch.empty((2, 0, 50), dtype=dtype, device="cuda")
        _check_backward(x, torch.ones((2, 50), device="cuda"), 1e-3, 1)
    x = _make((70, 500), torch.float32, 5)
    want, mean, rstd = ops.layer_norm(x)
    y = x.clone()
    fns = _lib.load()
    s = torch.cuda.current_stream().cuda_stream
    assert fns["layer_norm"](0, s, 0, 1, 70, 500, y.data_ptr(), 0, 500, None, None, 1e-3, y.data_ptr(), 0, 500, None, None) == 0
    assert torch.equal(y, want)
    dy = _make((70, 500), torch.float32, 6)
    dx, _, _ = ops.layer_norm_grad(dy, x, mean, rstd)
    assert fns["layer_norm_grad"](0, s, 0, 1, 70, 500, dy.data_ptr(), 0, 500, x.data_ptr(), 0, 500, mean.data_ptr(), rstd.data_ptr(), None,
                                  dy.data_ptr(), 0, 500, None, None, None, 0) == 0
    assert torch.equal(dy, dx)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_in_place_at_every_form(dtype):
    """y over x, dx over dy and dx over x: short rows, rows of 16 / 64 / 256 / 1024 threads with and without a moved last piece, rows read thrice."""
    from deepimpute_amd import ops
    fns = _lib.load()
    s = torch.cuda.current_stream().cuda_stream
    kind = 0 if dtype == torch.float32 else 1
    for width in (3, 37, 128, 301, 1027, 2401, 9001, 16385, 40003):
        rows = 300 if width < 3000 else 9
        x, dy = _make((rows, width), dtype, width), _make((rows, width), dtype, width + 1)
        gamma = 1 + 0.1 * _make((width,), torch.float32, 3)
        want, mean, rstd = ops.layer_norm(x, gamma)
        y = x.clone()
        assert fns["layer_norm"](0, s, kind, 1, rows, width, y.data_ptr(), 0, width, gamma.data_ptr(), None, 1e-3, y.data_ptr(), 0, width, None, None) == 0
        assert torch.equal(y, want), width
        dx, _, _ = ops.layer_norm_grad(dy, x, mean, rstd, gamma)
        for over in ("dy", "x"):
            a, b = dy.clone(), x.clone()
            out = a if over == "dy" else b
            assert fns["layer_norm_grad"](0, s, kind, 1, rows, width, a.data_ptr(), 0, width, b.data_ptr(), 0, width, mean.data_ptr(), rstd.data_ptr(),
                                          gamma.data_ptr(), out.data_ptr(), 0, width, None, None, None, 0) == 0
            assert torch.equal(out, dx), (width, over)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("width", [261, 389, 1027, 1285, 1541, 2049, 2051, 3077, 4099, 6149, 6151])
def test_the_same_bits_every_time(width, dtype):
    """Rows whose last piece is moved back over another thread's columns, of another wave too: both write them, and the result is the same bits
    call after call, in both directions and in place."""
    from deepimpute_amd import ops
    rows = 2500
    x, dy = _make((rows, width), dtype, width), _make((rows, width), dtype, width + 1)
    gamma, beta = _make((width,), torch.float32, 2), _make((width,), torch.float32, 3)
    want = ops.layer_norm(x, gamma, beta)
    grads = ops.layer_norm_grad(dy, x, want[1], want[2], gamma)
    for _ in range(12):
        for u, v in zip(ops.layer_norm(x, gamma, beta), want):
            assert torch.equal(u, v)
        for u, v in zip(ops.layer_norm_grad(dy, x, want[1], want[2], gamma), grads):
            assert torch.equal(u, v)


@pytest.mark.gpu
def test_longest_row():
    """A row of 2^26 elements, the most there may be; a thread adds 2^16 of them one after the other: 2^16 + 64 half steps of the largest term."""
    from deepimpute_amd import ops
    width = 1 << 26
    steps = (width / 1024 + 64) * F32
    x, dy = _make((1, width), torch.float32, 1), _make((1, width), torch.float32, 2)
    gamma = 1 + 0.1 * torch.rand(width, device="cuda")
    y, mean, rstd = ops.layer_norm(x, gamma, None)
    want, wmean, wrstd = _formula(x, gamma, None, 1e-3)
    top = float(x.abs().max())
    assert abs(float(mean) - float(wmean)) <= steps * top and abs(float(rstd) / float(wrstd) - 1) <= 2 * steps
    _close(y, want, 2 * steps * (want.abs() + 1.2 * top))
    dx, dgamma, dbeta = ops.layer_norm_grad(dy, x, mean, rstd, gamma)
    want, wg, wb, xh = _formula_grad(dy, x, mean, rstd, gamma)
    size = 1.2 * float(dy.abs().max()) * (1 + float(xh.abs().max()))
    _close(dx, want, float(rstd) * (steps * size * (1 + xh.abs()) + 8 * F32 * size))
    _close(dgamma, wg, 8 * F32 * wg.abs() + 1e-30)
    assert torch.equal(dbeta, dy[0])


@pytest.mark.gpu
def test_values_at_the_edges():
    """Constant rows (spread 0), rows far from zero, huge and tiny values, an infinity or NaN stays in its row."""
    from deepimpute_amd import ops
    x = torch.full((4, 100), 3.0, device="cuda")
    y, mean, rstd = ops.layer_norm(x, eps=1e-3)
    assert bool((y == 0).all()) and bool((mean == 3).all()) and float((rstd - 1e-3 ** -0.5).abs().max()) < 1e-4
    x = _make((16, 700), torch.float32, 1) + 4096.0                  # E[x^2] - mean^2 would lose the spread
    _check_forward(x, None, None, 1e-3)
    x = _make((5, 100), torch.float32, 2)
    want = ops.layer_norm(x)[0]
    x[1, 3], x[3, 99] = float("inf"), float("nan")
    y = ops.layer_norm(x)[0]
    assert bool(y[1].isnan().all()) and bool(y[3].isnan().all())
    for r in (0, 2, 4):
        assert torch.equal(y[r], want[r])


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences of sum(y * c) in float64 of the forward formula, at the float32 point the kernel differentiates."""
    from deepimpute_amd import ops
    x, c = _make((3, 11), torch.float32, 1), _make((3, 11), torch.float32, 2)
    gamma, beta = 1 + 0.3 * _make((11,), torch.float32, 3), _make((11,), torch.float32, 4)
    _, mean, rstd = ops.layer_norm(x, gamma, beta)
    dx, dgamma, dbeta = ops.layer_norm_grad(c, x, mean, rstd, gamma)
    f = lambda a, g, b: float((_formula(a, g, b, 1e-3)[0] * c.double()).sum())  # noqa: E731
    h = 1e-5
    for t, d in ((x, dx), (gamma, dgamma), (beta, dbeta)):
        for at in np.ndindex(*t.shape):
            up, down = t.double().clone(), t.double().clone()
            up[at] += h
            down[at] -= h
            args = [[v.double(), gamma.double(), beta.double()] for v in (x, x)]
            for a, v in zip(args, (up, down)):
                a[0 if t is x else (1 if t is gamma else 2)] = v
            diff = (f(*args[0]) - f(*args[1])) / (2 * h)             # error h^2 of a third derivative of order 10: 1e-9
            assert abs(float(d[at]) - diff) < 2e-5 * (1 + abs(diff))


@pytest.mark.gpu
def test_streams_graphs_and_repeats():
    """On a side stream, captured and replayed with other work between the replays, and twice on the same inputs: the same bits each time."""
    from deepimpute_amd import ops
    x = _make((500, 901), torch.bfloat16, 1)
    dy = _make((500, 901), torch.bfloat16, 2)
    gamma, beta = 1 + 0.3 * _make((901,), torch.float32, 3), _make((901,), torch.float32, 4)

    def both(x, dy):
        y, mean, rstd = ops.layer_norm(x, gamma, beta)
        return (y, mean, rstd) + ops.layer_norm_grad(dy, x, mean, rstd, gamma)
    want = both(x, dy)
    for a, b in zip(both(x, dy), want):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(x, dy)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    sx, sdy = x.clone(), dy.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(sx, sdy)
    for k in range(4):
        nx, ndy = _make((500, 901), torch.bfloat16, 20 + k), _make((500, 901), torch.bfloat16, 30 + k)
        sx.copy_(nx)
        sdy.copy_(ndy)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, both(nx, ndy)):
            assert torch.equal(a, b)


def test_every_form_is_some_width(monkeypatch):
    """The library has the forms (threads per row, pieces per thread) that some width takes, and no others (no GPU needed)."""
    import os
    import re
    monkeypatch.syspath_prepend(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tools"))
    import kernel_resources
    table, _ = kernel_resources.check(_lib.LIB_PATH)
    built = {(g, t, int(a), int(e), int(v)) for r in table.values()
             for g, t, a, e, v in re.findall(r"void rowops::k_norm(_grad)?<(float|unsigned short), (\d+), (\d+), (\d+)>", r["demangled"])}

    def form(bf, grad, width):
        v = 8 if bf else 4
        if width < v:
            return 16, 1, 1
        pieces = -(-width // v)
        most, most1k = (3 if grad else 5, 2) if bf else (6, 4)
        for threads, limit in ((16, 32), (64, 64 * most), (256, 256 * most), (1024, 1024 * most1k)):
            if pieces <= limit:
                return threads, -(-pieces // threads), v
        return None                                                  # longer rows: the kernels that read a row more than once
    wanted = {("_grad" if grad else "", "unsigned short" if bf else "float") + form(bf, grad, width)
              for bf in (0, 1) for grad in (0, 1) for width in range(1, 20000) if form(bf, grad, width)}
    assert built == wanted, (built - wanted, wanted - built)


def test_refusals_on_the_host():
    """What a call must not do is refused before anything reaches a GPU (no GPU needed): wrong sizes, types, null arrays."""
    fns = _lib.load()

    def message(rc, code):
        assert rc == code, rc
        return fns["last_error"]().decode()
    one = 4096                                                       # (an address that is never used: the call is refused before)
    norm = lambda kind=0, groups=1, rows=4, width=8, x=one, eps=1e-3, y=one: fns["layer_norm"](  # noqa: E731
        0, None, kind, groups, rows, width, x, 0, 8, None, None, eps, y, 0, 8, None, None)
    assert "element type" in message(norm(kind=7), -4)
    assert "width" in message(norm(width=0), -1)
    assert "width" in message(norm(width=1 << 40), -1)
    assert "width" in message(norm(width=(1 << 26) + 1), -1)
    assert "rows" in message(norm(rows=-1), -1)
    assert "null" in message(norm(x=None), -1)
    assert "null" in message(norm(y=None), -1)
    assert "eps" in message(norm(eps=-1.0), -1)
    assert "eps" in message(norm(eps=float("nan")), -1)
    assert norm(rows=0, x=None, y=None) == 0
    grad = lambda x=one, mean=one, dx=one: fns["layer_norm_grad"](  # noqa: E731
        0, None, 0, 1, 4, 8, one, 0, 8, x, 0, 8, mean, one, None, dx, 0, 8, None, None, None, 0)
    for bad in (dict(x=None), dict(mean=None), dict(dx=None)):
        assert "null" in message(grad(**bad), -1)


def test_refusals_of_tensors():
    from deepimpute_amd import ops
    x = torch.zeros((4, 8))
    with pytest.raises(ValueError, match="GPU"):
        ops.layer_norm(x)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        ops.layer_norm(x.double())
    with pytest.raises(ValueError, match="gamma has shape"):
        ops.layer_norm(x, torch.ones(7))
    with pytest.raises(ValueError, match="beta must be float32"):
        ops.layer_norm(x, torch.ones(8), torch.zeros(8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="groups"):
        ops.layer_norm(x, torch.ones((4, 8)))
    with pytest.raises(ValueError, match="at least one element"):
        ops.layer_norm(torch.zeros((4, 0)))
    with pytest.raises(ValueError, match="dy is"):
        ops.layer_norm_grad(x[:3], x, torch.zeros(4), torch.zeros(4))
    with pytest.raises(ValueError, match="mean has shape"):
        ops.layer_norm_grad(x, x, torch.zeros(3), torch.zeros(4))


@pytest.mark.gpu
def test_an_older_error_is_not_reported():
    """A HIP call of the same thread that failed before (a device that is not there) says nothing about these."""
    import ctypes
    from deepimpute_amd import ops
    x = _make((8, 40), torch.float32, 1)
    y, mean, rstd = ops.layer_norm(x)
    with open("/proc/self/maps") as f:
        path = next(line.split()[-1] for line in f if "libamdhip64" in line)
    hip = ctypes.CDLL(path)
    kernel, t = _make((40, 30), torch.float32, 2), torch.zeros(8, dtype=torch.int32, device="cuda")
    _, lse = ops.linear_cross_entropy(x, kernel, t)
    for call in (lambda: ops.layer_norm(x), lambda: ops.layer_norm_grad(y, x, mean, rstd), lambda: ops.linear_cross_entropy(x, kernel, t),
                 lambda: ops.linear_cross_entropy_grad(rstd, x, kernel, t, lse)):
        want = call()
        assert hip.hipSetDevice(4096) != 0
        for u, v in zip(call(), want):
            assert torch.equal(u, v)


@pytest.mark.gpu
def test_refusals_on_the_device():
    fns = _lib.load()
    x = _make((4, 8), torch.float32, 1)
    out = torch.empty_like(x)
    stats = torch.zeros(8, device="cuda")
    import ctypes as C
    n = C.c_int64()
    assert fns["layer_norm_grad_workspace"](0, 0, 1, 4, 8, C.byref(n)) == 0 and n.value > 0
    work = torch.empty(n.value + 16, dtype=torch.uint8, device="cuda")
    call = lambda w, size: fns["layer_norm_grad"](0, None, 0, 1, 4, 8, x.data_ptr(), 0, 8, x.data_ptr(), 0, 8, stats.data_ptr(), stats.data_ptr(), None,  # noqa: E731
                                                  out.data_ptr(), 0, 8, stats.data_ptr(), None, w, size)
    assert call(work.data_ptr(), n.value - 1) == -1 and b"workspace" in fns["last_error"]()
    assert call(work.data_ptr() + 4, n.value) == -1 and b"aligned" in fns["last_error"]()
    assert call(None, 0) == -1
    assert fns["layer_norm"](99, None, 0, 1, 4, 8, x.data_ptr(), 0, 8, None, None, 1e-3, out.data_ptr(), 0, 8, None, None) == -1
    assert b"device_id" in fns["last_error"]()
