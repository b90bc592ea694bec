"""Row operators on PyTorch-ROCm tensors: layer normalisation and the softmax cross entropy of a linear output layer, each with its
gradient (the kernels of include/dimn.h's dimn_layer_norm* / dimn_linear_cross_entropy*).

The general path calls the same kernels for `{"type": "layernormalization"}` entries of an architecture; this module is for programs that
hold their activations in tensors.  Nothing else of the package imports torch.

* Tensors live on one GPU; the kernels run on torch's current stream of that device, results and workspaces come from torch's allocator
  on the same stream, so the calls order like torch's own and can be captured into a graph.
* Activations and output kernels are float32 or bfloat16, everything else (parameters of a normalisation, biases, statistics, losses) is
  float32.  Sums are float32 and a bfloat16 result is rounded once -- but linear_cross_entropy_grad of bfloat16 tensors also rounds the gradient
  of the logits to bfloat16, from which dx and dkernel are summed (2.4e-3 from the float64 result in norm instead of 1.7e-3; float32 tensors: 6.5e-7).
* The operators stand outside autograd: they return plain tensors, and the *_grad functions are the backward pass (inside a
  torch.autograd.Function, say).  While gradients are recorded, tensors that require one are refused.
* A tensor whose last axis is not contiguous is copied first; every other stride, and any alignment, is taken as it is.
"""
import ctypes as C
import math

import torch

from . import _cabi, _lib
from .engine import DimnError

_TYPES = {torch.float32: 0, torch.bfloat16: 1}
_f = {}


def _fns():
    """The bound entry points (loaded at the first call)."""
    if not _f:
        _f.update(_lib.load())
    return _f


def _check(rc):
    if rc != 0:
        raise DimnError("libdimn error %d: %s" % (rc, (_fns()["last_error"]() or b"").decode("utf-8", "replace")))


def _device(what, x, *others):
    """Index of the one GPU all the tensors live on.  What autograd would record is refused: the results could not carry it on."""
    dev, lost = x.device, x.requires_grad
    for t in others:
        if t is not None:
            if t.device != dev:
                raise ValueError("%s: tensors on %s and %s" % (what, dev, t.device))
            if t.requires_grad:
                lost = True
    if lost and torch.is_grad_enabled():
        raise ValueError("%s: a tensor requires a gradient, which autograd would lose here: call it under torch.no_grad() or on detached tensors, with the "
                         "*_grad function as the backward pass" % what)
    if not x.is_cuda:
        raise ValueError("%s: tensors must live on a GPU (got %s)" % (what, x.device))
    return dev.index


# handle of torch's current stream on a device; the raw query when torch has it (0.1 us instead of 1.1 us per call)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _type(what, x):
    try:
        return _TYPES[x.dtype]
    except KeyError:
        raise ValueError("%s: float32 or bfloat16 tensors are implemented, got %s" % (what, x.dtype)) from None


def _f32(what, name, t, shape):
    """A contiguous float32 tensor of exactly `shape`, or None."""
    if t is None:
        return None
    if t.dtype is not torch.float32:
        raise ValueError("%s: %s must be float32, got %s" % (what, name, t.dtype))
    if t.shape != shape:
        raise ValueError("%s: %s has shape %s, expected %s" % (what, name, tuple(t.shape), tuple(shape)))
    return t if t.is_contiguous() else t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _planes(x, grouped):
    """x as [groups][rows][width]: (tensor, groups, rows, group stride, row stride)."""
    if x.stride(-1) != 1 and x.shape[-1] > 1:
        x = x.contiguous()
    shape = x.shape
    if grouped:
        if len(shape) != 3:
            x = x.reshape(shape[0], math.prod(shape[1:-1]), shape[-1])
        s = x.stride()
        return x, shape[0], x.shape[1], s[0], s[1]
    if len(shape) != 2:
        x = x.reshape(math.prod(shape[:-1]), shape[-1])
    return x, 1, x.shape[0], 0, x.stride(0)


def _norm_args(what, x, gamma, beta):
    kind = _type(what, x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("%s: rows of at least one element expected, got shape %s" % (what, tuple(x.shape)))
    grouped = any(p is not None and p.dim() == 2 for p in (gamma, beta))
    if grouped and x.dim() < 3:
        raise ValueError("%s: parameters of %d groups need x of shape [groups, ..., width], got %s"
                         % (what, (gamma if gamma is not None else beta).shape[0], tuple(x.shape)))
    shape = (x.shape[0], x.shape[-1]) if grouped else (x.shape[-1],)
    return kind, grouped, _f32(what, "gamma", gamma, shape), _f32(what, "beta", beta, shape)


def layer_norm(x, gamma=None, beta=None, eps=1e-3):
    """Layer normalisation over the last axis: (y, mean, rstd) with y = (x - mean) * rstd * gamma + beta and
    rstd = 1 / sqrt(var + eps) (keras.layers.LayerNormalization; 1e-3 is its default epsilon).

    x: [..., width], float32 or bfloat16.  gamma, beta: float32 [width], or [groups, width] for an x of shape [groups, ..., width]
    whose groups (sub-networks) have parameters of their own; None stands for ones / zeros.  y has x's shape and type, mean and rstd are
    float32 of shape x.shape[:-1]: layer_norm_grad takes them."""
    kind, grouped, gamma, beta = _norm_args("layer_norm", x, gamma, beta)
    dev = _device("layer_norm", x, gamma, beta)
    if not eps >= 0:
        raise ValueError("layer_norm: eps %r is negative or not a number" % (eps,))
    shape = x.shape
    width = shape[-1]
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    mean, rstd = y.new_empty((2,) + shape[:-1], dtype=torch.float32).unbind(0)
    x, groups, rows, xg, xr = _planes(x, grouped)
    rc = _fns()["layer_norm"](dev, _stream(dev), kind, groups, rows, width, x.data_ptr(), xg, xr, _ptr(gamma), _ptr(beta), eps,
                              y.data_ptr(), rows * width, width, mean.data_ptr(), rstd.data_ptr())
    if rc:
        _check(rc)
    return y, mean, rstd


_norm_space = {}


def layer_norm_grad(dy, x, mean, rstd, gamma=None):
    """The backward pass of layer_norm: (dx, dgamma, dbeta) from the gradient dy of y and the forward's x, mean, rstd and gamma.
    dx has x's shape and type; dgamma and dbeta are float32 of gamma's shape ([width] when gamma is None), summed over all rows of a group."""
    what = "layer_norm_grad"
    kind, grouped, gamma, _ = _norm_args(what, x, gamma, None)
    if dy.dtype != x.dtype or dy.shape != x.shape:
        raise ValueError("%s: dy is %s %s, x is %s %s" % (what, dy.dtype, tuple(dy.shape), x.dtype, tuple(x.shape)))
    shape, width = x.shape, x.shape[-1]
    mean, rstd = _f32(what, "mean", mean, shape[:-1]), _f32(what, "rstd", rstd, shape[:-1])
    dev = _device(what, x, dy, mean, rstd, gamma)
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    x, groups, rows, xg, xr = _planes(x, grouped)
    dy, _, _, dg, dr = _planes(dy, grouped)
    key = (dev, kind, groups, rows, width)
    need = _norm_space.get(key)                      # (bytes for these sizes: arithmetic, remembered because it costs a call)
    if need is None:
        n = C.c_int64()
        _check(_fns()["layer_norm_grad_workspace"](dev, kind, groups, rows, width, C.byref(n)))
        if len(_norm_space) > 4096:
            _norm_space.clear()
        need = _norm_space[key] = n.value
    work = dx.new_empty(need, dtype=torch.uint8)
    dgamma, dbeta = dx.new_empty((2, groups, width) if grouped else (2, width), dtype=torch.float32).unbind(0)
    _check(_fns()["layer_norm_grad"](dev, _stream(dev), kind, groups, rows, width, dy.data_ptr(), dg, dr, x.data_ptr(), xg, xr,
                                     mean.data_ptr(), rstd.data_ptr(), _ptr(gamma), dx.data_ptr(), rows * width, width,
                                     dgamma.data_ptr(), dbeta.data_ptr(), work.data_ptr(), need))
    return dx, dgamma, dbeta


_TARGETS = {torch.int32: 0, torch.int64: 1, torch.float32: 2, torch.bfloat16: 3}


def _output_loss(what, x, kernel, target, bias, *others):
    """The checked description of a linear output layer and its targets (struct dimn_output_loss) and the tensors it points into."""
    kind = _type(what, x)
    if kernel.dtype != x.dtype:
        raise ValueError("%s: x is %s, the kernel %s" % (what, x.dtype, kernel.dtype))
    if x.dim() != 2 or kernel.dim() != 2 or kernel.shape[0] != x.shape[1] or kernel.shape[0] < 1 or kernel.shape[1] < 1:
        raise ValueError("%s: x [rows, width] and kernel [width, classes] expected, got %s and %s" % (what, tuple(x.shape), tuple(kernel.shape)))
    rows, width = x.shape
    classes = kernel.shape[1]
    bias = _f32(what, "bias", bias, (classes,))
    target_kind = _TARGETS.get(target.dtype)
    if target_kind is None or target.shape != ((rows,) if target_kind < 2 else (rows, classes)):
        raise ValueError("%s: target must be int32 / int64 labels [%d] or a float32 / bfloat16 profile [%d, %d], got %s %s"
                         % (what, rows, rows, classes, target.dtype, tuple(target.shape)))
    dev = _device(what, x, kernel, target, bias, *others)
    if x.stride(1) != 1 and width > 1:
        x = x.contiguous()
    if target.stride(-1) != 1:
        target = target.contiguous()
    k_in, k_out = kernel.stride()
    if width == 1 and k_out != 1:                    # (the stride of an axis of one element says nothing)
        k_in = 1
    elif classes == 1 and k_in != 1:
        k_out = 1
    if k_in != 1 and k_out != 1:
        kernel = kernel.contiguous()
        k_in, k_out = kernel.stride()
    d = _cabi.OutputLoss(dev, kind, rows, width, classes, x.data_ptr(), x.stride(0), kernel.data_ptr(), k_in, k_out, _ptr(bias),
                         target.data_ptr(), target.stride(0) if target_kind > 1 else 0, target_kind)
    return d, (x, kernel, target, bias)


def _work(d, grad, device):
    n = C.c_int64()
    _check(_fns()["linear_cross_entropy_workspace"](d, grad, n))
    return torch.empty(n.value, dtype=torch.uint8, device=device), n.value


def linear_cross_entropy(x, kernel, target, bias=None):
    """Softmax cross entropy of the linear output layer z = x @ kernel + bias: (loss, lse), float32 [rows], the logits never kept.

    x: [rows, width], kernel: [width, classes] (a Dense kernel; its transpose in memory is taken as it is too), both float32 or both
    bfloat16; bias: float32 [classes].  target: integer labels [rows] -- negative: a row without a target, loss 0 -- or a profile
    [rows, classes] of weights t (float32 or bfloat16), whose loss is sum(t) * lse - sum(t * z).  lse = log(sum(exp(z))) per row is what
    linear_cross_entropy_grad takes.  The workspace holds operands that have to be laid out and one piece
    of the classes."""
    d, keep = _output_loss("linear_cross_entropy", x, kernel, target, bias)
    out = torch.empty((2, d.rows), dtype=torch.float32, device=x.device)
    work, size = _work(d, 0, x.device)
    loss, lse = out.unbind(0)
    _check(_fns()["linear_cross_entropy"](d, _stream(d.device_id), loss.data_ptr(), lse.data_ptr(), work.data_ptr(), size))
    return loss, lse


def linear_cross_entropy_grad(dloss, x, kernel, target, lse, bias=None):
    """The backward pass of linear_cross_entropy: (dx, dkernel, dbias) from the gradient dloss [rows] of the losses and the forward's lse.
    dx and dkernel have the types of x and kernel, dkernel lies in memory as the kernel does; dbias is float32 [classes].  Rows without a target, or
    with a dloss of 0, may hold anything in x: their dx is 0 and they add nothing to dkernel and dbias."""
    what = "linear_cross_entropy_grad"
    d, (x, kernel, _target, _bias) = _output_loss(what, x, kernel, target, bias, dloss, lse)
    dloss, lse = _f32(what, "dloss", dloss, (d.rows,)), _f32(what, "lse", lse, (d.rows,))
    if d.kernel_in == 1 and d.kernel_out != 1:
        dkernel = torch.empty((d.classes, d.width), dtype=x.dtype, device=x.device).t()
    else:
        dkernel = torch.empty((d.width, d.classes), dtype=x.dtype, device=x.device)
    dx = torch.empty((d.rows, d.width), dtype=x.dtype, device=x.device)
    dbias = torch.empty((d.classes,), dtype=torch.float32, device=x.device)
    if d.rows == 0:
        return dx, dkernel.zero_(), dbias.zero_()
    work, size = _work(d, 1, x.device)
    k_in, k_out = (1, d.width) if d.kernel_in == 1 and d.kernel_out != 1 else (d.classes, 1)
    _check(_fns()["linear_cross_entropy_grad"](d, _stream(d.device_id), dloss.data_ptr(), lse.data_ptr(), dx.data_ptr(), d.width,
                                               dkernel.data_ptr(), k_in, k_out, dbias.data_ptr(), work.data_ptr(), size))
    return dx, dkernel, dbias
