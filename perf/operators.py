"""Cases and plain forms of the row operators (deepimpute_amd.ops): layer normalisation and the softmax cross entropy of a
linear output layer, forward and backward.

A case is measured on either side of the module's switch `own`: False runs the elementary torch operations below, True the
framework's own kernels on the same tensors.  Parameters of a normalisation and biases are float32 everywhere, as in the
rest of the framework; activations and output kernels are float32 or bfloat16.
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPSILON = 1e-3


def listed():
    return [
        # one optimiser step of 40 sub-networks: a batch of 64 cells through a normalised hidden layer of 256 units
        {"name": "norm of a step", "op": "norm", "dtype": "f32", "groups": 40, "rows": 64, "width": 256, "pitch": 256},
        # a block of validation cells through the command line's 300 units plus one, rows padded to 16 bytes
        {"name": "norm of ragged rows", "op": "norm", "dtype": "f32", "groups": 1, "rows": 4999, "width": 301, "pitch": 304},
        # the predictors of every cell of the 50k-cell matrix, normalised in front of the first layer
        {"name": "norm of all cells", "op": "norm", "dtype": "bf16", "groups": 1, "rows": 50000, "width": 2400, "pitch": 2400},
        # the same step's backward pass
        {"name": "norm grad of a step", "op": "norm_grad", "dtype": "f32", "groups": 40, "rows": 64, "width": 256, "pitch": 256},
        # an odd batch of an odd width, nothing aligned
        {"name": "norm grad of ragged rows", "op": "norm_grad", "dtype": "bf16", "groups": 1, "rows": 4099, "width": 1025, "pitch": 1025},
        # all cells: the reduction of the weight's gradient runs over 50k rows
        {"name": "norm grad of all cells", "op": "norm_grad", "dtype": "f32", "groups": 1, "rows": 50000, "width": 2400, "pitch": 2400},
        # the score of a single row against a large output layer: one read of the kernel, latency
        {"name": "loss of one row", "op": "loss", "dtype": "bf16", "rows": 1, "width": 1024, "classes": 32000, "order": "out_in", "target": "labels"},
        # a batch of 64 cells, one sub-network that predicts every gene of the 20k-gene matrix as a profile
        {"name": "loss of profiles", "op": "loss", "dtype": "f32", "rows": 64, "width": 256, "classes": 20000, "order": "in_out", "target": "profile"},
        # a large batch against a large output layer: a matrix product with a softmax behind it
        {"name": "loss of a large batch", "op": "loss", "dtype": "bf16", "rows": 4096, "width": 2048, "classes": 100000, "order": "out_in", "target": "labels"},
        # the backward pass of the profiles
        {"name": "loss grad of profiles", "op": "loss_grad", "dtype": "f32", "rows": 64, "width": 256, "classes": 20000, "order": "in_out", "target": "profile"},
        # odd sizes everywhere, the command line's 300 hidden units
        {"name": "loss grad of ragged rows", "op": "loss_grad", "dtype": "bf16", "rows": 999, "width": 300, "classes": 20011, "order": "in_out", "target": "labels"},
        # a training step of a large output layer
        {"name": "loss grad of a large batch", "op": "loss_grad", "dtype": "bf16", "rows": 4096, "width": 2048, "classes": 64000, "order": "out_in", "target": "labels"},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "loss", "loss_grad"])
    dtype = rng.choice(["f32", "bf16"])
    if op in ("norm", "norm_grad"):
        width = _log_int(rng, 16, 16384)
        groups = rng.choice([1, 1, rng.randint(2, 40)])
        rows = _log_int(rng, 1, max(1, min(50000, 100_000_000 // (width * groups))))
        return {"op": op, "dtype": dtype, "groups": groups, "rows": rows, "width": width, "pitch": width + rng.choice([0, 0, 0, 3, 8])}
    width = _log_int(rng, 16, 4096)
    if rng.random() < 0.5:
        width = (width + 63) // 64 * 64
    classes = _log_int(rng, 100, min(100000, 200_000_000 // width))
    rows = _log_int(rng, 1, min(8192, 400_000_000 // classes, 500_000_000_000 // (classes * width)))
    return {"op": op, "dtype": dtype, "rows": rows, "width": width, "classes": classes,
            "order": rng.choice(["out_in", "in_out"]), "target": rng.choice(["labels", "labels", "profile"])}


def _inputs(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed * 7919 + 17)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device=DEVICE, dtype=torch.float32)

    dtype = TYPES[case["dtype"]]
    rows, width = case["rows"], case["width"]
    if case["op"] in ("norm", "norm_grad"):
        groups, pitch = case["groups"], case["pitch"]
        lead = (groups, rows) if groups > 1 else (rows,)

        def plane():
            # what a hidden layer hands on: values around a mean and a spread of their own in every row
            full = normal(groups * rows, pitch)
            full.mul_(0.2 + 2.0 * uniform(groups * rows, 1)).add_(normal(groups * rows, 1))
            return full.to(dtype).view(*lead, pitch)[..., :width]
        x = plane()
        of_group = (groups, width) if groups > 1 else (width,)
        got = {"x": x, "gamma": 1.0 + 0.2 * normal(*of_group), "beta": 0.1 * normal(*of_group)}
        if case["op"] == "norm_grad":
            got["dy"] = plane() / rows
            mean, rstd = _moments(x.float())
            got["mean"], got["rstd"] = mean, rstd
        return got
    classes = case["classes"]
    x = normal(rows, width).to(dtype)                               # a normalised hidden layer
    kernel = normal(classes, width).mul_(2.0 / math.sqrt(width)).to(dtype)
    kernel = kernel.t() if case["order"] == "out_in" else kernel.t().contiguous()
    got = {"x": x, "kernel": kernel, "bias": 0.5 * normal(classes)}
    if case["target"] == "labels":
        # frequent and rare classes; one row in twenty is padding (a negative label)
        label = (classes * uniform(rows) ** 3).to(torch.int32).clamp_(max=classes - 1)
        if rows > 1:
            label = torch.where(uniform(rows) < 0.05, torch.full_like(label, -1), label)
        got["target"] = label
    else:
        # log1p counts, two thirds of them zero, each row scaled to a sum around one
        count = torch.floor(torch.exp(2.0 * normal(rows, classes))) * (uniform(rows, classes) < 0.4)
        got["target"] = (torch.log1p(count) * (1.0 / classes)).to(dtype)
    if case["op"] == "loss_grad":
        got["dloss"] = (0.5 + uniform(rows)) / rows
        got["lse"] = _log_sum_exp(_logits(got["x"].float(), got["kernel"].float(), got["bias"]))
    return got


def prepare(case, seed):
    state = _inputs(case, seed)
    state["op"] = case["op"]
    return state


def _moments(x):
    mean = x.mean(-1)
    centred = x - mean.unsqueeze(-1)
    return mean, (centred.square().mean(-1) + EPSILON).rsqrt()


def _logits(x, kernel, bias):
    return torch.matmul(x, kernel) + bias


def _log_sum_exp(z):
    top = z.amax(-1)
    return top + (z - top.unsqueeze(-1)).exp().sum(-1).log()


def _of_groups(p, x):
    return p.unsqueeze(-2) if x.dim() == 3 else p


def _norm(s):
    x = s["x"].float()
    mean, rstd = _moments(x)
    y = (x - mean.unsqueeze(-1)) * rstd.unsqueeze(-1) * _of_groups(s["gamma"], x) + _of_groups(s["beta"], x)
    return {"y": y.to(s["x"].dtype), "mean": mean, "rstd": rstd}


def _norm_grad(s):
    x, dy, rstd = s["x"].float(), s["dy"].float(), s["rstd"].unsqueeze(-1)
    hat = (x - s["mean"].unsqueeze(-1)) * rstd
    g = dy * _of_groups(s["gamma"], x)
    dx = rstd * (g - g.mean(-1, keepdim=True) - hat * (g * hat).mean(-1, keepdim=True))
    return {"dx": dx.to(s["x"].dtype), "dgamma": (dy * hat).sum(-2), "dbeta": dy.sum(-2)}


def _loss(s):
    z = _logits(s["x"].float(), s["kernel"].float(), s["bias"])
    lse = _log_sum_exp(z)
    t = s["target"]
    if t.dim() == 1:
        picked = z.gather(1, t.clamp(min=0).long().unsqueeze(1)).squeeze(1)
        loss = torch.where(t < 0, torch.zeros_like(lse), lse - picked)
    else:
        t = t.float()
        loss = t.sum(-1) * lse - (t * z).sum(-1)
    return {"loss": loss, "lse": lse}


def _loss_grad(s):
    x, kernel = s["x"].float(), s["kernel"].float()
    p = (_logits(x, kernel, s["bias"]) - s["lse"].unsqueeze(-1)).exp()
    t = s["target"]
    if t.dim() == 1:
        at = t.clamp(min=0).long().unsqueeze(1)
        p.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32))
        g = p * torch.where(t < 0, torch.zeros_like(s["dloss"]), s["dloss"]).unsqueeze(-1)
    else:
        t = t.float()
        g = (t.sum(-1, keepdim=True) * p - t) * s["dloss"].unsqueeze(-1)
    dx = torch.matmul(g, kernel.t())
    if s["kernel"].stride(0) == 1 and s["kernel"].stride(1) != 1:      # the gradient lies in memory as the kernel does
        dkernel = torch.matmul(g.t(), x).to(s["kernel"].dtype).t()
    else:
        dkernel = torch.matmul(x.t(), g).to(s["kernel"].dtype)
    return {"dx": dx.to(s["x"].dtype), "dkernel": dkernel, "dbias": g.sum(0)}


def run(s):
    if own:
        from deepimpute_amd import ops
        if s["op"] == "norm":
            y, mean, rstd = ops.layer_norm(s["x"], s["gamma"], s["beta"], EPSILON)
            return {"y": y, "mean": mean, "rstd": rstd}
        if s["op"] == "norm_grad":
            dx, dgamma, dbeta = ops.layer_norm_grad(s["dy"], s["x"], s["mean"], s["rstd"], s["gamma"])
            return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
        if s["op"] == "loss":
            loss, lse = ops.linear_cross_entropy(s["x"], s["kernel"], s["target"], s["bias"])
            return {"loss": loss, "lse": lse}
        dx, dkernel, dbias = ops.linear_cross_entropy_grad(s["dloss"], s["x"], s["kernel"], s["target"], s["lse"], s["bias"])
        return {"dx": dx, "dkernel": dkernel, "dbias": dbias}
    return {"norm": _norm, "norm_grad": _norm_grad, "loss": _loss, "loss_grad": _loss_grad}[s["op"]](s)


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    rows, width = case["rows"], case["width"]
    if case["op"] in ("norm", "norm_grad"):
        groups = case["groups"]
        n = groups * rows
        planes, params = (2, 2) if case["op"] == "norm" else (3, 3)
        return {"bytes": planes * n * width * size + 8 * n + 4 * params * groups * width, "flops": (8 if case["op"] == "norm" else 14) * n * width}
    classes = case["classes"]
    target = rows * classes * size if case["target"] == "profile" else 4 * rows
    read = (rows * width + width * classes) * size + 4 * classes + target
    if case["op"] == "loss":
        return {"bytes": read + 8 * rows, "flops": 2 * rows * width * classes}
    # the logits are not kept, so they are multiplied again: three products
    return {"bytes": read + 8 * rows + (rows * width + width * classes) * size + 4 * classes, "flops": 6 * rows * width * classes}


def exact(case, seed):
    s = _inputs(case, seed)
    x = s["x"].double()
    if case["op"] in ("norm", "norm_grad"):
        per = (lambda v: v.double()[:, None, :]) if x.dim() == 3 else (lambda v: v.double())
        if case["op"] == "norm":
            var, mean = torch.var_mean(x, -1, correction=0)
            hat = (x - mean[..., None]) / torch.sqrt(var + EPSILON)[..., None]
            return {"y": hat * per(s["gamma"]) + per(s["beta"]), "mean": mean, "rstd": 1.0 / torch.sqrt(var + EPSILON)}
        dy, r = s["dy"].double(), s["rstd"].double()[..., None]
        hat = r * (x - s["mean"].double()[..., None])
        g = dy * per(s["gamma"])
        n = x.shape[-1]
        dx = (r / n) * (n * g - g.sum(-1, keepdim=True) - hat * (g * hat).sum(-1, keepdim=True))
        return {"dx": dx, "dgamma": (dy * hat).sum(-2), "dbeta": dy.sum(-2)}
    kernel, bias = s["kernel"].double(), s["bias"].double()
    z = torch.addmm(bias, x, kernel)
    t = s["target"]
    if case["op"] == "loss":
        lse = torch.logsumexp(z, 1)
        if t.dim() == 1:
            valid = t >= 0
            rows = torch.arange(t.numel(), device=t.device)
            loss = torch.zeros_like(lse)
            loss[valid] = lse[valid] - z[rows[valid], t[valid].long()]
        else:
            loss = -(t.double() * (z - lse[:, None])).sum(1)
        return {"loss": loss, "lse": lse}
    p = torch.exp(z - s["lse"].double()[:, None])
    dloss = s["dloss"].double()[:, None]
    if t.dim() == 1:
        valid = t >= 0
        one_hot = torch.zeros_like(p)
        one_hot[valid, t[valid].long()] = 1.0
        g = (p - one_hot) * valid.double()[:, None] * dloss
    else:
        t = t.double()
        g = dloss * (p * t.sum(1, keepdim=True) - t)
    dkernel = x.t() @ g
    if s["kernel"].stride(0) == 1 and s["kernel"].stride(1) != 1:
        dkernel = dkernel.t().contiguous().t()
    return {"dx": g @ kernel.t(), "dkernel": dkernel, "dbias": g.sum(0)}
