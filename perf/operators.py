"""The training-side operators' cases: layer norm with its gradients, 8-bit activation checkpoints (on their own and inside a train-mode ABN), and softmax cross
entropy over depth hypotheses.  `run` computes a case in plain torch operations, or (`own`) through the framework's entry points."""
import math
from types import SimpleNamespace

import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BLOCK = 32   # values that share a scale in the 8-bit format


# ---- the cases -------------------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one pixel-major position (32 channels): the latency of a call that has next to nothing to do
        {"name": "layer_norm one row", "op": "layer_norm", "n": 1, "c": 32, "s": 1, "rows": True, "dtype": "float32", "train": False, "slope": 0.01},
        # FeatureNet's full-resolution maps of a training step: 2 samples x 3 views at 640x512, 8 channels
        {"name": "layer_norm feature maps", "op": "layer_norm", "n": 6, "c": 8, "s": 512 * 640, "rows": False, "dtype": "float32", "train": True, "slope": 0.01},
        # the regulariser's innermost layer at cascade level 2 (64 channels, 6 x 16 x 20): few positions, many channels
        {"name": "layer_norm bottleneck", "op": "layer_norm", "n": 2, "c": 64, "s": 6 * 16 * 20, "rows": False, "dtype": "float32", "train": True, "slope": 0.01},
        # wide rows in bf16, odd sizes, no activation: the generic form of the operator
        {"name": "layer_norm rows bf16", "op": "layer_norm", "n": 8191, "c": 1000, "s": 1, "rows": True, "dtype": "bfloat16", "train": True, "slope": 1.0},
        # the first volume of the middle cascade level, one sample of 8 x 32 x 256 x 320
        {"name": "layer_norm volume", "op": "layer_norm", "n": 2, "c": 8, "s": 32 * 256 * 320, "rows": False, "dtype": "float32", "train": True, "slope": 0.01},
        # a small skip tensor of the regulariser packed and read back
        {"name": "pack8 small", "op": "pack8", "n": 32, "s": 2 * 8 * 10, "dtype": "float32"},
        # the coarse level's cost volume, 2 samples of 32 x 48 x 128 x 160: the largest tensor that a convolution keeps as its input
        {"name": "pack8 cost volume", "op": "pack8", "n": 2 * 32, "s": 48 * 128 * 160, "dtype": "float32"},
        # train-mode ABN with 8-bit checkpoints: the innermost layer, the full-resolution feature maps, the largest volume of a step
        {"name": "abn8 bottleneck", "op": "abn8", "n": 2, "c": 64, "s": 6 * 16 * 20, "slope": 0.01},
        {"name": "abn8 feature maps", "op": "abn8", "n": 6, "c": 8, "s": 512 * 640, "slope": 0.01},
        {"name": "abn8 volume", "op": "abn8", "n": 2, "c": 8, "s": 32 * 256 * 320, "slope": 0.01},
        # the coarse level of a training step (48 hypotheses at 160x128, per-pixel planes)
        {"name": "depth_ce level 2", "op": "depth_ce", "n": 2, "d": 48, "h": 128, "w": 160, "dtype": "float32", "per_pixel": True},
        # a single-level sweep over 192 planes, odd image, bf16 costs, one set of planes per sample
        {"name": "depth_ce deep bf16", "op": "depth_ce", "n": 1, "d": 192, "h": 295, "w": 399, "dtype": "bfloat16", "per_pixel": False},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("layer_norm", "layer_norm", "pack8", "abn8", "depth_ce", "depth_ce"))
    dtype = rng.choice(("float32", "float32", "bfloat16", "float16"))
    if op == "layer_norm":
        rows = rng.random() < 0.4
        slope = rng.choice((1.0, 0.01))
        train = rng.random() < 0.7
        if rows:   # from one token to many, narrow rows to wide ones
            c = _spread(rng, 1, 8192)
            return {"op": op, "n": _spread(rng, 1, min(16384, (1 << 24) // c)), "c": c, "s": 1, "rows": True, "dtype": dtype, "train": train, "slope": slope}
        c = rng.choice((8, 16, 32, 64, _spread(rng, 1, 512)))
        n = rng.randint(1, 6)
        return {"op": op, "n": n, "c": c, "s": _spread(rng, 1, (1 << 24) // (n * c)), "rows": False, "dtype": dtype, "train": train, "slope": slope}
    if op == "pack8":
        n = _spread(rng, 1, 256)
        return {"op": op, "n": n, "s": _spread(rng, 1, (1 << 25) // n), "dtype": dtype}
    if op == "abn8":
        n, c = rng.randint(1, 6), rng.choice((8, 16, 32, 64, rng.randint(1, 64)))
        return {"op": op, "n": n, "c": c, "s": _spread(rng, 16, (1 << 24) // (n * c)), "slope": rng.choice((0.01, 0.01, 0.0, 1.0))}
    n, d = rng.randint(1, 4), rng.choice((8, 32, 48, _spread(rng, 2, 512)))
    most = min(512, int(math.sqrt((1 << 23) / (n * d))))
    # (float16 costs would need a loss scale: a mean over many pixels has gradients below that type's normal numbers)
    dtype = rng.choice(("float32", "float32", "bfloat16"))
    return {"op": op, "n": n, "d": d, "h": _spread(rng, 8, most), "w": _spread(rng, 8, most), "dtype": dtype, "per_pixel": rng.random() < 0.7}


# ---- what a program has in hand ------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def rand(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    op = case["op"]
    dtype = _DTYPES[case.get("dtype", "float32")]
    if op == "layer_norm":
        n, c, s = case["n"], case["c"], case["s"]
        tail = () if case["rows"] else (s,)
        spread = (1, c) + (1,) * len(tail)
        x = (randn(n, c, *tail) * (rand(*spread) + 0.5) + randn(*spread) * 0.5).to(dtype)   # a layer's output: every channel has its own offset and size
        return {"x": x, "weight": rand(c) + 0.5, "bias": randn(c) * 0.3, "grad": randn(n, c, *tail).to(dtype) if case["train"] else None,
                "slope": case["slope"]}
    if op == "pack8":
        n, s = case["n"], case["s"]
        return {"x": (randn(n, s) * (rand(n, 1) * 3 + 0.1)).to(dtype)}
    if op == "abn8":
        n, c, s = case["n"], case["c"], case["s"]
        norm = SimpleNamespace(weight=rand(c) + 0.5, bias=randn(c) * 0.3, running_mean=torch.zeros(c, device="cuda"), running_var=torch.ones(c, device="cuda"),
                               momentum=0.1, eps=1e-5, activation_param=case["slope"], affine=True)
        return {"x": randn(n, c, s) * (rand(1, c, 1) + 0.5) + randn(1, c, 1) * 0.5, "norm": norm, "grad": randn(n, c, s)}
    n, d, h, w = case["n"], case["d"], case["h"], case["w"]
    interval = 2.65
    k = torch.arange(d, device="cuda", dtype=torch.float32)
    first = 425.0 + 200.0 * rand(n, h, w) if case["per_pixel"] else (425.0 + 20.0 * rand(n)).view(n, 1, 1).expand(n, h, w)
    true = rand(n, h, w) * (d + 1.0) - 1.0   # in intervals; some pixels lie outside the sweep
    values = first.unsqueeze(1) + interval * k.view(1, d, 1, 1)
    cost = randn(n, d, h, w) * 1.5 - 0.3 * (k.view(1, d, 1, 1) - true.unsqueeze(1)).abs().clamp(max=8.0)   # a sweep that has begun to find the surface
    return {"cost": cost.to(dtype), "values": values.contiguous() if case["per_pixel"] else values[:, :, 0, 0].contiguous(),
            "gt": (first + interval * true).contiguous(), "mask": rand(n, h, w) < 0.7}


def work(case):
    op = case["op"]
    size = {"float32": 4}.get(case.get("dtype", "float32"), 2)
    if op == "layer_norm":
        numel = case["n"] * case["c"] * case["s"]
        return {"bytes": numel * size * (4 if case["train"] else 2) + case["c"] * (16 if case["train"] else 8), "flops": numel * (22 if case["train"] else 8)}
    if op == "pack8":
        return {"bytes": case["n"] * case["s"] * 2 * size, "flops": 4 * case["n"] * case["s"]}
    if op == "abn8":
        numel = case["n"] * case["c"] * case["s"]
        return {"bytes": numel * 16 + case["c"] * 32, "flops": 20 * numel}
    pixels = case["n"] * case["h"] * case["w"]
    return {"bytes": pixels * case["d"] * (2 * size + (4 if case["per_pixel"] else 0)) + pixels * 5 + (0 if case["per_pixel"] else 4 * case["n"] * case["d"]),
            "flops": 10 * pixels * case["d"]}


# ---- one pass ----------------------------------------------------------------------------------------------------------------------------------------
def _over_channels(t):
    return [i for i in range(t.dim()) if i != 1]


def _plain_layer_norm(x, weight, bias, grad, slope, eps=1e-5):
    spread = (1, -1) + (1,) * (x.dim() - 2)
    # 64 bits: with an activation, for the side of its border that z lies on; with a few channels, where the gradient is what is left after cancellation
    few = x.shape[1] < 8
    v = x.double() if slope != 1.0 or few else x.float()
    mean = v.mean(1, keepdim=True)
    v = v - mean
    rstd = 1.0 / torch.sqrt((v * v).mean(1, keepdim=True) + eps)
    xhat = v * rstd
    z = xhat * weight.view(spread) + bias.view(spread)
    up = z > 0
    y = torch.where(up, z, z * slope).to(x.dtype)
    if grad is None:
        return {"y": y}
    g = grad.to(v.dtype if few else torch.float32) * torch.where(up, 1.0, slope)
    xhat, rstd = xhat.to(g.dtype), rstd.to(g.dtype)
    gw = g * weight.view(spread)
    gx = rstd * (gw - gw.mean(1, keepdim=True) - xhat * (gw * xhat).mean(1, keepdim=True))
    over = _over_channels(x)
    return {"y": y, "gx": gx.to(x.dtype), "gweight": (g * xhat).sum(over, dtype=torch.float64).float(), "gbias": g.sum(over, dtype=torch.float64).float()}


def _power_of_two(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _plain_8bit(v):
    """The values that the last axis of `v` (float64) is held as: blocks of 32, one power-of-two step per block, 7 bits and a sign."""
    n = v.shape[-1]
    blocks = -(-n // BLOCK)
    v = torch.nn.functional.pad(v, (0, blocks * BLOCK - n)).unflatten(-1, (blocks, BLOCK))
    largest = v.abs().amax(-1, keepdim=True)
    exponent = torch.where(largest > 0, torch.frexp(largest).exponent - 1, -127).clamp(min=-127)
    step = _power_of_two(exponent - 6)
    held = (v.abs() / step).round().clamp(max=127.0) * step
    return torch.where(v < 0, -held, held).flatten(-2)[..., :n]


def _plain_abn8(x, norm, grad, slope):
    count = x.numel() // x.shape[1]
    v = x.double()
    mean = v.mean((0, 2), keepdim=True)
    var = ((v - mean) ** 2).mean((0, 2), keepdim=True)
    rstd = 1.0 / torch.sqrt(var + norm.eps)
    xhat = (v - mean) * rstd
    z = xhat * norm.weight.view(1, -1, 1) + norm.bias.view(1, -1, 1)
    up = z > 0
    y = torch.where(up, z, z * slope).float()
    kept = _plain_8bit(xhat).float()
    norm.running_mean.mul_(1.0 - norm.momentum).add_(norm.momentum * mean.flatten().float())
    norm.running_var.mul_(1.0 - norm.momentum).add_(norm.momentum * (var.flatten() * (count / max(count - 1, 1))).float())
    g = grad * torch.where(up, 1.0, slope)
    gb, gw = g.sum((0, 2), dtype=torch.float64), (g * kept).sum((0, 2), dtype=torch.float64)
    scale = (norm.weight * rstd.flatten()).float().view(1, -1, 1)
    gx = scale * (g - (gb / count).float().view(1, -1, 1) - kept * (gw / count).float().view(1, -1, 1))
    return {"y": y, "gx": gx, "gweight": gw.float(), "gbias": gb.float(), "running_mean": norm.running_mean, "running_var": norm.running_var}


def _plain_depth_ce(cost, values, gt, mask):
    c = cost.float()
    if values.dim() == 2:
        values = values.view(*values.shape, 1, 1).expand_as(c)
    nearest = (values.double() - gt.double().unsqueeze(1)).abs().argmin(1, keepdim=True)   # next to a border between two planes: 64 bits
    counted = mask & (gt >= values.amin(1)) & (gt <= values.amax(1))
    count = counted.sum()
    top = c.amax(1, keepdim=True)
    e = torch.exp(c - top)
    total = e.sum(1, keepdim=True)
    each = (torch.log(total) + top - c.gather(1, nearest)).squeeze(1)
    share = torch.where(count > 0, 1.0 / count, 0.0)
    loss = (torch.where(counted, each, 0.0).sum(dtype=torch.float64) * share).float()
    weight = torch.where(counted, share, 0.0).unsqueeze(1).float()
    grad = e / total * weight
    grad.scatter_add_(1, nearest, -weight)
    return {"loss": loss, "gcost": grad.to(cost.dtype)}


def run(state):
    if "values" in state:
        if own:
            from casmvsnet_pl_amd import autograd
            cost = state["cost"].detach().requires_grad_()
            loss = autograd.depth_cross_entropy(cost, state["values"], state["gt"], state["mask"])
            return {"loss": loss, "gcost": torch.autograd.grad(loss, cost)[0]}
        return _plain_depth_ce(state["cost"], state["values"], state["gt"], state["mask"])
    if "norm" in state:
        norm = state["norm"]
        if own:
            from casmvsnet_pl_amd import training
            x, norm = state["x"].detach().requires_grad_(), SimpleNamespace(**vars(norm))
            norm.weight, norm.bias = norm.weight.detach().requires_grad_(), norm.bias.detach().requires_grad_()
            y = training.abn_train(norm, x, checkpoint="8bit")
            gx, gw, gb = torch.autograd.grad(y, (x, norm.weight, norm.bias), state["grad"])
            return {"y": y, "gx": gx, "gweight": gw, "gbias": gb, "running_mean": norm.running_mean, "running_var": norm.running_var}
        return _plain_abn8(state["x"], norm, state["grad"], norm.activation_param)
    if "weight" in state:
        x, weight, bias, grad = state["x"], state["weight"], state["bias"], state["grad"]
        slope, rows = state["slope"], x.dim() == 2
        if own:
            from casmvsnet_pl_amd import autograd, ops
            if grad is None:
                return {"y": ops.layer_norm(x, weight, bias, slope=slope, channels_last=rows)}
            x, weight, bias = x.detach().requires_grad_(), weight.detach().requires_grad_(), bias.detach().requires_grad_()
            y = autograd.layer_norm(x, weight, bias, slope=slope, channels_last=rows)
            gx, gw, gb = torch.autograd.grad(y, (x, weight, bias), grad)
            return {"y": y, "gx": gx, "gweight": gw, "gbias": gb}
        return _plain_layer_norm(x, weight, bias, grad, slope)
    if own:
        from casmvsnet_pl_amd import ops
        return {"values": ops.unpack8(ops.pack8(state["x"]))}
    return {"values": _plain_8bit(state["x"].double()).to(state["x"].dtype)}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "pack8":
        return {"values": _held(state["x"].double())}
    if op == "layer_norm":
        x, w, b = state["x"].double(), state["weight"].double(), state["bias"].double()
        x = x.movedim(1, -1)
        x = x - x.mean(-1, keepdim=True)
        size = torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-5)
        x /= size
        z = x * w + b
        factor = torch.ones_like(z).masked_fill_(z <= 0, case["slope"])
        y = (z * factor).movedim(-1, 1)
        if state["grad"] is None:
            return {"y": y}
        del z
        g = state["grad"].double().movedim(1, -1) * factor
        del factor
        over = tuple(range(g.dim() - 1))
        gw, gb = (g * x).sum(over), g.sum(over)
        g = g * w
        gx = (g - g.mean(-1, keepdim=True) - x * (x * g).mean(-1, keepdim=True)) / size
        return {"y": y, "gx": gx.movedim(-1, 1), "gweight": gw, "gbias": gb}
    if op == "abn8":
        norm = state["norm"]
        x = state["x"].double().transpose(0, 1)
        c, n, s = x.shape
        mean, var = x.mean((1, 2)), x.var((1, 2), unbiased=False)
        size = torch.sqrt(var + norm.eps)
        x = (x - mean.view(c, 1, 1)) / size.view(c, 1, 1)
        z = x * norm.weight.double().view(c, 1, 1) + norm.bias.double().view(c, 1, 1)
        factor = torch.ones_like(z).masked_fill_(z <= 0, case["slope"])
        y = (z * factor).transpose(0, 1)
        del z
        x = _held(x)
        g = state["grad"].double().transpose(0, 1) * factor
        gw, gb = (g * x).sum((1, 2)), g.sum((1, 2))
        g = g - (gb / (n * s)).view(c, 1, 1) - x * (gw / (n * s)).view(c, 1, 1)
        g = g * (norm.weight.double() / size).view(c, 1, 1)
        unbiased = var * (n * s) / max(n * s - 1, 1)
        return {"y": y, "gx": g.transpose(0, 1), "gweight": gw, "gbias": gb, "running_mean": 0.1 * mean, "running_var": 0.9 + 0.1 * unbiased}
    cost, values, gt = state["cost"].double(), state["values"].double(), state["gt"].double()
    n, d, h, w = cost.shape
    if values.dim() == 2:
        values = values.reshape(n, d, 1, 1).expand(n, d, h, w)
    counted = (state["mask"] & (values.min(1).values <= gt) & (gt <= values.max(1).values)).double()
    count = counted.sum().clamp(min=1.0)
    hot = torch.zeros_like(cost)
    hot.scatter_(1, (values - gt.unsqueeze(1)).abs().min(1, keepdim=True).indices, 1.0)
    log_p = torch.log_softmax(cost, 1)
    loss = -((log_p * hot).sum(1) * counted).sum() / count
    return {"loss": loss, "gcost": (log_p.exp() - hot) * (counted / count).unsqueeze(1)}


def _held(v):
    """What the 8-bit format holds of the last axis of `v`: 127 steps up and down of 2^(floor(log2 largest) - 6) for each run of 32 values."""
    n = v.shape[-1]
    out = torch.zeros(v.shape[:-1] + ((n + 31) // 32 * 32,), dtype=torch.float64, device=v.device)
    out[..., :n] = v
    out = out.reshape(v.shape[:-1] + (-1, 32))
    top = out.abs().max(-1, keepdim=True).values
    # the power of two at or below the largest magnitude, by its bits
    unit = (top.view(torch.int64) & (0x7FF << 52)).view(torch.float64).clamp(min=2.0 ** -127) / 64.0
    out = torch.round(out / unit).clamp(-127.0, 127.0) * unit
    return out.reshape(v.shape[:-1] + (-1,))[..., :n]
