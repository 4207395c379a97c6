"""GPU tests of the training-side operators: layer norm (forward, gradients), 8-bit checkpoints (packing, the ABN and the convolution that use them), cross entropy
over depth hypotheses, and a training step that uses them together - each against its definition in float64.

Tolerances.  A rounding to type t is off by at most half a step, finfo(t).eps / 2 of the value.  Layer norm and ABN form statistics, x - mean and the side of zero
in 64 bits; y's few float32 roundings are counted where it is checked (a 16-bit type's own comes on top).  Gradients: every term passes at most 16 float32 roundings on its way; weight gradients at
most 64 of them before 64-bit sums take over; each bound is that many half steps of the terms' magnitudes, plus the output's own rounding."""
import math

import pytest
import torch

import casmvsnet_pl_amd as M
from casmvsnet_pl_amd import autograd as A
from casmvsnet_pl_amd import ops
from casmvsnet_pl_amd import training as T

pytestmark = pytest.mark.gpu
U = 2.0 ** -24   # half a step of float32
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a MI355X"
    return torch.device("cuda:0")


def rounding(want, dtype):
    """Half a step of `dtype` at `want` (its subnormals included), float32's on the way to a 16-bit type."""
    f = torch.finfo(dtype)
    return want.abs() * (f.eps / 2 + (U if dtype != F32 else 0.0)) + f.smallest_normal * f.eps / 2


def rebuilt(x):
    """The input that a convolution with 8-bit checkpoints takes its weight gradient at."""
    tensors, rebuild = T.kept_input(x)
    return rebuild(*tensors)


def within(got, want, limit):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    limit = limit.cpu() if isinstance(limit, torch.Tensor) else limit
    off = (got - want).abs()
    worst = float(torch.where(off == 0, 0.0, off / limit).max()) if got.numel() else 0.0
    assert got.shape == want.shape and worst <= 1.0, f"{worst:.3g} times the bound, at most {float(off.max()):.3g} off"


# ---- layer norm ---------------------------------------------------------------------------------------------------------------------------------
def ln_reference(x, w, b, gy, eps, slope, dim):
    """y, gx, gw, gb in float64 and the magnitudes their bounds go by."""
    x = x.double().movedim(dim, -1)
    gy = gy.double().movedim(dim, -1)
    C = x.shape[-1]
    w = torch.ones(C, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(C, dtype=torch.float64) if b is None else b.double()
    d = x - x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + float(torch.tensor(eps)))
    h = d * r
    z = h * w + b
    factor = torch.where(z > 0, 1.0, float(torch.tensor(slope)))
    y, g = z * factor, gy * factor
    gw, m1, m2 = g * w, (g * w).mean(-1, keepdim=True), (g * w * h).mean(-1, keepdim=True)
    gx = r * (gw - m1 - h * m2)
    terms = r * (gw.abs() + gw.abs().mean(-1, keepdim=True) + h.abs() * (gw * h).abs().mean(-1, keepdim=True))
    over = tuple(range(x.dim() - 1))
    # the mean's own rounding in 64 bits: at most 72 additions and the division, each 2^-53 of the sum of |x|; it moves z by its size times r |w|, which a row far from
    # zero sees where z itself is small (an offset of 3e6: 3e6 * 2^-53 = 3e-10, against half a float32 step of 6e-10 at z = 0.01)
    far = 80 * 2.0 ** -53 * x.abs().mean(-1, keepdim=True) * r * w.abs()
    # z in float32 from the rounded x - mean (8 channels and more): that rounding, r's, two products and the sum's - four half steps of |h w|, one of |z| - and one of
    # the slope's product.  (At fewer channels and next to zero z is 64 bits wide and is rounded once.)
    far = far + torch.where(z > 0, 1.0, abs(slope)) * U * (4 * (h * w).abs() + 2 * z.abs()) * 1.001
    return (y.movedim(-1, dim), far.movedim(-1, dim), gx.movedim(-1, dim), (g * h).sum(over), g.sum(over), terms.movedim(-1, dim), (g * h).abs().sum(over), g.abs().sum(over))


def ln_check(dev, x, w, b, gy, eps=1e-5, slope=0.01, channels_last=False):
    dim = -1 if channels_last else 1
    y, far, gx, gw, gb, terms, aw, ab = ln_reference(x, w, b, gy, eps, slope, dim)
    xd = x.to(dev).requires_grad_()
    wd, bd = (None if t is None else t.to(dev).requires_grad_() for t in (w, b))
    got = A.layer_norm(xd, wd, bd, eps, slope, channels_last)
    assert got.dtype == x.dtype and got.shape == x.shape
    assert torch.equal(got, ops.layer_norm(xd, wd, bd, eps, slope, channels_last))
    within(got, y, rounding(y, x.dtype) + far)
    got.backward(gy.to(dev))
    assert xd.grad.dtype == x.dtype
    within(xd.grad, gx, rounding(gx, x.dtype) + 16 * U * terms)
    if w is not None:
        within(wd.grad, gw, 64 * U * aw + rounding(gw, F32))
        within(bd.grad, gb, 64 * U * ab + rounding(gb, F32))


_LN_MAPS = [(2, 8, 6, 10), (1, 16, 3, 4, 8), (2, 32, 5, 7), (3, 64, 33), (1, 1, 9), (2, 2, 40), (2, 3, 64), (1, 20, 6), (1, 100, 17), (1, 512, 24), (1, 513, 12),
            (2, 700, 3), (6, 8, 1000), (1, 8, 4097), (1, 5, 3)]
_LN_ROWS = [(1, 32), (1, 1), (5, 3), (7, 8), (300, 16), (4, 31), (9, 64), (33, 100), (3, 1000), (70, 1001), (2, 2048), (3, 2050), (2, 8192), (2, 8193), (1, 20000), (2, 3, 40)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("slope", [0.01, 1.0])
@pytest.mark.parametrize("shape,rows", [(s, False) for s in _LN_MAPS] + [(s, True) for s in _LN_ROWS])
def test_layer_norm_and_gradients_against_float64(dev, shape, rows, slope, dtype):
    g = torch.Generator().manual_seed(sum(shape) + len(shape))
    C = shape[-1] if rows else shape[1]
    x = (torch.randn(shape, generator=g) * 1.7 + 0.6).to(dtype)
    ln_check(dev, x, torch.rand(C, generator=g) + 0.5, torch.randn(C, generator=g) * 0.3, torch.randn(shape, generator=g).to(dtype), slope=slope, channels_last=rows)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape,rows", [((5000, 264), True), ((70000, 9), True), ((600, 2100), True), ((1100, 1030), True), ((70000, 6), True), ((2, 8, 300002), False),
                                        ((1, 20, 100003), False), ((2, 100, 20004), False), ((3, 3, 300000), False)])
def test_layer_norm_where_a_workgroup_takes_several_turns(dev, shape, rows, dtype):
    """More rows / tiles than the passes have workgroups for: what is loaded ahead for the next turn, and the last turn that only some of them have."""
    g = torch.Generator().manual_seed(sum(shape))
    C = shape[-1] if rows else shape[1]
    x = (torch.randn(shape, generator=g) * 1.7 + 0.6).to(dtype)
    ln_check(dev, x, torch.rand(C, generator=g) + 0.5, torch.randn(C, generator=g) * 0.3, torch.randn(shape, generator=g).to(dtype), channels_last=rows)


@pytest.mark.parametrize("rows", [False, True])
def test_layer_norm_without_affine_and_with_the_relu_slope(dev, rows):
    g = torch.Generator().manual_seed(1)
    shape = (40, 24) if rows else (2, 24, 20)
    ln_check(dev, torch.randn(shape, generator=g), None, None, torch.randn(shape, generator=g), slope=0.0, channels_last=rows)


@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("offset", [1e4, 3e6])
def test_layer_norm_far_from_zero(dev, rows, offset):
    """Rows whose mean is many times their spread: the 64-bit statistics see what float32 holds of them; and constant rows: 0 before the affine."""
    g = torch.Generator().manual_seed(2)
    shape = (30, 48) if rows else (2, 48, 21)
    x = torch.randn(shape, generator=g) + offset
    ln_check(dev, x, torch.rand(48, generator=g) + 0.5, torch.randn(48, generator=g), torch.randn(shape, generator=g), channels_last=rows)
    w, b = torch.rand(48, generator=g).to(dev), torch.randn(48, generator=g).to(dev)
    y = ops.layer_norm(torch.full(shape, offset, device=dev), w, b, channels_last=rows)
    assert torch.equal(y, b.expand(shape) if rows else b.view(1, 48, 1).expand(shape))


@pytest.mark.parametrize("rows", [False, True])
def test_layer_norm_non_finite_positions_stay_apart(dev, rows):
    g = torch.Generator().manual_seed(3)
    x = torch.randn((50, 24), generator=g) if rows else torch.randn((2, 24, 50), generator=g)
    clean = ops.layer_norm(x.to(dev), channels_last=rows)
    bad = x.clone()
    pick = (lambda t, p: t[p]) if rows else (lambda t, p: t[1, :, p])
    pick(bad, 7)[3] = float("inf")
    pick(bad, 31)[0] = float("nan")
    xb = bad.to(dev).requires_grad_()
    w = torch.ones(24, device=dev, requires_grad=True)
    got = A.layer_norm(xb, w, None, channels_last=rows)
    got.backward(torch.ones_like(got))
    hit = torch.zeros_like(x, dtype=torch.bool)
    pick(hit, 7)[:] = True
    pick(hit, 31)[:] = True
    assert bool(torch.isnan(got[hit.to(dev)]).all()) and torch.equal(got[~hit.to(dev)], clean[~hit.to(dev)])
    assert bool(torch.isfinite(xb.grad[~hit.to(dev)]).all()) and bool(torch.isnan(xb.grad[hit.to(dev)]).all()) and bool(torch.isnan(w.grad).all())


def test_layer_norm_empty_strided_and_partial_gradients(dev):
    w, b = torch.rand(8, device=dev, requires_grad=True), torch.rand(8, device=dev, requires_grad=True)
    for shape, rows in (((0, 8), True), ((0, 8, 5), False), ((2, 8, 0), False)):
        y = A.layer_norm(torch.zeros(shape, device=dev, requires_grad=True), w, b, channels_last=rows)
        gw, gb = torch.autograd.grad(y.sum(), (w, b))
        assert y.shape == shape and not gw.any() and not gb.any()
    g = torch.Generator().manual_seed(4)
    base = torch.randn((3, 9, 7, 8), generator=g).to(dev)
    x = base.permute(0, 3, 1, 2)[:, :, ::2]   # channels-last memory, every other row
    assert not x.is_contiguous()
    assert torch.equal(ops.layer_norm(x, w, b), ops.layer_norm(x.contiguous(), w, b))
    xc = x.contiguous().requires_grad_()
    y = A.layer_norm(xc, w, b)
    full = torch.autograd.grad(y, (xc, w, b), torch.ones((), device=dev).expand_as(y), retain_graph=True)   # an expanded gradient
    assert torch.equal(torch.autograd.grad(y, xc, torch.ones_like(y), retain_graph=True)[0], full[0])
    yw = A.layer_norm(xc.detach(), w, b)   # only the affine wants gradients
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(yw.sum(), (w, b)), full[1:]))
    shifted = torch.empty(xc.numel() + 1, device=dev)[1:].view(xc.shape).copy_(xc.detach())   # not on a 16-byte boundary
    assert shifted.data_ptr() % 16 == 4 and torch.equal(ops.layer_norm(shifted, w, b), y.detach())
    gx, gw, gb = ops.layer_norm_backward(shifted, torch.ones_like(shifted), w, b)
    assert torch.equal(gx, full[0]) and float((gw - full[1]).abs().max()) < 1e-3 and float((gb - full[2]).abs().max()) < 1e-3


@pytest.mark.parametrize("rows", [False, True])
def test_layer_norm_gradient_against_differences(dev, rows):
    g = torch.Generator().manual_seed(5)
    shape = (6, 12) if rows else (2, 12, 3)
    x, w, b, gy = torch.randn(shape, generator=g), torch.rand(12, generator=g) + 0.5, torch.randn(12, generator=g) * 0.3, torch.randn(shape, generator=g)
    dim = -1 if rows else 1
    xd, wd, bd = x.to(dev).requires_grad_(), w.to(dev).requires_grad_(), b.to(dev).requires_grad_()
    A.layer_norm(xd, wd, bd, channels_last=rows).backward(gy.to(dev))
    value = lambda x_, w_, b_: float((ln_reference(x_, w_, b_, gy, 1e-5, 1.0, dim)[0] * gy.double()).sum())
    for got, at in ((xd.grad, 0), (wd.grad, 1), (bd.grad, 2)):
        args = [x.double(), w.double(), b.double()]
        flat = got.cpu().flatten()
        for i in range(0, flat.numel(), 5):
            e = 1e-5
            ends = []
            for sign in (1, -1):
                moved = [t.clone() for t in args]
                moved[at].view(-1)[i] += sign * e
                ends.append(value(*moved))
            # central differences: the third derivative's term is of the order e^2
            assert abs((ends[0] - ends[1]) / (2 * e) - float(flat[i])) < 2e-5 * (1 + abs(float(flat[i])))


def test_layer_norm_refuses_what_does_not_fit(dev):
    x = torch.zeros(2, 8, 4, device=dev)
    with pytest.raises(ValueError, match="weight"):
        ops.layer_norm(x, torch.ones(4, device=dev))
    with pytest.raises(TypeError, match="float32"):
        ops.layer_norm(x, torch.ones(8, device=dev, dtype=F16))
    with pytest.raises(TypeError, match="float64"):
        ops.layer_norm(x.double())
    with pytest.raises(ValueError, match="channel axis"):
        ops.layer_norm(torch.zeros(4, device=dev))
    with pytest.raises(ValueError, match="eps"):
        ops.layer_norm(x, eps=float("nan"))
    with pytest.raises(ValueError, match="channels"):
        ops.layer_norm(torch.zeros(2, 70000, device=dev))
    with pytest.raises(ValueError, match="grad_y"):
        ops.layer_norm_backward(x, torch.zeros(2, 8, 5, device=dev))
    with pytest.raises(ValueError, match="LayerNormAct"):
        M.LayerNormAct(4).to(dev)(x)


# ---- 8 bits ---------------------------------------------------------------------------------------------------------------------------------------
def held(x):
    """What the 8-bit format holds of float64 planes (rows, n), and each value's step."""
    rows, n = x.shape
    nb = -(-n // 32)
    p = torch.zeros(rows, nb * 32, dtype=torch.float64)
    p[:, :n] = x
    p = p.view(rows, nb, 32)
    top = p.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -140))).clamp(min=-127)
    step = torch.pow(2.0, torch.where(torch.isfinite(e), e, 0.0) - 6)
    q = torch.round(p.abs() / step).clamp(max=127) * step * torch.where(torch.signbit(p), -1.0, 1.0)
    q = torch.where(torch.isfinite(top), q, float("nan"))
    return q.view(rows, -1)[:, :n], step.expand(rows, nb, 32).reshape(rows, -1)[:, :n]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(1,), (33,), (5, 31), (4, 32), (3, 100), (2, 3, 7, 9), (2, 8, 4, 16, 20), (1, 1, 1), (64, 960), (3, 4, 20001), ()])
def test_pack8_holds_what_the_format_says(dev, shape, dtype):
    g = torch.Generator().manual_seed(len(shape) + sum(shape))
    x = torch.randn(shape, generator=g) * torch.exp(2 * torch.randn(shape, generator=g))
    x = (x * (torch.rand(shape, generator=g) > 0.3)).to(dtype)
    packed = ops.pack8(x.to(dev))
    got = ops.unpack8(packed)
    rows, n = ops._planes(shape)
    want, step = held(x.double().reshape(rows, n))
    assert got.dtype == dtype and got.shape == x.shape and packed.nbytes == rows * -(-n // 32) * 33
    assert torch.equal(got.cpu().reshape(rows, n), want.to(dtype))
    within(got.cpu().reshape(rows, n).double(), x.double().reshape(rows, n), step + rounding(want, dtype))   # a step at most (where the largest saturates), else half


def test_pack8_special_values(dev):
    tiny, low = 2.0 ** -149, torch.finfo(F32).min
    blocks = torch.zeros(7, 32)
    blocks[0, 3], blocks[1, 5], blocks[2, 31] = float("inf"), float("nan"), float("-inf")
    blocks[3] = tiny * torch.arange(32)
    blocks[4] = torch.linspace(-1, 1, 32) * torch.finfo(F32).max
    blocks[5] = torch.tensor([127.5, 126.5, 125.5, 0.5, 1.5, -0.5, -127.9, 64.0] * 4)   # halves go to even, the largest saturate
    blocks[6, :2] = torch.tensor([low, low / 3])
    got = ops.unpack8(ops.pack8(blocks.to(dev))).cpu()
    assert bool(torch.isnan(got[:3]).all())
    want, _ = held(blocks[3:].double())
    assert torch.equal(got[3:].double(), want)
    assert torch.equal(got[5], torch.tensor([127.0, 126.0, 126.0, 0.0, 2.0, -0.0, -127.0, 64.0] * 4))
    x = torch.randn(3, 4, 10, device=dev)[:, :, ::2]
    assert torch.equal(ops.unpack8(ops.pack8(x)), ops.unpack8(ops.pack8(x.contiguous())))
    empty = ops.unpack8(ops.pack8(torch.zeros(2, 0, 5, device=dev)))
    assert empty.shape == (2, 0, 5)
    shifted = torch.empty(65, device=dev)[1:].copy_(torch.randn(64, device=dev)).view(2, 32)
    assert torch.equal(ops.unpack8(ops.pack8(shifted)), ops.unpack8(ops.pack8(shifted.clone())))


@pytest.mark.parametrize("shape", [(2, 3, 50), (1, 4, 4, 8, 8)])
def test_unpack8_with_an_affine(dev, shape):
    g = torch.Generator().manual_seed(6)
    x, w, b = torch.randn(shape, generator=g).to(dev), torch.randn(shape[1], generator=g).to(dev), torch.randn(shape[1], generator=g).to(dev)
    packed = ops.pack8(x)
    q = ops.unpack8(packed).double()
    packed.affine = (w, b, 0.01)
    view = (1, -1) + (1,) * (len(shape) - 2)
    z = q * w.double().view(view) + b.double().view(view)
    slope = float(torch.tensor(0.01))
    z = torch.where(z > 0, z, z * slope)
    within(ops.unpack8(packed), z, 2 * U * (z.abs() + 1e-30) + 2.0 ** -149)   # the fma and the slope
    packed.affine = (w[:-1], b[:-1], 0.01)
    with pytest.raises(ValueError, match="affine"):
        ops.unpack8(packed)


# ---- ABN with 8-bit checkpoints ----------------------------------------------------------------------------------------------------------------------
def abn8_reference(x, w, b, gy, slope, eps, inplace):
    x, gy = x.double(), gy.double()
    N, C = x.shape[:2]
    x, gy = x.reshape(N, C, -1), gy.reshape(N, C, -1)
    count = N * x.shape[2]
    mean, var = x.mean((0, 2)), x.var((0, 2), unbiased=False)
    r = 1 / torch.sqrt(var + float(torch.tensor(eps)))
    gamma = (w.abs() + torch.tensor(eps)).double() if inplace else w.double()
    v = lambda t: t.view(1, C, 1)
    h = (x - v(mean)) * v(r)
    z = h * v(gamma) + v(b.double())
    factor = torch.where(z > 0, 1.0, float(torch.tensor(slope)))
    q, _ = held(h.reshape(N * C, -1))
    q, g = q.view_as(h), gy * factor
    gb, gw = g.sum((0, 2)), (g * q).sum((0, 2))
    gx = v(gamma * r) * (g - v(gb / count) - q * v(gw / count))
    terms = v(gamma.abs() * r) * (g.abs() + v(g.abs().sum((0, 2)) / count) + q.abs() * v((g * q).abs().sum((0, 2)) / count))
    return z * factor, gx, gw * (torch.sign(w.double()) if inplace else 1.0), gb, terms, (g * q).abs().sum((0, 2)), g.abs().sum((0, 2)), mean, var * count / max(count - 1, 1)


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("shape,slope", [((2, 8, 6, 10), 0.01), ((1, 3, 33), 0.0), ((2, 16, 4, 8, 8), 0.01), ((6, 8, 100, 100), 0.01), ((1, 64, 6, 16, 20), 1.0), ((3, 5, 8193), 0.01),
                                         ((2, 1, 4), 0.01), ((4, 2, 1), 0.01), ((1, 2, 8192 + 64), 0.01)])
def test_abn8_against_float64(dev, shape, slope, inplace):
    g = torch.Generator().manual_seed(sum(shape))
    C = shape[1]
    cls = M.InPlaceABN if inplace else M.ABN
    norm, plain = cls(C, activation_param=slope).to(dev), cls(C, activation_param=slope).to(dev)
    x = torch.randn(shape, generator=g) * 1.5 + torch.randn((1, C) + (1,) * (len(shape) - 2), generator=g)
    gy, w, b = torch.randn(shape, generator=g), torch.randn(C, generator=g) * 0.6, torch.randn(C, generator=g) * 0.3
    for m in (norm, plain):
        with torch.no_grad():
            m.weight.copy_(w)
            m.bias.copy_(b)
    y, gx, gw, gb, terms, aw, ab, mean, unbiased = abn8_reference(x, w, b, gy, slope, 1e-5, inplace)
    xd, xp = x.to(dev).requires_grad_(), x.to(dev).requires_grad_()
    got, same = T.abn_train(norm, xd, checkpoint="8bit"), T.abn_train(plain, xp)
    # y = fma(x, scale, shift) with scale and shift rounded to float32 once each, the slope once; the f32 mode's statistics are float32 sums of 64 on the way
    r = 1 / torch.sqrt(x.double().transpose(0, 1).flatten(1).var(1, unbiased=False) + 1e-5)
    scale = ((w.abs() + 1e-5 if inplace else w).double() * r).abs().view(1, C, 1)
    size = x.double().abs().reshape(y.shape) * scale + mean.abs().view(1, C, 1) * scale + b.double().abs().view(1, C, 1)
    within(got.reshape(y.shape), y, 6 * U * size)
    within(got.reshape(y.shape), same.reshape(y.shape), 128 * U * size)
    got.backward(gy.to(dev))
    within(xd.grad.reshape(gx.shape), gx, rounding(gx, F32) + 16 * U * terms)
    within(norm.weight.grad, gw, 64 * U * aw + rounding(gw, F32) + 1e-12)
    within(norm.bias.grad, gb, 64 * U * ab + rounding(gb, F32))
    within(norm.running_mean, 0.1 * mean, 1e-6 * (1 + mean.abs()))
    # what the convolution behind rebuilds of y: one step of xhat times gamma away at most
    again = rebuilt(got)
    gamma = (w.abs() + 1e-5) if inplace else w
    N = shape[0]
    h = (x.double().reshape(N, C, -1) - mean.view(1, C, 1)) / torch.sqrt(x.double().reshape(N, C, -1).var((0, 2), unbiased=False) + 1e-5).view(1, C, 1)
    _, step = held(h.reshape(N * C, -1))
    within(again.reshape(N, C, -1), y, step.view(N, C, -1) * gamma.abs().double().view(1, C, 1) + 1e-5 * (1 + y.abs()))


def test_abn8_keeps_less_and_carries_non_finite_input(dev):
    x = torch.randn(2, 8, 32, 64, 64, device=dev, requires_grad=True)
    norm = M.ABN(8).to(dev)

    def kept(mode):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = T.abn_train(norm, x, checkpoint=mode)
        held_bytes = torch.cuda.memory_allocated() - before - y.numel() * 4
        del y
        return held_bytes
    # beyond y, which the caller holds here: 8 + 1 + 8 / 32 bits per element (33 + 4 bytes per 32) and per-channel vectors
    assert kept("8bit") <= x.numel() * 37 / 32 + (1 << 16)
    bad = x.detach().clone()
    bad[1, 3, 0, 0, 0] = float("nan")
    bad.requires_grad_()
    y = T.abn_train(norm, bad, checkpoint="8bit")
    y.backward(torch.ones_like(y))
    assert bool(torch.isnan(bad.grad[:, 3]).all()) and bool(torch.isfinite(bad.grad[:, :3]).all()) and bool(torch.isfinite(bad.grad[:, 4:]).all())


@pytest.mark.parametrize("source", ["abn", "abn written to", "layer norm", "plain layer norm", "layer norm written to", "sum", "leaf"])
def test_conv8_takes_its_weight_gradient_at_the_checkpoint(dev, source):
    g = torch.Generator().manual_seed(7)
    w = (torch.randn(16, 8, 3, 3, 3, generator=g) * 0.2).to(dev).requires_grad_()
    base = torch.randn(2, 8, 8, 12, 16, generator=g).to(dev).requires_grad_()
    norm = M.ABN(8).to(dev)
    if source.startswith("abn"):
        x = T.abn_train(norm, base, checkpoint="8bit")
        if source == "abn written to":
            x.mul_(1.5)
            want_x = ops.unpack8(ops.pack8(x.detach()))
        else:
            want_x = rebuilt(x)
            assert not torch.equal(want_x, ops.unpack8(ops.pack8(x.detach())))   # its own, not a new one
    elif "layer norm" in source:
        x = T.abn_train(M.LayerNormAct(8, affine=not source.startswith("plain")).to(dev), base, checkpoint="8bit")
        if source.endswith("written to"):
            x.add_(0.5)
        want_x = ops.unpack8(ops.pack8(x.detach())) if source.endswith("written to") else x   # formed again exactly
    elif source == "sum":
        x = base + 1.0
        want_x = ops.unpack8(ops.pack8(x.detach()))
    else:
        base.requires_grad_(False)
        x = want_x = base
    y = T.conv(x, w, None, ops.CONV_S2, checkpoint="8bit")
    assert torch.equal(y, T.conv(x, w, None, ops.CONV_S2))
    gy = torch.randn(y.shape, generator=g).to(dev)
    y.backward(gy)
    assert torch.equal(w.grad, T.conv_wgrad(ops.CONV_S2, want_x.detach(), gy, tuple(w.shape)))
    if source != "leaf":
        assert bool(torch.isfinite(base.grad).all())


# ---- cross entropy over depth hypotheses ------------------------------------------------------------------------------------------------------------
def ce_reference(cost, values, gt, mask):
    cost, values, gt = cost.double(), values.double(), gt.double()
    if values.dim() == 2:
        values = values[:, :, None, None].expand_as(cost)
    far = (values - gt.unsqueeze(1)).abs()
    k = torch.arange(cost.shape[1]).view(1, -1, 1, 1)
    at = torch.where(far == far.amin(1, keepdim=True), k, cost.shape[1]).amin(1)   # the lowest index of the smallest distance
    counted = (gt >= values.amin(1)) & (gt <= values.amax(1)) & (cost.amax(1) != -math.inf)
    if mask is not None:
        counted &= mask
    count = int(counted.sum())
    safe = torch.where(counted.unsqueeze(1), cost, 0.0)
    lse = torch.logsumexp(safe, 1)
    each = lse - safe.gather(1, at.unsqueeze(1)).squeeze(1)
    loss = each[counted].sum() / max(count, 1)
    p = torch.exp(safe - lse.unsqueeze(1))
    grad = torch.where(counted.unsqueeze(1), (p - (k == at.unsqueeze(1)).double()) / max(count, 1), 0.0)
    size = (each.abs() + safe.amax(1).abs() + 1)[counted].sum() / max(count, 1)
    return loss, grad, count, p, float(size), (k == at.unsqueeze(1)).double()


def ce_check(dev, cost, values, gt, mask, scale=1.0):
    loss, grad, count, p, size, hot = ce_reference(cost, values, gt, mask)
    c = cost.to(dev).requires_grad_()
    got = A.depth_cross_entropy(c, values.to(dev), gt.to(dev), None if mask is None else mask.to(dev))
    assert got.dtype == F32 and got.dim() == 0
    (got * scale).backward()
    grad = grad * scale
    if math.isinf(float(loss)):
        assert float(got) == float(loss)
    else:
        # exp and log within 2 half steps, D terms of the running sum, one subtraction
        within(got, loss, U * size * (8 + cost.shape[1]))
    # the exponential's argument is rounded once (at most 2^-24 of the largest difference), then 1 / s, the product and the share.  The 1 of the class is a term of
    # its own: grad = (p - 1) * (share * gloss) with share = fl(1 / count) passes four roundings (share, share * gloss, the difference, the product), each of at
    # most 2^-24 of |p - 1| / count <= 1 / count, also where p itself is next to nothing
    spread = float((cost.double().clamp(min=-100).amax() - cost.double().clamp(min=-100).amin()).clamp(max=100))
    within(c.grad, grad, rounding(grad, cost.dtype) + U * scale * ((16 + cost.shape[1] + spread) * (p + 1e-30) + 4 * hot) / max(count, 1))


def ce_inputs(B, D, h, w, per_pixel, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    cost = (torch.randn((B, D, h, w), generator=g) * spread).to(dtype)
    first = 400 + 50 * torch.rand((B, h, w) if per_pixel else (B,), generator=g)
    k = torch.arange(D, dtype=F32)
    values = first[:, None] + 2.65 * (k.view(1, D, 1, 1) if per_pixel else k)
    base = first if per_pixel else first[:, None, None]
    gt = base + 2.65 * (torch.rand((B, h, w), generator=g) * (D + 1.0) - 1.0)
    return cost, values, gt, torch.rand((B, h, w), generator=g) < 0.7


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("per_pixel", [True, False])
@pytest.mark.parametrize("B,D,h,w", [(1, 1, 4, 5), (2, 2, 3, 3), (2, 8, 16, 20), (1, 32, 9, 13), (3, 48, 7, 31), (1, 7, 1, 1), (1, 192, 12, 11), (1, 513, 5, 8), (2, 33, 40, 64)])
def test_depth_cross_entropy_against_float64(dev, B, D, h, w, per_pixel, dtype):
    cost, values, gt, mask = ce_inputs(B, D, h, w, per_pixel, dtype, B + D + h + w)
    ce_check(dev, cost, values, gt, mask, scale=3.0)
    ce_check(dev, cost, values, gt, None)


def test_depth_cross_entropy_edges(dev):
    cost, values, gt, mask = ce_inputs(1, 8, 6, 6, True, F32, 1)
    gt = values[:, 3] + 0.5 * (values[:, 4] - values[:, 3])   # (about) between two planes
    values = torch.round(values)   # whole numbers: exact ties
    gt = torch.round(gt) + 0.5
    ce_check(dev, cost, values, gt, None)
    # nothing counts: loss and gradient 0, whatever the costs hold
    wild = torch.full_like(cost, float("nan"))
    for m, t in ((torch.zeros_like(mask), gt), (None, torch.full_like(gt, 1e9)), (None, torch.full_like(gt, float("nan")))):
        c = wild.to(dev).requires_grad_()
        loss = A.depth_cross_entropy(c, values.to(dev), t.to(dev), None if m is None else m.to(dev))
        loss.backward()
        assert float(loss.detach()) == 0.0 and not c.grad.any()
    # -inf and the type's lowest value mask hypotheses out; a pixel with nothing left does not count
    for low in (-math.inf, torch.finfo(F32).min):
        c = cost.clone()
        c[0, ::2, 2] = low
        c[0, 1:, 3, 3] = low
        ce_check(dev, c, values, values[:, 1].contiguous(), None)
    c = cost.clone()
    c[0, :, 4, 4] = -math.inf
    ce_check(dev, c, values, values[:, 1].contiguous(), None)
    c[0, 0, 1, 1] = -math.inf   # the class itself is masked out: an infinite loss, finite gradients elsewhere
    t = values[:, 1].clone()
    t[0, 1, 1] = values[0, 0, 1, 1]
    loss, grad, *_ = ce_reference(c, values, t, None)
    cd = c.to(dev).requires_grad_()
    got = A.depth_cross_entropy(cd, values.to(dev), t.to(dev))
    got.backward()
    assert float(got) == math.inf and bool(torch.isfinite(cd.grad).all())
    # a NaN or +inf cost shows, at its pixel
    for bad in (math.nan, math.inf):
        c = cost.clone()
        c[0, 2, 5, 1] = bad
        cd = c.to(dev).requires_grad_()
        got = A.depth_cross_entropy(cd, values.to(dev), values[:, 1].contiguous().to(dev))
        got.backward()
        assert math.isnan(float(got)) and bool(torch.isnan(cd.grad[0, :, 5, 1]).any()) and int(torch.isnan(cd.grad).any(1).sum()) == 1
    # costs far from zero: the maximum and the sum are kept apart
    big = (cost * 1000).round() / 1000 + 4096.0
    ce_check(dev, big, values, gt, None)
    # descending hypotheses and a strided volume
    ce_check(dev, cost, values.flip(1), gt, mask)
    wide = torch.randn(1, 8, 6, 12)
    c1, c2 = (wide.to(dev)[:, :, :, ::2], wide[:, :, :, ::2].contiguous().to(dev))
    assert torch.equal(A.depth_cross_entropy(c1, values.to(dev), gt.to(dev)), A.depth_cross_entropy(c2, values.to(dev), gt.to(dev)))


def test_depth_cross_entropy_gradient_against_differences(dev):
    cost, values, gt, mask = ce_inputs(1, 6, 3, 4, True, F32, 3)
    c = cost.to(dev).requires_grad_()
    A.depth_cross_entropy(c, values.to(dev), gt.to(dev), mask.to(dev)).backward()
    for i in range(0, cost.numel(), 3):
        ends = []
        for sign in (1, -1):
            moved = cost.double().clone()
            moved.view(-1)[i] += sign * 1e-5
            ends.append(float(ce_reference(moved, values, gt, mask)[0]))
        assert abs((ends[0] - ends[1]) / 2e-5 - float(c.grad.flatten()[i])) < 2e-6


def test_depth_cross_entropy_refuses_what_does_not_fit(dev):
    cost, values, gt, mask = (t.to(dev) for t in ce_inputs(1, 4, 3, 4, True, F32, 3))
    for args, error, text in (((cost[0], values, gt), ValueError, "expected"), ((cost, values[:, :3], gt), ValueError, "depth_values"), ((cost, values, gt[:, :2]), ValueError, "depth_gt"),
                              ((cost, values, gt, mask.float()), ValueError, "mask"), ((cost.double(), values, gt), TypeError, "float64"), ((cost, values.half(), gt), TypeError, "float32"),
                              ((cost[:, :0], values[:, :0], gt), ValueError, "no hypotheses"), ((cost, values.cpu(), gt), RuntimeError, "no CPU fallback")):
        with pytest.raises(error, match=text):
            A.depth_cross_entropy(*args)


# ---- streams, graphs, order, size -------------------------------------------------------------------------------------------------------------------
def _calls(dev):
    g = torch.Generator().manual_seed(8)
    x, w, b = torch.randn(2, 8, 40, 36, generator=g).to(dev), torch.rand(8, generator=g).to(dev), torch.randn(8, generator=g).to(dev)
    rows, gy = torch.randn(100, 96, generator=g).to(dev), torch.randn(2, 8, 40, 36, generator=g).to(dev)
    cost, values, gt, mask = (t.to(dev) for t in ce_inputs(2, 16, 20, 24, True, F32, 9))

    def layer_norm():
        return (ops.layer_norm(x, w, b, slope=0.01), ops.layer_norm(rows, channels_last=True), *ops.layer_norm_backward(x, gy, w, b, slope=0.01),
                *ops.layer_norm_backward(rows, rows, channels_last=True))

    def pack():
        p = ops.pack8(x)
        return p.codes, p.scales, ops.unpack8(p)

    norm = M.ABN(8).to(dev)
    norm.running_mean = norm.running_var = None   # (they would differ from call to call)

    def abn():
        xr = x.detach().requires_grad_()
        y = T.abn_train(norm, xr, checkpoint="8bit")
        return (y.detach(), rebuilt(y), *torch.autograd.grad(y, (xr, norm.weight, norm.bias), gy))

    def ce():
        c = cost.detach().requires_grad_()
        loss = A.depth_cross_entropy(c, values, gt, mask)
        return loss.detach(), torch.autograd.grad(loss, c)[0]
    return {"layer_norm": layer_norm, "pack8": pack, "abn8": abn, "depth_ce": ce}


@pytest.mark.parametrize("name", ["layer_norm", "pack8", "abn8", "depth_ce"])
def test_the_same_bits_again_on_another_stream_and_in_a_graph(dev, name):
    call = _calls(dev)[name]
    want = [t.clone() for t in call()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = call()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    with torch.cuda.stream(side):   # warm up where the capture runs
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = call()
    for _ in range(4):
        for t in captured:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(captured, want))
        assert all(torch.equal(p, q) for p, q in zip(call(), want))   # eager work between the replays


def test_two_threads_at_once(dev):
    """Every operator from two host threads, each on a stream of its own, over and over: the same bits as alone."""
    import threading
    calls = [_calls(dev) for _ in range(2)]   # (their norms and inputs apart)
    want = {name: [t.clone() for t in call()] for name, call in calls[0].items()}
    torch.cuda.synchronize()
    wrong = []

    def work(mine):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                for name, call in mine.items():
                    got = call()
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(p, q) for p, q in zip(got, want[name])):
                        wrong.append(name)
    threads = [threading.Thread(target=work, args=(mine,)) for mine in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


def test_gradients_add_up_over_calls_and_have_no_second_derivative(dev):
    g = torch.Generator().manual_seed(17)
    x = torch.randn(2, 8, 6, 10, generator=g).to(dev).requires_grad_()
    cost, values, gt, mask = (t.to(dev) for t in ce_inputs(1, 8, 6, 10, True, F32, 5))
    cost.requires_grad_()
    for norm, checkpoint in ((M.LayerNormAct(8), "f32"), (M.ABN(8), "8bit"), (None, None)):
        if norm is None:
            leaves, out = [cost], lambda: A.depth_cross_entropy(cost, values, gt, mask)
        else:
            norm = norm.to(dev).train()
            leaves, out = [x, norm.weight, norm.bias], lambda: (T.abn_train(norm, x, checkpoint) ** 2).sum()
        for t in leaves:
            t.grad = None
        out().backward()
        once = [t.grad.clone() for t in leaves]
        out().backward()   # into the gradients that are there
        assert all(torch.equal(t.grad, 2 * p) for t, p in zip(leaves, once))
        torch.nn.utils.clip_grad_norm_(leaves, 1e-3)   # writes them in place
        for t in leaves:
            t.grad.zero_()
        first = torch.autograd.grad(out(), leaves[0], create_graph=True)[0]
        assert torch.equal(first.detach(), once[0])
        # (torch's own words for it: the gradient is cut off from the leaf, or from everything where grad_output is a constant)
        with pytest.raises(RuntimeError, match="to not have been used in the graph|does not require grad"):
            torch.autograd.grad(first.sum(), leaves[0])


def test_offsets_beyond_32_bits(dev):
    """More elements than 2^32: the last positions and blocks come out as on their own."""
    n = (1 << 29) + 40
    x = torch.empty((1, 8, n), dtype=BF16, device=dev)
    x.view(8, n)[:] = torch.randn(8, 1, device=dev)
    tail = torch.randn(1, 8, 64, device=dev).to(BF16)
    x[:, :, -64:] = tail
    y = ops.layer_norm(x, slope=0.01)
    assert torch.equal(y[:, :, -64:], ops.layer_norm(tail, slope=0.01)) and torch.equal(y[:, :, 5], y[:, :, 1 << 28])
    gx, gw, gb = ops.layer_norm_backward(x, y, slope=0.01)
    assert torch.equal(gx[:, :, -64:], ops.layer_norm_backward(tail, y[:, :, -64:].contiguous(), slope=0.01)[0])
    del y, gx
    p = ops.pack8(x)
    held_tail = ops.unpack8(ops.pack8(x[:, :, -72:]))   # blocks start at multiples of 32 of the plane: n - 72 is one
    assert (n - 72) % 32 == 0 and torch.equal(ops.unpack8(p)[:, :, -72:], held_tail)


# ---- together ------------------------------------------------------------------------------------------------------------------------------------------
def _step(dev, norm_act, mode, loss, seed=0, size=(64, 96), B=1):
    from casmvsnet_pl_amd.synthetic import make_inputs, randomize_state_dict
    model = M.CascadeMVSNet(num_groups=1, norm_act=norm_act)
    randomize_state_dict(model.state_dict(), seed=seed)
    model = model.to(dev).train()
    model.checkpoint_mode, model.return_cost = mode, loss == "cross_entropy"
    imgs, proj, dmin, dint = make_inputs(B, 3, *size, seed=seed)
    res = model(imgs.to(dev), proj.to(dev), dmin, dint)
    g = torch.Generator().manual_seed(seed)
    depths = {f"level_{l}": (dmin + 100 * torch.rand((B, size[0] >> l, size[1] >> l), generator=g)).to(dev) for l in range(3)}
    masks = {f"level_{l}": (torch.rand((B, size[0] >> l, size[1] >> l), generator=g) < 0.8).to(dev) for l in range(3)}
    value = (T.cross_entropy_loss if loss == "cross_entropy" else T.sl1_loss)(res, depths, masks)
    value.backward()
    T.release_plan()
    return model, res, value.detach(), {k: p.grad for k, p in model.named_parameters()}


@pytest.mark.parametrize("norm_act", [M.ABN, M.InPlaceABN, M.LayerNormAct])
def test_training_step_with_8_bit_checkpoints(dev, norm_act):
    """The same forward to float32's rounding; gradients near the float32 ones: within a few percent of their size."""
    _, res, value, want = _step(dev, norm_act, "f32", "sl1")
    _, res8, value8, got = _step(dev, norm_act, "8bit", "sl1")
    assert all(float((res[f"depth_{l}"] - res8[f"depth_{l}"]).abs().max()) < 1e-3 * float(res[f"depth_{l}"].abs().max()) for l in range(3))
    assert abs(float(value) - float(value8)) < 1e-3 * float(value)
    _, _, _, again = _step(dev, norm_act, "8bit", "sl1")
    assert all(torch.equal(got[k], again[k]) for k in got)   # bit-reproducible
    a = torch.cat([want[k].flatten() for k in sorted(want)]).double()
    b = torch.cat([got[k].flatten() for k in sorted(want)]).double()
    assert bool(torch.isfinite(b).all()) and float((a - b).norm() / a.norm()) < 0.05


@pytest.mark.parametrize("mode", ["f32", "8bit"])
@pytest.mark.parametrize("norm_act", [M.ABN, M.LayerNormAct])
def test_training_step_with_the_cross_entropy_loss(dev, norm_act, mode):
    model, res, value, grads = _step(dev, norm_act, mode, "cross_entropy")
    assert len(grads) == 130 and all(g is not None and bool(torch.isfinite(g).all()) for g in grads.values()) and math.isfinite(float(value)) and float(value) > 0
    assert res["cost_0"].shape == res["depth_values_0"].shape == (1, 8, 64, 96)


@pytest.mark.parametrize("loss", ["sl1", "cross_entropy"])
def test_train_steps_with_either_loss(dev, loss):
    """The training loop's first loss is the step's; the model's switches are as they were afterwards."""
    from casmvsnet_pl_amd.synthetic import make_inputs
    model, _, value, _ = _step(dev, M.LayerNormAct, "8bit", loss)
    model.return_cost = False
    imgs, proj, dmin, dint = make_inputs(1, 3, 64, 96, seed=0)
    g = torch.Generator().manual_seed(0)
    depths = {f"level_{l}": dmin + 100 * torch.rand((64 >> l, 96 >> l), generator=g) for l in range(3)}
    masks = {f"level_{l}": torch.rand((64 >> l, 96 >> l), generator=g) < 0.8 for l in range(3)}
    batch = {"imgs": imgs, "proj_mats": proj, "init_depth_min": dmin, "depth_interval": dint, "depths": [depths], "masks": [masks]}
    before = [p.detach().clone() for p in model.parameters()]
    losses = T.train_steps(model, [batch] * 2, torch.optim.SGD(model.parameters(), lr=1e-4), dev, loss=loss)
    # (the same kernels on the same values in the same order; torch's own SmoothL1 mean may split its sum otherwise)
    assert abs(losses[0] - float(value)) <= 1e-6 * float(value) and len(losses) == 2 and losses[1] == losses[1]
    assert model.return_cost is False and any(not torch.equal(p, q) for p, q in zip(model.parameters(), before))


def test_layer_norm_model_in_train_mode_against_torch_on_the_cpu(dev):
    """LayerNormAct in the reference's layers: FeatureNet's and CostRegNet's forwards and weight gradients against torch autograd in float64."""
    import torch.nn.functional as F
    g = torch.Generator().manual_seed(11)
    net = M.CostRegNet(8, M.LayerNormAct)
    for p in net.parameters():
        p.data = torch.randn(p.shape, generator=g) * (0.2 if p.dim() > 1 else 0.3) + (1.0 if p.dim() == 1 else 0.0)
    x = torch.randn((1, 8, 8, 16, 24), generator=g)
    sd = {k: v.detach().double().requires_grad_() for k, v in net.state_dict().items()}

    def ln(z, name):
        w, b = sd[name + ".weight"], sd[name + ".bias"]
        return F.leaky_relu(F.layer_norm(z.movedim(1, -1), (z.shape[1],), w, b, 1e-5).movedim(-1, 1), 0.01)

    def layer(z, name, stride=1):
        return ln(F.conv3d(z, sd[name + ".conv.weight"], None, stride, 1), name + ".bn")

    def up(z, name):
        return ln(F.conv_transpose3d(z, sd[name + ".0.weight"], None, 2, 1, 1), name + ".1")
    xr = x.double()
    c0 = layer(xr, "conv0")
    c2 = layer(layer(c0, "conv1", 2), "conv2")
    c4 = layer(layer(c2, "conv3", 2), "conv4")
    z = layer(layer(c4, "conv5", 2), "conv6")
    z = c4 + up(z, "conv7")
    z = c2 + up(z, "conv9")
    z = c0 + up(z, "conv11")
    want = F.conv3d(z, sd["prob.weight"], sd["prob.bias"], 1, 1)
    gy = torch.randn(want.shape, generator=g)
    want.backward(gy.double())
    net = net.to(dev).train()
    got = net(x.to(dev))
    got.backward(gy.to(dev))
    scale = lambda a, b: float((a.detach().double().cpu() - b.detach()).abs().max() / b.detach().abs().max())
    # ten float32 convolutions in a row (each within 3e-5 of its range, see the convolution tests)
    assert scale(got, want) < 3e-4
    for k, p in net.named_parameters():
        assert scale(p.grad, sd[k].grad) < 3e-3, k
    net.eval()
    with torch.no_grad():
        assert torch.equal(net(x.to(dev)), got)   # layer norm has no train / eval difference


def test_layer_norm_model_in_eval_mode(dev):
    from casmvsnet_pl_amd.synthetic import make_inputs, randomize_state_dict
    model = M.CascadeMVSNet(num_groups=1, norm_act=M.LayerNormAct)
    randomize_state_dict(model.state_dict(), seed=1)
    model = model.to(dev)
    imgs, proj, dmin, dint = make_inputs(1, 3, 64, 96, seed=1)
    imgs, proj = imgs.to(dev), proj.to(dev)
    model.train()
    want = model(imgs, proj, dmin, dint)
    T.release_plan()
    model.eval()
    got = model(imgs, proj, dmin, dint)
    assert set(got) == {f"{k}_{l}" for k in ("depth", "confidence") for l in range(3)} and not any(v.requires_grad for v in got.values())
    for l in range(3):   # (train mode runs the same layers; the regression is the same kernel)
        assert float((got[f"depth_{l}"] - want[f"depth_{l}"]).abs().max()) <= 1e-3 * float(want[f"depth_{l}"].abs().max())
    layer = model.feature.conv0[0]
    assert not layer(imgs[0]).requires_grad


def test_layer_norm_model_follows_its_weights_in_a_captured_forward(dev):
    """GraphedForward of a layer-norm model: its replays equal the eager forward, before and after a training step has changed the weights."""
    from casmvsnet_pl_amd.graph import GraphedForward
    from casmvsnet_pl_amd.synthetic import make_inputs
    model, *_ = _step(dev, M.LayerNormAct, "8bit", "sl1")   # (its PackPlan is warm)
    model.eval()
    imgs, proj, dmin, dint = make_inputs(1, 3, 64, 96, seed=5)
    imgs, proj = imgs.to(dev), proj.to(dev)
    graphed = GraphedForward(model, imgs, proj, dmin, dint)
    for round_ in range(3):
        want = {k: v.clone() for k, v in model(imgs, proj, dmin, dint).items()}
        got = graphed(imgs, proj)
        torch.cuda.synchronize()
        assert all(torch.equal(got[k], want[k]) for k in want), round_
        with torch.no_grad():
            for p in model.parameters():
                p.mul_(1.01)


def test_a_training_step_of_all_of_them_in_a_graph(dev):
    """Layer norm, 8-bit checkpoints and the cross entropy in one captured step (forward, loss, backward to the parameters' gradients): every replay equals eager."""
    g = torch.Generator().manual_seed(12)
    x = torch.randn(2, 8, 8, 16, 24, generator=g).to(dev)
    values = (400 + 2.65 * torch.arange(8, dtype=F32).view(1, 8, 1, 1) + torch.rand(2, 1, 16, 24, generator=g)).expand(2, 8, 16, 24).contiguous().to(dev)
    gt, mask = (values[:, 3] + 1.0).contiguous(), (torch.rand(2, 16, 24, generator=g) < 0.7).to(dev)
    for norm_act in (M.LayerNormAct, M.ABN):
        torch.manual_seed(3)
        net = M.CostRegNet(8, norm_act).to(dev).train()
        for m in net.modules():
            if hasattr(m, "running_mean"):
                m.running_mean = m.running_var = None
        params = list(net.parameters())

        def step():
            cost = T.cost_reg_net_train(net, x, "8bit").squeeze(1)
            loss = A.depth_cross_entropy(cost, values, gt, mask)
            return (loss.detach(), *torch.autograd.grad(loss, params))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = [t.clone() for t in step()]
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = step()
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(captured, want))
            assert all(torch.equal(p, q) for p, q in zip(step(), want))
