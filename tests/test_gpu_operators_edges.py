"""GPU tests of the training-side operators at the edge of what their entry points allow: layer norm without an eps,
8-bit ABN far from zero, what is kept across writes, under other grad modes and in memory, captured forwards, mixed norms.  Definitions, bounds and fixtures are
test_gpu_operators.py's."""
import math

import pytest
import torch

import casmvsnet_pl_amd as M
from casmvsnet_pl_amd import ops
from casmvsnet_pl_amd import training as T

from test_gpu_operators import BF16, F16, F32, U, _step, abn8_reference, dev, ln_check, rounding, within   # noqa: F401  (dev is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape,rows", [((2, 8, 65), False), ((2, 8, 1000), False), ((1, 16, 52), False), ((2, 32, 12), False), ((2, 64, 1921), False), ((1, 20, 100), False),
                                        ((1, 3, 100), False), ((1, 100, 17), False), ((1, 300, 40), False), ((2, 520, 3), False), ((1, 8, 1024), False), ((5, 20), True),
                                        ((7, 5), True), ((3, 300), True), ((2, 2048), True)])
def test_layer_norm_without_an_eps(dev, shape, rows, dtype):   # noqa: F811
    """eps = 0: a thread without a position has no spread to divide by; nothing of it reaches the weight gradient."""
    g = torch.Generator().manual_seed(sum(shape))
    C = shape[-1] if rows else shape[1]
    x = (torch.randn(shape, generator=g) * 1.7 + 0.6).to(dtype)
    ln_check(dev, x, torch.rand(C, generator=g) + 0.5, torch.randn(C, generator=g) * 0.3, torch.randn(shape, generator=g).to(dtype), eps=0.0, channels_last=rows)


@pytest.mark.parametrize("written", ["nothing", "source", "weight", "bias", "eps and slope", "another weight"])
def test_conv8_behind_a_layer_norm_whose_source_is_written_to(dev, written):   # noqa: F811
    """What the convolution forms its input from again are the tensors that the norm read: written to since, they no longer make it, and it packs its input instead."""
    g = torch.Generator().manual_seed(7)
    w = (torch.randn(16, 8, 3, 3, 3, generator=g) * 0.2).to(dev).requires_grad_()
    source = torch.randn(2, 8, 8, 12, 16, generator=g).to(dev).requires_grad_() * 1.0
    norm = M.LayerNormAct(8).to(dev)
    x = T.abn_train(norm, source, checkpoint="8bit")
    want_x = x.detach().clone()
    with torch.no_grad():
        if written == "source":
            source.mul_(source)
        elif written in ("weight", "bias"):
            getattr(norm, written).add_(0.5)
        elif written == "eps and slope":
            norm.eps, norm.activation_param = 0.5, 0.3
        elif written == "another weight":
            norm.weight = torch.nn.Parameter(norm.weight + 0.5)
    if written in ("source", "weight", "bias"):
        want_x = ops.unpack8(ops.pack8(want_x))
    y = T.conv(x, w, None, ops.CONV_S2, checkpoint="8bit")
    gy = torch.randn(y.shape, generator=g).to(dev)
    # (the norm's own backward pass, which would refuse what was written to, is not part of this gradient)
    assert torch.equal(torch.autograd.grad(y, w, gy)[0], T.conv_wgrad(ops.CONV_S2, want_x, gy, tuple(w.shape)))


def test_abn8_backward_allocates_its_gradients_only(dev):   # noqa: F811
    """No tensor as large as what was kept is made (and filled) on the way: the peak of the backward pass is grad_x, the two vectors and the workspace."""
    x = torch.randn(2, 8, 32, 64, 64, device=dev, requires_grad=True)
    norm, gy = M.ABN(8).to(dev), torch.randn(2, 8, 32, 64, 64, device=dev)
    y = T.abn_train(norm, x, checkpoint="8bit")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    torch.autograd.grad(y, (x, norm.weight, norm.bias), gy)
    # (8.4 MB of grad_x; 4.8 MB are kept, and the allocator rounds up to 2 MB)
    assert torch.cuda.max_memory_allocated() - before <= x.numel() * 4 + (1 << 21)


def test_abn8_without_a_gradient_of_its_output(dev):   # noqa: F811
    """A node behind that hands no gradient back: none arrives at the input either."""
    class Cut(torch.autograd.Function):
        @staticmethod
        def forward(ctx, t):
            return t * 1.0

        @staticmethod
        def backward(ctx, g):
            return None
    x = torch.randn(2, 8, 6, 10, device=dev, requires_grad=True)
    norm = M.ABN(8).to(dev)
    Cut.apply(T.abn_train(norm, x, checkpoint="8bit")).sum().backward()
    assert all(t.grad is None or not t.grad.any() for t in (x, norm.weight, norm.bias))


def test_abn8_graph_holds_8_bits_where_f32_holds_two_tensors(dev):   # noqa: F811
    """What the graph alone holds, its input and output dropped by everyone else."""
    base = torch.randn(2, 8, 32, 64, 64, device=dev, requires_grad=True)
    norm = M.ABN(8).to(dev)

    def kept(mode):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = T.abn_train(norm, base * 1.0, checkpoint=mode).sum()   # (neither the product with a number nor the sum keeps a tensor)
        return torch.cuda.memory_allocated() - before, out
    eight, _ = kept("8bit")
    two, _ = kept("f32")
    # (a block of the allocator's may be up to 1 MB larger than what was asked for; x and y in float32 are 16.8 MB, the 8 bits and their scales and signs 2.4)
    assert eight <= base.numel() * 37 / 32 + (1 << 20) and two >= base.numel() * 8


@pytest.mark.parametrize("norm_act,most", [(M.ABN, 0.5), (M.LayerNormAct, 0.75)])
def test_training_step_with_8_bit_checkpoints_peaks_lower(dev, norm_act, most):   # noqa: F811
    """(640x512: 0.36 of the float32 mode's peak with ABN, 0.64 with layer norm, which keeps its float32 input)"""
    def peak(mode):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        _step(dev, norm_act, mode, "sl1", size=(256, 320))
        return torch.cuda.max_memory_allocated() - before
    assert peak("8bit") < most * peak("f32")


@pytest.mark.parametrize("norm_act", [M.ABN, M.LayerNormAct])
def test_8_bit_mode_without_a_graph(dev, norm_act):   # noqa: F811
    """Under no_grad and inference_mode there is nothing to keep: the float32 mode's results, in train mode too."""
    net = M.CostRegNet(8, norm_act).to(dev).train()
    x = torch.randn(1, 8, 8, 16, 24, device=dev)
    want = T.cost_reg_net_train(net, x).detach()
    for without in (torch.no_grad, torch.inference_mode):
        with without():
            assert torch.equal(T.cost_reg_net_train(net, x, "8bit"), want)
    norm = norm_act(8).to(dev)
    with torch.no_grad():
        assert not hasattr(T.abn_train(norm, x, "8bit"), "_casmvs_made_by")


def test_abn8_of_many_channels_keeps_no_workspace(dev):   # noqa: F811
    base = torch.randn(1, 8192, 8, device=dev, requires_grad=True)
    norm = M.ABN(8192).to(dev)
    torch.cuda.synchronize()   # (everything below 1 MB: the allocator counts what was asked for, in steps of 512 bytes)
    before = torch.cuda.memory_allocated()
    out = T.abn_train(norm, base * 1.0, checkpoint="8bit").sum()
    # a block of 37 bytes and 16 bytes of vectors per channel; the forward pass's sums are another 16
    assert torch.cuda.memory_allocated() - before <= 8192 * (37 + 16) + 4096 and out.requires_grad


def test_layer_norm_model_refreshes_a_captured_forward(dev):   # noqa: F811
    """GraphedForward.refresh_weights after a weight update: nothing is folded ahead of a layer-norm model's replay, so there is nothing to pack again."""
    from casmvsnet_pl_amd.graph import ConcurrentForwards, GraphedForward
    from casmvsnet_pl_amd.synthetic import make_inputs, randomize_state_dict
    model = M.CascadeMVSNet(num_groups=1, norm_act=M.LayerNormAct)
    randomize_state_dict(model.state_dict(), seed=2)
    model = model.to(dev).eval()
    imgs, proj, dmin, dint = make_inputs(1, 3, 64, 96, seed=5)
    imgs, proj = imgs.to(dev), proj.to(dev)
    graphed, two = GraphedForward(model, imgs, proj, dmin, dint), ConcurrentForwards(model, imgs, proj, dmin, dint)
    with torch.no_grad():
        for p in model.parameters():
            p.mul_(1.01)
    graphed.refresh_weights()
    two.refresh_weights()
    want = {k: v.clone() for k, v in model(imgs, proj, dmin, dint).items()}
    for got in (graphed(imgs, proj), *two.run([(imgs, proj)] * 2)):
        torch.cuda.synchronize()
        assert all(torch.equal(got[k], want[k]) for k in want)


def test_norms_of_both_kinds_train_and_are_refused_in_eval_mode(dev):   # noqa: F811
    net = M.CostRegNet(8, lambda c: M.LayerNormAct(c) if c == 8 else M.ABN(c)).to(dev).train()
    x = torch.randn(1, 8, 8, 16, 24, device=dev)
    assert bool(torch.isfinite(net(x)).all())
    before = {k: v.clone() for k, v in net.state_dict().items()}
    with pytest.raises(RuntimeError, match="both"):
        net.eval()(x)
    assert all(torch.equal(v, before[k]) for k, v in net.state_dict().items())


@pytest.mark.parametrize("shape", [(2, 3, 70), (2, 8, 4, 16, 20), (1, 2, 8192 + 64), (3, 4, 40001)])
@pytest.mark.parametrize("offset", [0.0, 1e4, -3e6])
def test_abn8_far_from_zero(dev, shape, offset):   # noqa: F811
    """Channels whose mean is many times their spread: y, the side of zero and the gradients as at zero; constant channels are their bias."""
    g = torch.Generator().manual_seed(sum(shape))
    C, count = shape[1], math.prod(shape) // shape[1]
    norm = M.ABN(C).to(dev)
    x, gy = torch.randn(shape, generator=g) * 1.5 + offset, torch.randn(shape, generator=g)
    w, b = torch.randn(C, generator=g) * 0.6, torch.randn(C, generator=g) * 0.3
    with torch.no_grad():
        norm.weight.copy_(w)
        norm.bias.copy_(b)
    y, gx, gw, gb, terms, aw, ab, mean, unbiased = abn8_reference(x, w, b, gy, 0.01, 1e-5, False)
    xd = x.to(dev).requires_grad_()
    got = T.abn_train(norm, xd, checkpoint="8bit")
    # z in 64 bits: the mean is off by a rounding of its own size (8 of them: the reference's too), the variance by less than count of them.  y in float32 from x - mean,
    # the mean as two floats: both differences, the scale and the product half a step each of |h w|, the sum and the slope of |z|
    r = (1 / torch.sqrt(unbiased * (count - 1) / count + 1e-5)).view(1, C, 1)
    far = mean.abs().view(1, C, 1) * r * w.double().abs().view(1, C, 1)
    z = torch.where(y > 0, y, y / float(torch.tensor(0.01)))
    hw = (z - b.double().view(1, C, 1)).abs()
    z_off = 2.0 ** -53 * (8 * far + 4 * count * hw) + 1e-12 * (hw + 1)
    within(got.reshape(y.shape), y, torch.where(y > 0, 1.0, 0.01) * (U * 1.001 * (4 * hw + 2 * z.abs()) + 2 * U * U * far + z_off))
    got.backward(gy.to(dev))
    within(xd.grad.reshape(gx.shape), gx, rounding(gx, F32) + 16 * U * terms)
    within(norm.weight.grad, gw, 64 * U * aw + rounding(gw, F32))
    within(norm.bias.grad, gb, 64 * U * ab + rounding(gb, F32))
    within(norm.running_mean, 0.1 * mean, 4 * U * 0.1 * mean.abs() + 1e-12)
    within(norm.running_var, 0.9 + 0.1 * unbiased, 4 * U * (0.9 + 0.1 * unbiased))
    flat = T.abn_train(norm, torch.full(shape, offset, device=dev, requires_grad=True), checkpoint="8bit")
    assert torch.equal(flat, torch.where(norm.bias > 0, norm.bias, norm.bias * 0.01).view(1, C, *[1] * (len(shape) - 2)).expand(shape))


@pytest.mark.parametrize("first", [float("nan"), float("inf"), 1e6])
def test_abn8_whatever_the_first_element_is(dev, first):   # noqa: F811
    """A channel's sums are taken about its first element: far from all others it costs no digits, not finite it makes the channel NaN and no other."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 4, 9, 21, generator=g)
    x[0, 2, 0, 0] = first
    norm = M.ABN(4).to(dev)
    xd = x.to(dev).requires_grad_()
    y = T.abn_train(norm, xd, checkpoint="8bit")
    y.backward(torch.ones_like(y))
    if abs(first) < float("inf"):
        want, _, _, _, _, _, _, mean, unbiased = abn8_reference(x, torch.ones(4), torch.zeros(4), torch.ones_like(x), 0.01, 1e-5, False)
        within(y.reshape(want.shape), want, 6 * U * want.abs() * 1.001 + 2 * U * U * mean.abs().view(1, 4, 1) + 1e-10)   # (as above, without a bias)
        within(norm.running_var, 0.9 + 0.1 * unbiased, 4 * U * (0.9 + 0.1 * unbiased))
    else:
        assert bool(torch.isnan(y[:, 2]).all()) and bool(torch.isnan(xd.grad[:, 2]).all())
        others = [0, 1, 3]
        assert bool(torch.isfinite(y[:, others]).all()) and bool(torch.isfinite(xd.grad[:, others]).all())


@pytest.mark.parametrize("shape", [(2, 8, 6, 10), (3, 5, 40001)])
def test_abn8_gradients_of_the_affine_alone(dev, shape):   # noqa: F811
    """An input that no gradient goes to: the two vectors are those of the whole backward pass."""
    g = torch.Generator().manual_seed(4)
    x, gy = torch.randn(shape, generator=g).to(dev), torch.randn(shape, generator=g).to(dev)
    norm = M.InPlaceABN(shape[1]).to(dev)
    xr = x.clone().requires_grad_()
    _, *want = torch.autograd.grad(T.abn_train(norm, xr, checkpoint="8bit"), (xr, norm.weight, norm.bias), gy)
    got = torch.autograd.grad(T.abn_train(norm, x, checkpoint="8bit"), (norm.weight, norm.bias), gy)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_train_steps_of_a_wrapped_model_with_the_cross_entropy_loss(dev):   # noqa: F811
    """The switch is the model's, not its data-parallel wrapper's: the same losses either way, and the switch as it was afterwards."""
    from casmvsnet_pl_amd.synthetic import make_inputs, randomize_state_dict
    imgs, proj, dmin, dint = make_inputs(1, 3, 64, 96, seed=0)
    g = torch.Generator().manual_seed(0)
    depths = {f"level_{l}": dmin + 100 * torch.rand((64 >> l, 96 >> l), generator=g) for l in range(3)}
    masks = {f"level_{l}": torch.rand((64 >> l, 96 >> l), generator=g) < 0.8 for l in range(3)}
    batch = {"imgs": imgs, "proj_mats": proj, "init_depth_min": dmin, "depth_interval": dint, "depths": [depths], "masks": [masks]}
    losses = []
    for wrap in (lambda m: m, lambda m: torch.nn.DataParallel(m, device_ids=[0])):
        model = M.CascadeMVSNet(num_groups=1, norm_act=M.LayerNormAct)
        randomize_state_dict(model.state_dict(), seed=0)
        wrapped = wrap(model.to(dev))
        losses.append(T.train_steps(wrapped, [batch], torch.optim.SGD(model.parameters(), lr=1e-4), dev, loss="cross_entropy"))
        assert model.return_cost is False
    assert losses[0] == losses[1] and losses[0][0] > 0
