"""Training support, op by op: torch.autograd.Function wrappers whose forward AND backward are HIP
kernels of libcasmvs_hip.so.  `CascadeMVSNet.forward` itself stays the inference engine (eval-mode ABN folded into
the conv epilogues); these are the differentiable forms of the two ops of the hot path whose gradients are not plain
convolution gradients:

  homo_warp(src_feat, proj_mat, depth_values)      models/modules.py:52-92.  Gradient with respect to src_feat only:
      the sampling grid depends on proj_mat and on depth hypotheses that the reference detaches (mvsnet.py:231).
  softmax_depth_regression(cost, depth_values)     models/mvsnet.py:175-177 + modules.py:95-104: depth = sum_k
      softmax(cost)_k d_k, gradient with respect to the cost volume (the hypotheses are detached; the confidence is
      computed under torch.no_grad() in the reference, mvsnet.py:179-193, and is returned without a graph here).

A variance / correlation cost volume built from `homo_warp` outputs with torch's elementwise ops (the reference's own
training-mode code, mvsnet.py:150-153) is therefore differentiable end to end down to the feature maps.

Two more that a training step uses and the reference does not have:

  layer_norm(x, weight, bias, eps, slope, channels_last)     normalisation per position over the channels + leaky ReLU, in the place of
      batch statistics (norm.LayerNormAct is the module); gradients w.r.t. x, weight and bias.
  depth_cross_entropy(cost, depth_values, depth_gt, mask)    the depth as a classification over the hypotheses, the other loss beside
      SmoothL1 on softmax_depth_regression; gradient w.r.t. the cost volume.
"""
import ctypes
import functools

import torch

from . import _lib, ops


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr())


def _stream(t):
    from . import streams
    return streams.launch_stream(t)


class _HomoWarp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, src_feat, proj_mat, depth_values):
        ctx.save_for_backward(proj_mat, depth_values)
        ctx.src_shape = tuple(src_feat.shape)
        return ops.homo_warp(src_feat.detach(), proj_mat.detach(), depth_values.detach())

    @staticmethod
    def backward(ctx, grad_out):
        proj_mat, depth_values = ctx.saved_tensors
        B, C, H, W = ctx.src_shape
        D = depth_values.shape[1]
        grad_out = grad_out.contiguous().float()
        proj_mat, depth_values = proj_mat.contiguous().float(), depth_values.contiguous().float()
        grad_src = torch.empty((B, C, H, W), dtype=torch.float32, device=grad_out.device)
        # caller-owned scratch: the 64-bit fixed-point map of the order-independent scatter (same bits run to run) + the channels' largest magnitudes
        ws = torch.empty(_lib.load().casmvs_homo_warp_backward_workspace_bytes(B, C, D, H, W) // 8 + 1, dtype=torch.int64, device=grad_out.device)
        with torch.cuda.device(grad_out.device):
            rc = _lib.load().casmvs_homo_warp_backward_f32(_ptr(grad_out), _ptr(proj_mat), _ptr(depth_values), _ptr(grad_src), _ptr(ws),
                                                           B, C, H, W, D, _stream(grad_out))
        _lib.check(rc, "casmvs_homo_warp_backward_f32")
        return grad_src, None, None


class _SoftmaxDepthRegression(torch.autograd.Function):
    @staticmethod
    def forward(ctx, cost, depth_values):
        cost, depth_values = cost.detach().contiguous().float(), depth_values.detach().contiguous().float()
        ctx.save_for_backward(cost, depth_values)
        depth, confidence = ops.softmax_regress(cost, depth_values)
        ctx.mark_non_differentiable(confidence)
        return depth, confidence

    @staticmethod
    def backward(ctx, grad_depth, _grad_confidence):
        cost, depth_values = ctx.saved_tensors
        B, D, h, w = cost.shape
        grad_depth = grad_depth.contiguous().float()
        grad_cost = torch.empty_like(cost)
        with torch.cuda.device(cost.device):
            rc = _lib.load().casmvs_softmax_regress_backward_f32(_ptr(cost), _ptr(depth_values), _ptr(grad_depth), _ptr(grad_cost),
                                                                 B, D, h, w, _stream(cost))
        _lib.check(rc, "casmvs_softmax_regress_backward_f32")
        return grad_cost, None


def homo_warp(src_feat, proj_mat, depth_values):
    """Differentiable models/modules.py:52-92: (B,C,H,W), (B,3,4), (B,D,H,W) -> (B,C,D,H,W); d/d src_feat by HIP scatter-add."""
    if not src_feat.is_cuda:
        raise RuntimeError("casmvsnet_pl_amd.autograd.homo_warp runs on the MI355X only; there is no CPU fallback")
    return _HomoWarp.apply(src_feat, proj_mat, depth_values)


def softmax_depth_regression(cost, depth_values):
    """Differentiable models/mvsnet.py:175-193: cost, depth_values (B,D,h,w) -> depth (B,h,w) [graph], confidence (B,h,w) [no graph]."""
    if not cost.is_cuda:
        raise RuntimeError("casmvsnet_pl_amd.autograd.softmax_depth_regression runs on the MI355X only; there is no CPU fallback")
    return _SoftmaxDepthRegression.apply(cost, depth_values)


def _once(backward):
    """A backward pass that has no second derivative: torch's once_differentiable where a graph is being built (create_graph), which makes a second derivative raise;
    without a graph there is nothing to guard, and the guard's no_grad context is skipped (5 us of a call)."""
    guarded = torch.autograd.function.once_differentiable(backward)

    @functools.wraps(backward)
    def either(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return either


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, slope, channels_last):
        x, weight, bias, *sizes = ops._layer_norm_args(x, weight, bias, eps, slope, channels_last)
        ctx.save_for_backward(x, weight, bias)
        ctx.args = (*sizes, eps, slope)
        return ops._layer_norm_forward(x, weight, bias, *ctx.args)

    @staticmethod
    @_once
    def backward(ctx, gy):
        x, weight, bias = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        gx, gw, gb = ops._layer_norm_backward(x, gy.contiguous(), weight, bias, *ctx.args, need_x, need_w or need_b)
        return gx, gw if need_w else None, gb if need_b else None, None, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5, slope=1.0, channels_last=False):
    """Differentiable ops.layer_norm: x (N,C,*spatial) or (..,C) with channels_last, float32 / float16 / bfloat16; weight, bias (C,) float32 or None.
    What it keeps for the backward pass is x."""
    if not x.is_cuda:
        raise RuntimeError("casmvsnet_pl_amd.autograd.layer_norm runs on the MI355X only; there is no CPU fallback")
    return _LayerNorm.apply(x, weight, bias, float(eps), float(slope), bool(channels_last))


class _DepthCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, cost, depth_values, depth_gt, mask):
        cost = ops._float_dev(cost, "cost")
        if cost.dim() != 4:
            raise ValueError(f"depth_cross_entropy: cost {tuple(cost.shape)}, expected (B,D,h,w)")
        B, D, h, w = cost.shape
        depth_values, depth_gt = (ops._same_device(cost, ops._dev(t, name), name) for t, name in ((depth_values, "depth_values"), (depth_gt, "depth_gt")))
        if tuple(depth_values.shape) not in ((B, D, h, w), (B, D)) or tuple(depth_gt.shape) != (B, h, w):
            raise ValueError(f"depth_cross_entropy: cost {tuple(cost.shape)}, depth_values {tuple(depth_values.shape)}, depth_gt {tuple(depth_gt.shape)}")
        if mask is not None:
            if mask.dtype != torch.bool or tuple(mask.shape) != (B, h, w):
                raise ValueError(f"depth_cross_entropy: mask {tuple(mask.shape)} {mask.dtype}, expected a bool ({B}, {h}, {w})")
            mask = ops._same_device(cost, mask, "mask").contiguous()
        if B * D == 0:
            raise ValueError(f"depth_cross_entropy: cost {tuple(cost.shape)} has no hypotheses")
        code, pixels = ops._DTYPES[cost.dtype], B * h * w
        loss = torch.empty((), dtype=torch.float32, device=cost.device)
        # one buffer: per pixel the running maximum and 1 / sum (two floats) and the class (an int), 1 / count, and (8-byte aligned) the forward's workspace
        at_target, at_share = 8 * pixels, 12 * pixels
        at_ws = at_share + 4 + (at_share + 4) % 8
        kept = torch.empty(at_ws + ops._workspace_bytes("casmvs_depth_ce_workspace_bytes", B, D, h * w), dtype=torch.uint8, device=cost.device)
        base = kept.data_ptr()
        ops._launch("casmvs_depth_ce_forward", cost, cost.data_ptr(), depth_values.data_ptr(), depth_gt.data_ptr(), ops._at(mask), base, base + at_target, loss.data_ptr(),
                    base + at_share, base + at_ws, code, B, D, h * w, int(depth_values.dim() == 4))
        ctx.save_for_backward(cost, kept)
        return loss

    @staticmethod
    @_once
    def backward(ctx, gloss):
        cost, kept = ctx.saved_tensors
        B, D, h, w = cost.shape
        gcost = torch.empty_like(cost)
        base, pixels = kept.data_ptr(), B * h * w
        ops._launch("casmvs_depth_ce_backward", cost, cost.data_ptr(), base, base + 8 * pixels, base + 12 * pixels, gloss.contiguous().data_ptr(), gcost.data_ptr(),
                    ops._DTYPES[cost.dtype], B, D, h * w)
        return gcost, None, None, None


def depth_cross_entropy(cost, depth_values, depth_gt, mask=None):
    """Softmax cross entropy over the depth hypotheses, the mean over the pixels that count (a float32 scalar): cost (B,D,h,w) float32 / float16 / bfloat16,
    depth_values (B,D,h,w) or (B,D) and depth_gt (B,h,w) float32 (finite), mask (B,h,w) bool or None.  The class of a pixel is the hypothesis nearest to
    depth_gt, the lowest index on ties; a pixel counts if its mask is set and depth_gt lies inside the range of its hypotheses (and not all of its costs are -inf).
    Where no pixel counts the loss and its gradient are 0.  Gradient with respect to cost only."""
    if not cost.is_cuda:
        raise RuntimeError("casmvsnet_pl_amd.autograd.depth_cross_entropy runs on the MI355X only; there is no CPU fallback")
    return _DepthCrossEntropy.apply(cost, depth_values, depth_gt, mask)
