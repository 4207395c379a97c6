"""Layer norm as a `norm_act` of the model's layers: CascadeMVSNet(norm_act=LayerNormAct).

The reference's ABN / InPlaceABN (modules.py:14,27) normalises with batch statistics; at the one or two samples per GPU that its training fits, they are
noisy, and they differ between train and eval mode.  This one normalises every position over its channels, in both modes alike.  It cannot be folded into a
convolution's weights, so a model with it runs the layer-by-layer forward of training.py in eval mode too (under no_grad), not the fused inference engine.
"""
import torch
import torch.nn as nn


class LayerNormAct(nn.Module):
    """Layer norm over the channel axis (N,C,*spatial), eps 1e-5, followed by an activation (leaky_relu 0.01 by default): the constructor and the attributes of
    inplace_abn.ABN, without running statistics."""

    def __init__(self, num_features, eps=1e-5, affine=True, activation="leaky_relu", activation_param=0.01):
        super().__init__()
        self.num_features, self.eps, self.affine = num_features, eps, affine
        self.activation, self.activation_param = activation, activation_param
        if affine:
            self.weight = nn.Parameter(torch.ones(num_features))
            self.bias = nn.Parameter(torch.zeros(num_features))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)

    def leaky_slope(self):
        if self.activation == "leaky_relu":
            return float(self.activation_param)
        if self.activation == "relu":
            return 0.0
        if self.activation == "identity":
            return 1.0
        raise RuntimeError(f"unsupported LayerNormAct activation {self.activation!r}")

    def forward(self, x):
        from . import autograd
        if x.dim() < 2 or x.shape[1] != self.num_features:
            raise ValueError(f"LayerNormAct({self.num_features}): x {tuple(x.shape)}")
        return autograd.layer_norm(x, self.weight, self.bias, self.eps, self.leaky_slope())

    def extra_repr(self):
        return f"{self.num_features}, eps={self.eps}, activation={self.activation}[{self.activation_param}]"
