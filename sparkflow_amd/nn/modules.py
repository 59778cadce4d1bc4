"""NN modules backed by the CDNA4 HIP ops.

These are the building blocks for user model-builder functions (the
``build_graph`` convention).  They mirror the TF-1.x layers the reference
examples use (tf.layers.dense / conv2d / max_pooling2d — reference
examples/simple_dnn.py:16-18, examples/cnn_example.py:13-21) with TF's
default glorot-uniform weight init and zero bias init, so convergence
behavior matches.

Weight layouts are chosen for the kernels, not for TF compatibility:
Linear keeps W as [in, out] (row-major GEMM B-operand), Conv2d keeps
[Cout, Cin, Kh, Kw] (NCHW implicit-GEMM).
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from sparkflow_amd.ops import functional as F


def _glorot(shape, fan_in, fan_out, generator=None):
    limit = math.sqrt(6.0 / (fan_in + fan_out))
    return torch.empty(*shape).uniform_(-limit, limit, generator=generator)


class Linear(nn.Module):
    def __init__(self, in_features: int, out_features: int,
                 activation: str = "none", bias: bool = True):
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        self.activation = activation
        self.weight = nn.Parameter(
            _glorot((in_features, out_features), in_features, out_features))
        self.bias = nn.Parameter(torch.zeros(out_features)) if bias else None

    def forward(self, x):
        return F.linear_act(x, self.weight, self.bias, self.activation)

    def extra_repr(self):
        return f"{self.in_features}->{self.out_features}, act={self.activation}"


class Conv2d(nn.Module):
    """``layout="nchw"`` (default) keeps weights [Cout, Cin, Kh, Kw] and
    NCHW tensors; ``layout="nhwc"`` keeps weights [Cout, Kh, Kw, Cin] and
    channel-last tensors (the ResNet-config fast path — channel-
    contiguous float4 im2col reads)."""

    def __init__(self, in_channels: int, out_channels: int, kernel_size: int,
                 stride: int = 1, padding="same", activation: str = "none",
                 bias: bool = True, layout: str = "nchw"):
        super().__init__()
        k = kernel_size
        if padding == "same":
            if stride != 1:
                raise ValueError("padding='same' requires stride=1")
            padding = (k - 1) // 2
        self.stride, self.padding, self.activation = stride, int(padding), activation
        self.layout = layout
        fan_in = in_channels * k * k
        fan_out = out_channels * k * k
        shape = ((out_channels, k, k, in_channels) if layout == "nhwc"
                 else (out_channels, in_channels, k, k))
        self.weight = nn.Parameter(_glorot(shape, fan_in, fan_out))
        self.bias = nn.Parameter(torch.zeros(out_channels)) if bias else None

    def forward(self, x):
        if self.layout == "nhwc":
            return F.conv2d_act_nhwc(x, self.weight, self.bias, self.stride,
                                     self.padding, self.activation)
        return F.conv2d_act(x, self.weight, self.bias, self.stride,
                            self.padding, self.activation)


class MaxPool2d(nn.Module):
    def __init__(self, kernel_size: int, stride: int = None, padding: int = 0,
                 layout: str = "nchw"):
        super().__init__()
        self.kernel_size = kernel_size
        self.stride = stride or kernel_size
        self.padding = padding
        self.layout = layout

    def forward(self, x):
        if self.layout == "nhwc":
            from sparkflow_amd import ops as _ops

            if x.is_cuda and _ops.available():
                return F.maxpool2d_nhwc(x, self.kernel_size, self.stride,
                                        self.padding)
            y = F.maxpool2d(x.permute(0, 3, 1, 2).contiguous(),
                            self.kernel_size, self.stride, self.padding)
            return y.permute(0, 2, 3, 1).contiguous()
        return F.maxpool2d(x, self.kernel_size, self.stride, self.padding)


class Flatten(nn.Module):
    def forward(self, x):
        return x.reshape(x.shape[0], -1)


class BatchNorm2d(nn.Module):
    """BatchNorm2d on the custom CDNA4 kernels (training mode), with an
    optional fused trailing ReLU (``fuse_relu=True`` replaces a separate
    bn -> relu pair).  Eval/CPU fall back to torch batch_norm."""

    def __init__(self, num_features: int, eps: float = 1e-5,
                 momentum: float = 0.1, fuse_relu: bool = False,
                 layout: str = "nchw"):
        super().__init__()
        self.num_features = num_features
        self.eps, self.momentum, self.fuse_relu = eps, momentum, fuse_relu
        self.layout = layout
        self.weight = nn.Parameter(torch.ones(num_features))
        self.bias = nn.Parameter(torch.zeros(num_features))
        self.register_buffer("running_mean", torch.zeros(num_features))
        self.register_buffer("running_var", torch.ones(num_features))

    def forward(self, x, residual=None):
        if self.layout == "nhwc":
            return F.batchnorm2d_act_nhwc(x, self.weight, self.bias,
                                          self.running_mean,
                                          self.running_var, self.momentum,
                                          self.eps, self.fuse_relu,
                                          self.training, residual=residual)
        y = F.batchnorm2d_act(x, self.weight, self.bias,
                              self.running_mean, self.running_var,
                              self.momentum, self.eps,
                              self.fuse_relu and residual is None,
                              self.training)
        if residual is not None:  # NCHW path: plain add (+relu)
            y = y + residual
            if self.fuse_relu:
                y = torch.relu(y)
        return y

    def extra_repr(self):
        return f"{self.num_features}, fuse_relu={self.fuse_relu}"


class Dropout(nn.Module):
    """Inverted dropout; inert in eval mode (the inference path — parity
    with the reference's keep-prob feed at prediction, ml_util.py:70-71).

    With a ``seed`` the masks come from a counter-based generator and are
    not stored for backward (F.dropout): each forward draws the next one,
    also at every replay of a captured step.  The seed belongs to the
    builder, so every worker of a job draws the same sequence from it;
    ``reseed`` starts another.  Without one, torch's generator and a stored
    mask are used.

    A forward that is run again to save memory (torch.utils.checkpoint, which
    winds back torch's generator and not this one) would draw another mask
    for its backward: take the state outside, ``F.dropout_next(rng_state)``,
    and call F.dropout with it inside.
    """

    def __init__(self, p: float = 0.5, seed: int = None):
        super().__init__()
        self.p = p
        # not part of the state dict: artifacts stay loadable either way
        self.register_buffer(
            "rng_state", None if seed is None else F.dropout_state(seed),
            persistent=False)

    def reseed(self, seed: int, offset: int = 0) -> None:
        if getattr(self, "rng_state", None) is None:
            raise ValueError("this Dropout was built without a seed")
        # in place: a captured step keeps reading this tensor
        self.rng_state.copy_(F.dropout_state(seed, offset))

    def forward(self, x):
        if not self.training or self.p <= 0:
            return x
        state = getattr(self, "rng_state", None)  # None in older artifacts
        if state is not None:
            return F.dropout(x, self.p, F.dropout_next(state))
        keep = 1.0 - self.p
        mask = (torch.rand_like(x) < keep).to(x.dtype) / keep
        return x * mask


class AdapterLinear(nn.Module):
    """A frozen Linear with low-rank adapters beside it:
    act(x W + bias + scale (x A_e^T) B_e^T), e the adapter of the row.

    Only the adapters train, so only they are packed, pushed and pulled: at
    rank r a layer sends r (in + out) numbers an adapter and not in * out.
    ``forward(x, ids)`` takes x [..., in_features] and one adapter a row
    (negative: none), in the leading shape of x, or the F.adapter_groups of
    them; without ids every row goes through adapter 0.
    B starts at zero, so a new layer answers as its Linear does.
    """

    def __init__(self, in_features: int, out_features: int, rank: int,
                 adapters: int = 1, scale: float = 1.0,
                 activation: str = "none", bias: bool = True):
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        self.rank, self.adapters, self.scale = rank, adapters, float(scale)
        self.activation = activation
        self.weight = nn.Parameter(
            _glorot((in_features, out_features), in_features, out_features),
            requires_grad=False)
        self.bias = nn.Parameter(torch.zeros(out_features),
                                 requires_grad=False) if bias else None
        self.a = nn.Parameter(
            _glorot((adapters, rank, in_features), in_features, rank))
        self.b = nn.Parameter(torch.zeros(adapters, out_features, rank))

    @classmethod
    def from_linear(cls, linear: Linear, rank: int, adapters: int = 1,
                    scale: float = 1.0) -> "AdapterLinear":
        """Adapters beside a trained layer, whose weights are copied."""
        layer = cls(linear.in_features, linear.out_features, rank, adapters,
                    scale, linear.activation, linear.bias is not None)
        layer.to(linear.weight.device)
        with torch.no_grad():
            layer.weight.copy_(linear.weight)
            if linear.bias is not None:
                layer.bias.copy_(linear.bias)
        return layer

    def forward(self, x, ids=None):
        if ids is None:
            ids = torch.zeros(x.shape[:-1], dtype=torch.int64,
                              device=x.device)
        # the dense kernels take contiguous rows of two axes
        rows = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
        base = F.linear_act(rows.contiguous(), self.weight, self.bias, "none")
        if x.dim() != 2:
            base = base.reshape(x.shape[:-1] + base.shape[1:])
        return F.adapter_add(base, x, self.a, self.b, ids, self.scale,
                             self.activation)

    def extra_repr(self):
        return (f"{self.in_features}->{self.out_features}, "
                f"adapters={self.adapters} of rank {self.rank}, "
                f"act={self.activation}")


class SoftmaxCrossEntropy(nn.Module):
    """Mean softmax cross-entropy (one-hot or index labels)."""

    def forward(self, logits, labels):
        return F.softmax_xent(logits, labels)


class MSE(nn.Module):
    def forward(self, pred, target):
        return F.mse_loss(pred, target)
