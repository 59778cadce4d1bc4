"""Autograd wrappers over the CDNA4 HIP kernels (fp32).

Each op is a ``torch.autograd.Function`` whose GPU path calls the gfx950
extension and whose CPU path implements identical fp32 math with plain
torch ops (used by the no-GPU tests; numerics tests compare the HIP path
against this path).

Replaces the reference's implicit TF ops: dense
GEMM+bias+activation, conv2d, maxpool, softmax-cross-entropy, MSE, argmax.
"""
from __future__ import annotations

import contextlib
import threading
from typing import NamedTuple, Optional

import torch

from sparkflow_amd import ops

ACT_NONE, ACT_RELU, ACT_SIGMOID = 0, 1, 2
ACT_CODES = {"none": ACT_NONE, "linear": ACT_NONE, "relu": ACT_RELU,
             "sigmoid": ACT_SIGMOID}

_TLS = threading.local()


def _want_loss_value() -> bool:
    import os

    if os.environ.get("SPARKFLOW_GRAD_ONLY", "1") == "0":
        return True  # debug toggle: always compute the scalar
    return not getattr(_TLS, "grad_only", False)


@contextlib.contextmanager
def grad_only():
    """Inside this context the loss ops may skip computing the scalar loss
    VALUE (it is undefined) while producing exact gradients — used by the
    training hot loop, where the value is never read.  Saves the
    zero-fill / atomic-reduce / mean kernels per step (GPU path only; the
    CPU path always computes the value)."""
    prev = getattr(_TLS, "grad_only", False)
    _TLS.grad_only = True
    try:
        yield
    finally:
        _TLS.grad_only = prev


@contextlib.contextmanager
def defer_wgrad(records: list):
    """Inside this context LinearAct.backward appends
    ``(weight_data_ptr, workspace)`` to ``records`` instead of reducing
    the wgrad split-K workspace to per-tensor grads (the weight/bias
    grads it returns are then None).  The captured step feeds the raw
    workspaces to ``reduce_apply_adam`` — one launch replaces every
    wgrad reduce, pack_segments, and the Adam apply.  GPU biased-Linear
    layers only; other ops ignore the context (the caller checks
    coverage and falls back)."""
    prev = getattr(_TLS, "defer_wgrad", None)
    _TLS.defer_wgrad = records
    try:
        yield
    finally:
        _TLS.defer_wgrad = prev


def _defer_records():
    return getattr(_TLS, "defer_wgrad", None)


def _dev_scale(dloss: torch.Tensor) -> torch.Tensor:
    """Upstream loss grad as a device fp32 scalar for the HIP bwd kernels.

    Kept on-device (the kernel dereferences it) so the backward pass never
    d2h-syncs — a host `float(dloss)` would break hipGraph capture of the
    full training step."""
    return dloss.detach().to(dtype=torch.float32).contiguous()


def _act_fwd(pre: torch.Tensor, act: int) -> torch.Tensor:
    if act == ACT_RELU:
        return torch.relu(pre)
    if act == ACT_SIGMOID:
        return torch.sigmoid(pre)
    return pre


def _act_bwd_from_out(y: torch.Tensor, dy: torch.Tensor, act: int) -> torch.Tensor:
    # activation grads recomputed from the *output* (saves the preactivation)
    if act == ACT_RELU:
        return dy * (y > 0).to(dy.dtype)
    if act == ACT_SIGMOID:
        return dy * y * (1.0 - y)
    return dy


class LinearAct(torch.autograd.Function):
    """y = act(x @ W + b) with x:[M,K], W:[K,N] (TF dense layout), b:[N]."""

    @staticmethod
    def forward(ctx, x, w, b, act: int):
        if ops.use_hip(x):
            y = ops.hip.gemm_act(x, w, b if b is not None else torch.empty(0, device=x.device), act)
        else:
            pre = x @ w
            if b is not None:
                pre = pre + b
            y = _act_fwd(pre, act)
        ctx.save_for_backward(x, w, y)
        ctx.act = act
        ctx.has_bias = b is not None
        # Captured at FORWARD time (defer_wgrad is entered on the thread
        # running the step; autograd executes backward on its own engine
        # thread where the thread-local would be invisible).
        ctx.defer_sink = _defer_records()
        return y

    @staticmethod
    def backward(ctx, dy):
        import os

        x, w, y = ctx.saved_tensors
        act = ctx.act
        need_dx = ctx.needs_input_grad[0]
        dy = dy.contiguous()
        fused = os.environ.get("SPARKFLOW_FUSED_ACTBWD", "1") != "0"
        if not (ctx.needs_input_grad[1] or ctx.needs_input_grad[2]):
            # a frozen layer (adapters train beside it): no weight grads
            if not need_dx:
                return None, None, None, None
            if ops.use_hip(x):
                if act != ACT_NONE and fused:
                    dx = ops.hip.gemm_dgrad_act(dy, y, w, act)
                else:
                    dpre = ops.hip.act_bwd(y, dy, act) \
                        if act != ACT_NONE else dy
                    dx = ops.hip.gemm_dgrad(dpre, w)
            else:
                dx = _act_bwd_from_out(y, dy, act) @ w.t()
            return dx, None, None, None
        if ops.use_hip(x):
            recs = ctx.defer_sink
            if recs is not None and ctx.has_bias:
                # deferred-reduce mode: hand the raw split-K workspace to
                # the fused reduce+apply; weight/bias grads stay None
                if act != ACT_NONE and fused:
                    dx = ops.hip.gemm_dgrad_act(dy, y, w, act) \
                        if need_dx else None
                    ws = ops.hip.gemm_wgrad_bias_act_ws(x, dy, y, act)
                else:
                    dpre = ops.hip.act_bwd(y, dy, act) \
                        if act != ACT_NONE else dy
                    dx = ops.hip.gemm_dgrad(dpre, w) if need_dx else None
                    ws = ops.hip.gemm_wgrad_bias_ws(x, dpre)
                recs.append((w.data_ptr(), ws))
                return dx, None, None, None
            if act != ACT_NONE and ctx.has_bias and fused:
                # activation backward fused into BOTH backward GEMMs'
                # operand loads — no standalone act_bwd pass or dpre buf
                dx = ops.hip.gemm_dgrad_act(dy, y, w, act) \
                    if need_dx else None
                dwb = ops.hip.gemm_wgrad_bias_act(x, dy, y, act)
                k = x.shape[1]
                dw, db = dwb[:k], dwb[k]
                return dx, dw, db, None
            dpre = ops.hip.act_bwd(y, dy, act) if act != ACT_NONE else dy
            dx = ops.hip.gemm_dgrad(dpre, w) if need_dx else None
            if ctx.has_bias:
                # bias grad rides the wgrad GEMM as a virtual ones-row
                dwb = ops.hip.gemm_wgrad_bias(x, dpre)
                k = x.shape[1]
                dw, db = dwb[:k], dwb[k]
            else:
                dw, db = ops.hip.gemm_wgrad(x, dpre), None
        else:
            dpre = _act_bwd_from_out(y, dy, act)
            dx = dpre @ w.t() if need_dx else None
            dw = x.t() @ dpre
            db = dpre.sum(dim=0) if ctx.has_bias else None
        return dx, dw, db, None


def linear_act(x, w, b=None, act="none"):
    return LinearAct.apply(x, w, b, ACT_CODES[act] if isinstance(act, str) else act)


class SoftmaxXent(torch.autograd.Function):
    """Mean softmax-cross-entropy over rows; labels are one-hot [M,C]."""

    @staticmethod
    def forward(ctx, logits, onehot):
        if ops.use_hip(logits):
            loss, probs = ops.hip.softmax_xent_fwd(logits, onehot,
                                                   _want_loss_value())
        else:
            lse = torch.logsumexp(logits, dim=1, keepdim=True)
            logp = logits - lse
            loss = -(onehot * logp).sum(dim=1).mean()
            probs = torch.exp(logp)
        ctx.save_for_backward(probs, onehot)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        probs, onehot = ctx.saved_tensors
        m = probs.shape[0]
        if ops.use_hip(probs):
            dlogits = ops.hip.softmax_xent_bwd(probs, onehot,
                                               _dev_scale(dloss), 1.0 / m)
        else:
            dlogits = (probs - onehot) * (dloss / m)
        return dlogits, None


class SoftmaxXentIdx(torch.autograd.Function):
    """Class-index label path — no one-hot materialization (the fused
    kernel reads int64 OR integral-float labels directly).

    Under ``grad_only()`` the forward kernel writes the GRADIENT
    ``(probs - onehot)/m`` instead of the probs and backward returns it
    as-is — the whole loss fwd+bwd is ONE kernel.  That contract assumes
    a unit upstream gradient (which ``grad_only`` callers guarantee by
    backpropagating a ones root)."""

    @staticmethod
    def forward(ctx, logits, labels):
        grad_fused = False
        if ops.use_hip(logits):
            grad_fused = not _want_loss_value()
            loss, probs = ops.hip.softmax_xent_idx_fwd(
                logits, labels, not grad_fused, grad_fused)
        else:
            lab = labels.long()
            lse = torch.logsumexp(logits, dim=1, keepdim=True)
            logp = logits - lse
            loss = -logp.gather(1, lab.view(-1, 1)).mean()
            probs = torch.exp(logp)
        ctx.save_for_backward(probs, labels)
        ctx.grad_fused = grad_fused
        return loss

    @staticmethod
    def backward(ctx, dloss):
        probs, labels = ctx.saved_tensors
        m = probs.shape[0]
        if ctx.grad_fused:
            return probs, None  # probs holds (softmax - onehot)/m already
        if ops.use_hip(probs):
            dlogits = ops.hip.softmax_xent_idx_bwd(probs, labels,
                                                   _dev_scale(dloss), 1.0 / m)
        else:
            dlogits = probs.clone()
            dlogits[torch.arange(m, device=probs.device),
                    labels.long()] -= 1.0
            dlogits.mul_(dloss / m)
        return dlogits, None


def softmax_xent(logits, labels):
    """labels: one-hot [M,C], class-index [M], or class-index [M,1]
    (the engine's ``handle_features`` wraps scalar labels to [y])."""
    if labels.dim() == 2 and labels.size(1) == 1 and logits.size(1) != 1:
        labels = labels.reshape(-1)
    if labels.dim() == 1:
        if ops.use_hip(logits) and labels.dtype in (torch.float32,
                                                    torch.int64):
            # HIP kernels read float labels directly — no cast kernel
            return SoftmaxXentIdx.apply(logits, labels.contiguous())
        return SoftmaxXentIdx.apply(logits, labels.long().contiguous())
    return SoftmaxXent.apply(logits, labels.to(logits.dtype).contiguous())


class MseLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, pred, target):
        ctx.save_for_backward(pred, target)
        if ops.use_hip(pred):
            return ops.hip.mse_fwd(pred, target, _want_loss_value())
        return ((pred - target) ** 2).mean()

    @staticmethod
    def backward(ctx, dloss):
        pred, target = ctx.saved_tensors
        n = pred.numel()
        if ops.use_hip(pred):
            dpred = ops.hip.mse_bwd(pred, target, _dev_scale(dloss), 2.0 / n)
        else:
            dpred = (pred - target) * (2.0 * dloss / n)
        return dpred, None


def mse_loss(pred, target):
    return MseLoss.apply(pred, target)


class Conv2dAct(torch.autograd.Function):
    """NCHW conv2d + bias + activation. w: [Cout, Cin, Kh, Kw]."""

    @staticmethod
    def forward(ctx, x, w, b, stride: int, pad: int, act: int):
        if ops.use_hip(x):
            y = ops.hip.conv_gemm_fwd(
                x, w, b if b is not None else torch.empty(0, device=x.device),
                stride, pad, act)
        else:
            pre = torch.nn.functional.conv2d(x, w, b, stride=stride, padding=pad)
            y = _act_fwd(pre, act)
        ctx.save_for_backward(x, w, y)
        ctx.conf = (stride, pad, act, b is not None)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w, y = ctx.saved_tensors
        stride, pad, act, has_bias = ctx.conf
        need_dx = ctx.needs_input_grad[0]
        dy = dy.contiguous()
        if ops.use_hip(x):
            dpre = ops.hip.act_bwd(y, dy, act) if act != ACT_NONE else dy
            if not need_dx:
                dx = None
            else:
                # dgrad IS a conv: dx = corr(dy, W swapped+rotated) with
                # padding K-1-p on the implicit-GEMM MFMA path; stride>1
                # zero-stuffs dy first (the trailing remainder rows/cols
                # recover the exact input size) — ~10x over the direct
                # strided dgrad kernel on ResNet shapes.
                wt = w.transpose(0, 1).flip(2, 3).contiguous()
                kk = w.shape[2]
                if stride == 1:
                    src = dpre
                else:
                    rh = (x.shape[2] + 2 * pad - kk) % stride
                    rw = (x.shape[3] + 2 * pad - kk) % stride
                    src = ops.hip.conv_dilate(dpre, stride, rh, rw)
                dx = ops.hip.conv_gemm_fwd(
                    src, wt, torch.empty(0, device=x.device), 1,
                    kk - 1 - pad, ACT_NONE)
            dw = ops.hip.conv_gemm_wgrad(x, dpre, w.shape[2], w.shape[3],
                                         stride, pad)
            db = ops.hip.conv_bias_grad(dpre) if has_bias else None
        else:
            dpre = _act_bwd_from_out(y, dy, act)
            dx = torch.nn.grad.conv2d_input(x.shape, w, dpre, stride=stride,
                                            padding=pad) if need_dx else None
            dw = torch.nn.grad.conv2d_weight(x, w.shape, dpre, stride=stride,
                                             padding=pad)
            db = dpre.sum(dim=(0, 2, 3)) if has_bias else None
        return dx, dw, db, None, None, None


def conv2d_act(x, w, b=None, stride=1, pad=0, act="none"):
    return Conv2dAct.apply(x, w, b, stride, pad,
                           ACT_CODES[act] if isinstance(act, str) else act)


class Conv2dActNHWC(torch.autograd.Function):
    """Channel-last conv: x [N,H,W,Cin], w [Cout,Kh,Kw,Cin] — im2col
    gathers and output stores are channel-contiguous float4s (the NCHW
    kernels were gather-latency-bound on ResNet shapes).  CPU fallback
    permutes through torch's NCHW conv."""

    @staticmethod
    def forward(ctx, x, w, b, stride: int, pad: int, act: int):
        # MEASURED NEGATIVE (round 2): zero-padding Cin 1->4 / 3->4 to
        # reach the float4 gather path multiplies the GEMM K work by
        # 4/Cin, which costs more than the scalar gathers it removes
        # (MNIST CNN -10%, ResNet-18 -1.3%).  Keep the scalar path.
        cpad = 0
        if ops.use_hip(x):
            y = ops.hip.conv_nhwc_fwd(
                x, w, b if b is not None else torch.empty(0, device=x.device),
                stride, pad, act)
        else:
            xc = x.permute(0, 3, 1, 2)
            wc = w.permute(0, 3, 1, 2)
            pre = torch.nn.functional.conv2d(xc, wc, b, stride=stride,
                                             padding=pad)
            y = _act_fwd(pre, act).permute(0, 2, 3, 1).contiguous()
        ctx.save_for_backward(x, w, y)
        ctx.conf = (stride, pad, act, b is not None, cpad)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w, y = ctx.saved_tensors
        stride, pad, act, has_bias, cpad = ctx.conf
        need_dx = ctx.needs_input_grad[0]
        dy = dy.contiguous()
        kk = w.shape[1]
        if ops.use_hip(x):
            dpre = ops.hip.act_bwd(y, dy, act) if act != ACT_NONE else dy
            if not need_dx:
                dx = None
            else:
                # dgrad IS a stride-1 conv of dpre with spatially-
                # flipped, in/out-swapped weights.  stride > 1 uses the
                # direct s^2-sub-convolution kernel (no zero-stuffed
                # dilation: the dilated form ran s^2 x the useful MFMA
                # work); the dilate path stays as the Cout%4!=0 fallback.
                wt = w.flip(1, 2).permute(3, 1, 2, 0).contiguous()
                if stride == 1:
                    dx = ops.hip.conv_nhwc_fwd(
                        dpre, wt, torch.empty(0, device=x.device), 1,
                        kk - 1 - pad, ACT_NONE)
                elif w.shape[0] % 4 == 0:
                    dx = ops.hip.conv_nhwc_dgrad_strided(
                        dpre, wt, x.shape[1], x.shape[2], stride, pad)
                else:
                    rh = (x.shape[1] + 2 * pad - kk) % stride
                    rw = (x.shape[2] + 2 * pad - kk) % stride
                    src = ops.hip.conv_nhwc_dilate(dpre, stride, rh, rw)
                    dx = ops.hip.conv_nhwc_fwd(
                        src, wt, torch.empty(0, device=x.device), 1,
                        kk - 1 - pad, ACT_NONE)
            dw = ops.hip.conv_nhwc_wgrad(x, dpre, kk, w.shape[2], stride,
                                         pad)
            db = ops.hip.conv_nhwc_bias_grad(dpre) if has_bias else None
        else:
            dpre = _act_bwd_from_out(y, dy, act)
            xc = x.permute(0, 3, 1, 2)
            wc = w.permute(0, 3, 1, 2)
            dpc = dpre.permute(0, 3, 1, 2)
            dx = None
            if need_dx:
                dx = torch.nn.grad.conv2d_input(
                    xc.shape, wc, dpc, stride=stride, padding=pad) \
                    .permute(0, 2, 3, 1).contiguous()
            dw = torch.nn.grad.conv2d_weight(
                xc, wc.shape, dpc, stride=stride, padding=pad) \
                .permute(0, 2, 3, 1).contiguous()
            db = dpre.sum(dim=(0, 1, 2)) if has_bias else None
        return dx, dw, db, None, None, None


def conv2d_act_nhwc(x, w, b=None, stride=1, pad=0, act="none"):
    return Conv2dActNHWC.apply(x, w, b, stride, pad,
                               ACT_CODES[act] if isinstance(act, str)
                               else act)


class BatchNorm2dActNHWC(torch.autograd.Function):
    """NHWC training BN with optional fused trailing ReLU AND optional
    fused ResNet-block residual add: out = relu(bn(x) + res).  Fusing
    the add+relu into the norm kernel (and the relu-masked d_res into
    the bwd-dx kernel) removes two full activation-tensor passes per
    block boundary."""

    @staticmethod
    def forward(ctx, x, gamma, beta, run_mean, run_var, momentum, eps,
                relu, res=None):
        empty = torch.empty(0, device=x.device, dtype=x.dtype)
        y, mean, invstd = ops.hip.bn2d_nhwc_fwd(
            x, gamma, beta, run_mean, run_var, momentum, eps, relu,
            res.contiguous() if res is not None else empty)
        ctx.save_for_backward(x, y, gamma, mean, invstd)
        ctx.relu = relu
        ctx.has_res = res is not None
        return y

    @staticmethod
    def backward(ctx, dy):
        x, y, gamma, mean, invstd = ctx.saved_tensors
        dx, dgamma, dbeta, dres = ops.hip.bn2d_nhwc_bwd(
            x, dy.contiguous(), y, gamma, mean, invstd, ctx.relu,
            ctx.has_res)
        return (dx, dgamma, dbeta, None, None, None, None, None,
                dres if ctx.has_res else None)


def batchnorm2d_act_nhwc(x, gamma, beta, run_mean, run_var, momentum=0.1,
                         eps=1e-5, relu=False, training=True,
                         residual=None):
    """x: [N, H, W, C] channel-last.  ``residual`` fuses a ResNet block
    boundary: out = relu(bn(x) + residual)."""
    if training and ops.use_hip(x):
        return BatchNorm2dActNHWC.apply(x.contiguous(), gamma, beta,
                                        run_mean, run_var, momentum, eps,
                                        relu, residual)
    xc = x.permute(0, 3, 1, 2)
    y = torch.nn.functional.batch_norm(xc, run_mean, run_var, gamma, beta,
                                       training, momentum, eps)
    y = y.permute(0, 2, 3, 1)
    if residual is not None:
        y = y + residual
    if relu:
        y = torch.relu(y)
    return y.contiguous()


class MaxPool2d(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, k: int, stride: int, pad: int):
        if ops.use_hip(x):
            y, idx = ops.hip.maxpool2d_fwd(x, k, stride, pad)
        else:
            y, idx = torch.nn.functional.max_pool2d(x, k, stride, padding=pad,
                                                    return_indices=True)
        ctx.save_for_backward(idx)
        ctx.conf = (x.shape, k, stride, pad)
        return y

    @staticmethod
    def backward(ctx, dy):
        (idx,) = ctx.saved_tensors
        shape, k, stride, pad = ctx.conf
        dy = dy.contiguous()
        if ops.use_hip(dy):
            dx = ops.hip.maxpool2d_bwd(dy, idx, shape[2], shape[3])
        else:
            # scatter_add, NOT max_unpool2d: with overlapping windows
            # (stride < k) one input can be the max of several windows
            # and unpool would overwrite instead of accumulating
            n, c = shape[0], shape[1]
            dx = torch.zeros(n, c, shape[2] * shape[3], dtype=dy.dtype)
            dx.scatter_add_(2, idx.reshape(n, c, -1), dy.reshape(n, c, -1))
            dx = dx.reshape(shape)
        return dx, None, None, None


def maxpool2d(x, k, stride=None, pad=0):
    return MaxPool2d.apply(x, k, stride or k, pad)


class MaxPool2dNHWC(torch.autograd.Function):
    """Channel-last maxpool (GPU only; the module's CPU path permutes
    through the torch NCHW pool)."""

    @staticmethod
    def forward(ctx, x, k: int, stride: int, pad: int):
        y, idx = ops.hip.maxpool_nhwc_fwd(x, k, stride, pad)
        ctx.save_for_backward(idx)
        ctx.conf = (x.shape[1], x.shape[2], k, stride, pad)
        return y

    @staticmethod
    def backward(ctx, dy):
        (idx,) = ctx.saved_tensors
        H, W, k, stride, pad = ctx.conf
        return ops.hip.maxpool_nhwc_bwd(dy.contiguous(), idx, H, W, k,
                                        stride, pad), \
            None, None, None


def maxpool2d_nhwc(x, k, stride=None, pad=0):
    return MaxPool2dNHWC.apply(x, k, stride or k, pad)


class BatchNorm2dAct(torch.autograd.Function):
    """Training-mode BatchNorm2d with optional fused ReLU on the custom
    CDNA4 kernels (MIOpen's spatial BN was 27% of the ResNet-shape step).
    Updates running stats in-place as a forward side effect."""

    @staticmethod
    def forward(ctx, x, gamma, beta, run_mean, run_var, momentum, eps,
                relu):
        y, mean, invstd = ops.hip.bn2d_fwd(x, gamma, beta, run_mean,
                                           run_var, momentum, eps, relu)
        ctx.save_for_backward(x, y, gamma, mean, invstd)
        ctx.relu = relu
        return y

    @staticmethod
    def backward(ctx, dy):
        x, y, gamma, mean, invstd = ctx.saved_tensors
        dx, dgamma, dbeta = ops.hip.bn2d_bwd(x, dy.contiguous(), y, gamma,
                                             mean, invstd, ctx.relu)
        return dx, dgamma, dbeta, None, None, None, None, None


def batchnorm2d_act(x, gamma, beta, run_mean, run_var, momentum=0.1,
                    eps=1e-5, relu=False, training=True):
    if training and ops.use_hip(x):
        return BatchNorm2dAct.apply(x.contiguous(), gamma, beta, run_mean,
                                    run_var, momentum, eps, relu)
    y = torch.nn.functional.batch_norm(x, run_mean, run_var, gamma, beta,
                                       training, momentum, eps)
    return torch.relu(y) if relu else y


# -- dropout from a counter ---------------------------------------------------

_FLOAT_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check_float(name: str, t: torch.Tensor) -> None:
    if t.dtype not in _FLOAT_TYPES:
        raise ValueError("%s must be fp32, bf16 or fp16, got %s"
                         % (name, t.dtype))


def dropout_state(seed: int, offset: int = 0, device=None) -> torch.Tensor:
    """The two 64-bit numbers that a dropout mask is drawn from: the
    generator's key and the number of the draw."""
    def signed(v):
        return (int(v) + 2 ** 63) % 2 ** 64 - 2 ** 63

    return torch.tensor([signed(seed), signed(offset)], dtype=torch.int64,
                        device=device)


def _check_state(state: torch.Tensor) -> None:
    if state.dtype != torch.int64 or state.numel() != 2 \
            or not state.is_contiguous():
        raise ValueError("state must be two contiguous int64 (see "
                         "dropout_state)")


def dropout_next(state: torch.Tensor) -> torch.Tensor:
    """The state for one draw; steps ``state`` on to the next draw in
    place.  On a GPU both happen on the device in one launch, so a
    captured step draws a new mask at each replay."""
    _check_state(state)
    if ops.use_hip(state):
        return ops.hip.dropout_next(state)
    out = state.clone()
    state[1] += 1
    return out


def _mul32(a: int, c: torch.Tensor):
    """(high, low) 32 bits of a * c for 32-bit values held in int64: the
    product is taken in two halves of 48 bits, its low part modulo 2^64."""
    high = (a * (c >> 16) + ((a * (c & 0xFFFF)) >> 16)) >> 16
    return high, (a * c) & 0xFFFFFFFF


def _philox_words(state: torch.Tensor, n: int) -> torch.Tensor:
    """The first n words of the CPU path, in int64 (the GPU kernel's words;
    see ops/hip/dropout.hip)."""
    mask = 0xFFFFFFFF
    seed, offset = (int(v) for v in state)
    at = torch.arange((n + 3) // 4, dtype=torch.int64)
    c0, c1 = at & mask, at >> 32
    c2 = torch.full_like(at, offset & mask)
    c3 = torch.full_like(at, (offset >> 32) & mask)
    k0, k1 = seed & mask, (seed >> 32) & mask
    for _ in range(10):
        h0, l0 = _mul32(0xD2511F53, c0)
        h1, l1 = _mul32(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return torch.stack((c0, c1, c2, c3), 1).reshape(-1)[:n]


class _DropoutCPU(torch.autograd.Function):
    """The mask is a function of the state and the element's index; only
    the state is kept, and backward draws the same mask again."""

    @staticmethod
    def forward(ctx, x, state, keep: int, scale: float):
        ctx.save_for_backward(state)
        ctx.conf = (keep, scale)
        kept = (_philox_words(state, x.numel()) < keep).reshape(x.shape)
        y = (x.to(torch.float32) * scale).to(x.dtype)
        return torch.where(kept, y, torch.zeros_like(y))

    @staticmethod
    def backward(ctx, dy):
        (state,) = ctx.saved_tensors
        return _DropoutCPU.apply(dy, state, *ctx.conf), None, None, None


def dropout(x, p: float, state, training: bool = True):
    """Inverted dropout with a mask that is drawn from ``state`` (see
    ``dropout_state`` and ``dropout_next``) and never stored.

    An element is kept with probability 1 - p and scaled by 1 / (1 - p); a
    dropped one is 0 whatever it held.  The same state gives the same mask
    for the same number of elements, on any device, in any type.  x: fp32,
    bf16 or fp16, any shape, on a GPU less than 64 GiB; other layouts than
    contiguous are copied.  Without ``training``, or with p = 0, x comes
    back as it is.
    """
    _check_float("x", x)
    if not 0.0 <= p <= 1.0:
        raise ValueError("p must be within 0 and 1, got %r" % (p,))
    _check_state(state)
    if state.device != x.device:
        raise ValueError("x is on %s and state on %s"
                         % (x.device, state.device))
    if not training or p == 0.0:
        return x
    keep = round((1.0 - p) * 2 ** 32)  # of 2^32 words
    scale = 1.0 / (1.0 - p) if keep else 0.0
    if ops.use_hip(x):
        return ops.hip.dropout_apply(x, state, keep, scale)
    return _DropoutCPU.apply(x, state, keep, scale)


# -- log-probabilities of given tokens ----------------------------------------

_TOP_MAX = 32


class TokenLogProbs(NamedTuple):
    """``logp`` and ``entropy``: one fp32 a row; ``top_logp`` (fp32) and
    ``top_ids`` (int64): the ``top_k`` best classes, best first."""
    logp: torch.Tensor
    entropy: torch.Tensor
    top_logp: torch.Tensor
    top_ids: torch.Tensor


class _TokenLogProbsCPU(torch.autograd.Function):

    @staticmethod
    def forward(ctx, logits, tokens, k: int, ignore: int):
        ctx.set_materialize_grads(False)
        logp, entropy, stat, top, ids = _logprobs_cpu(logits, tokens, k,
                                                      ignore)
        ctx.save_for_backward(logits, tokens, stat, entropy, ids)
        ctx.ignore = ignore
        ctx.mark_non_differentiable(ids)
        return logp, entropy, top, ids

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logp, g_entropy, g_top, _):
        dx = _logprobs_grad_cpu(*ctx.saved_tensors, g_logp, g_entropy, g_top,
                                ctx.ignore)
        return dx, None, None, None


def _logprobs_cpu(logits, tokens, k, ignore):
    x = logits.to(torch.float32)
    m, c = x.shape
    live = tokens != ignore
    known = (tokens >= 0) & (tokens < c)
    best = x.amax(1, keepdim=True)
    # a row of -inf alone: no class is possible
    empty = (best == -float("inf")).squeeze(1)
    shift = torch.where(best == -float("inf"), torch.zeros_like(best), best)
    log_sum = torch.exp(x - shift).sum(1, keepdim=True).log()
    log_sum = torch.where(empty.unsqueeze(1), torch.zeros_like(log_sum),
                          log_sum)
    all_logp = torch.where(x == -float("inf"), x, (x - shift) - log_sum)
    p = torch.where(empty.unsqueeze(1), torch.zeros_like(x),
                    torch.exp(all_logp))
    entropy = -torch.where(p == 0, torch.zeros_like(p), p * all_logp).sum(1)
    logp = all_logp.gather(
        1, torch.where(known, tokens, 0).unsqueeze(1)).squeeze(1)
    logp = torch.where(known, logp, torch.full_like(logp, float("nan")))
    ids = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :k]
    top = all_logp.gather(1, ids)
    broken = torch.isnan(log_sum)  # a NaN or +inf: no distribution
    logp = torch.where(broken.squeeze(1), log_sum.squeeze(1), logp)
    top = torch.where(broken, log_sum, top)
    ids = torch.where(broken, torch.full_like(ids, -1), ids)
    # rows that are not read
    logp, entropy = (torch.where(live, t, torch.zeros_like(t))
                     for t in (logp, entropy))
    top = torch.where(live.unsqueeze(1), top, torch.zeros_like(top))
    ids = torch.where(live.unsqueeze(1), ids, torch.full_like(ids, -1))
    return logp, entropy, torch.cat((best, log_sum), 1), top, ids


def _logprobs_grad_cpu(logits, tokens, stat, entropy, ids, g_logp, g_entropy,
                       g_top, ignore):
    x = logits.to(torch.float32)
    m, c = x.shape
    live = (tokens != ignore).unsqueeze(1)
    known = ((tokens >= 0) & (tokens < c)).unsqueeze(1)
    one_hot = torch.zeros_like(x)
    if g_logp is not None:
        g = g_logp.unsqueeze(1)
        g = torch.where(known, g, torch.full_like(g, float("nan")))
        one_hot.scatter_add_(
            1, torch.where(known.squeeze(1), tokens, 0).unsqueeze(1), g)
    if g_top is not None:
        one_hot.scatter_add_(1, ids.clamp(min=0), g_top)
    share = one_hot.sum(1, keepdim=True)
    best, log_sum = stat[:, :1], stat[:, 1:]
    h = entropy.unsqueeze(1)
    logp = (x - best) - log_sum
    p = torch.exp(logp)
    d = one_hot - p * share
    if g_entropy is not None:
        d = d - g_entropy.unsqueeze(1) * torch.where(
            p == 0, torch.zeros_like(p), p * (logp + h))
    if g_logp is not None:
        d = torch.where(known, d, torch.full_like(d, float("nan")))
    constant = (best == -float("inf")) & (log_sum == 0) & (
        known if g_logp is not None else torch.ones_like(known))
    d = torch.where(live & ~constant, d, torch.zeros_like(d))
    return d.to(logits.dtype)


def token_logprobs(logits, tokens, top_k: int = 0,
                   ignore_index: int = -100) -> TokenLogProbs:
    """Log-probability of one given class a row, with the entropy of the
    row's distribution and its ``top_k`` best classes; gradients flow from
    all three.

    logits: [..., classes] in fp32, bf16 or fp16, read in place where the
    classes lie side by side (rows may be strided, as in a slice of a
    padded vocabulary).  tokens: the leading shape of logits, or that with
    a last extent of 1 (the engine's labels); whole numbers in an integer
    type or fp32.  ``top_k`` is at most 32 and the number of classes; of
    equal logits the lower class is the better one.  On a GPU rows are less
    than 2^24, with up to 1024 classes 2^26.

    * A row whose token is ``ignore_index`` is not read: zeros, top ids
      of -1, and a gradient of zero.  A mean over rows has to leave the
      ignored ones out.
    * A token outside 0 .. classes - 1 cannot be refused without waiting
      for the device: its log-probability is NaN, and so is its row of the
      gradient if one flows from there.
    * A logit of -inf has probability 0 and adds nothing to the entropy; in
      its gradient the probability's terms are 0.  What flows to a class
      that is named, as the token or as an alternative, reaches its logit
      all the same, as in a log-softmax: where fewer classes than ``top_k``
      are possible, leave the impossible alternatives (a ``top_logp`` of
      -inf) out of the loss.  A row of nothing else has -inf for every
      class, an entropy of 0 and a gradient of zero.
    * A row that holds NaN or +inf has no distribution: NaN everywhere and
      top ids of -1.
    """
    _check_float("logits", logits)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("logits must be [..., classes], got %s"
                         % (tuple(logits.shape),))
    classes = logits.shape[-1]
    if tokens.dim() == logits.dim() and tokens.shape[-1] == 1:
        tokens = tokens.squeeze(-1)
    if tokens.shape != logits.shape[:-1]:
        raise ValueError("tokens of shape %s do not fit logits of shape %s"
                         % (tuple(tokens.shape), tuple(logits.shape)))
    if tokens.device != logits.device:
        raise ValueError("logits are on %s and tokens on %s"
                         % (logits.device, tokens.device))
    if tokens.dtype == torch.bool or tokens.is_complex() or (
            tokens.is_floating_point() and tokens.dtype != torch.float32):
        raise ValueError("tokens must be whole numbers in an integer type "
                         "or fp32, got %s" % (tokens.dtype,))
    if not 0 <= top_k <= min(_TOP_MAX, classes):
        raise ValueError("top_k must be within 0 and min(%d, %d classes), "
                         "got %r" % (_TOP_MAX, classes, top_k))
    tokens = tokens.detach()
    if tokens.dtype not in (torch.float32, torch.int64):
        tokens = tokens.long()
    if ops.use_hip(logits):
        return TokenLogProbs(*ops.hip.logprobs_apply(
            logits, tokens, top_k, ignore_index))
    shape = tokens.shape
    logp, entropy, top, ids = _TokenLogProbsCPU.apply(
        logits.reshape(-1, classes), tokens.reshape(-1).long(), top_k,
        ignore_index)
    return TokenLogProbs(logp.reshape(shape), entropy.reshape(shape),
                         top.reshape(shape + (top_k,)),
                         ids.reshape(shape + (top_k,)))


# -- low-rank adapters --------------------------------------------------------

_RANK_MAX, _ADAPTERS_MAX = 128, 1024


class AdapterGroups:
    """The rows of a batch grouped by adapter, for every ``adapter_add`` on
    the same rows (the layers of a model): see ``adapter_groups``."""

    def __init__(self, ids, adapters: int):
        self.adapters = adapters
        self.shape = ids.shape
        # its own copy: what the caller does to ids later changes nothing
        self.ids = ids.detach().reshape(-1).to(torch.int64, copy=True)
        self.device = ids.device
        self.plan = ops.hip.adapter_plan(self.ids, adapters) \
            if ops.use_hip(ids) else None


def adapter_groups(ids, adapters: int) -> AdapterGroups:
    """Groups rows by adapter once, for several ``adapter_add``.

    ids: whole numbers in an integer type, one a row.  0 .. adapters - 1
    name an adapter, a negative number none.
    """
    _check_ids(ids, adapters)
    return AdapterGroups(ids, adapters)


def _check_ids(ids, adapters: int) -> None:
    if ids.dtype == torch.bool or ids.is_floating_point() \
            or ids.is_complex():
        raise ValueError("ids must be whole numbers in an integer type, "
                         "got %s" % (ids.dtype,))
    if not 1 <= adapters <= _ADAPTERS_MAX:
        raise ValueError("adapters must be within 1 and %d, got %r"
                         % (_ADAPTERS_MAX, adapters))


class _AdapterAddCPU(torch.autograd.Function):

    @staticmethod
    def forward(ctx, base, x, a, b, scales, scale, ids, act: int):
        z, y = _adapter_cpu(base, x, a, b, scales, scale, ids, act)
        ctx.save_for_backward(x, a, b, z, scales, ids,
                              y if act != ACT_NONE else None)
        ctx.conf = (scale, act)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        grads = _adapter_grad_cpu(*ctx.saved_tensors, dy, *ctx.conf)
        return tuple(g if need else None for g, need in zip(
            grads, ctx.needs_input_grad)) + (None,) * 4


def _adapter_rows(ids, adapters, scales, scale):
    for e in range(adapters):
        rows = (ids == e).nonzero().squeeze(1)
        if len(rows):
            yield e, rows, scale if scales is None else scales[e]


def _adapter_cpu(base, x, a, b, scales, scale, ids, act):
    f32 = torch.float32
    y = base.to(f32).clone()
    z = torch.zeros(x.shape[0], a.shape[1], dtype=f32)
    for e, rows, s in _adapter_rows(ids, len(a), scales, scale):
        z[rows] = s * (x[rows].to(f32) @ a[e].to(f32).t())
        y[rows] += z[rows] @ b[e].to(f32).t()
    y[ids >= len(a)] = float("nan")
    return z, _act_fwd(y, act).to(base.dtype)


def _adapter_grad_cpu(x, a, b, z, scales, ids, y, dy, scale, act):
    f32 = torch.float32
    if act != ACT_NONE:
        dy = _act_bwd_from_out(y.to(f32), dy.to(f32), act).to(dy.dtype)
    dx, da, db = (torch.zeros(t.shape, dtype=f32) for t in (x, a, b))
    for e, rows, s in _adapter_rows(ids, len(a), scales, scale):
        g = dy[rows].to(f32)
        dz = s * (g @ b[e].to(f32))
        dx[rows] = dz @ a[e].to(f32)
        da[e] = dz.t() @ x[rows].to(f32)
        db[e] = g.t() @ z[rows]
    dx[ids >= len(a)] = float("nan")
    return dy, dx.to(x.dtype), da.to(a.dtype), db.to(b.dtype)


def adapter_add(base, x, a, b, ids, scale=1.0, act="none"):
    """act(base + scale * (x A^T) B^T), each row through its own adapter:
    low-rank adapters of many requests beside a shared projection.

    base: [..., outputs], what the projection gave (before its activation);
    x: [..., inputs], what it was given; both are read in place where their
    last axis lies side by side.  a: [adapters, rank, inputs], b: [adapters,
    outputs, rank], all in one type of fp32, bf16 or fp16; sums are 32 bits
    wide and every result is rounded once.  Behind an activation the other
    gradients start from base's, which is rounded to the type and takes the
    slope of the rounded output: a sigmoid's where it is nearly 0 or 1 keeps
    few of its digits in 16 bits.  rank is at most 128, adapters 1024; on a
    GPU rows are less than 2^26.

    ids: one whole number a row (the leading shape of x), or the
    ``adapter_groups`` of them, which the layers of a model share.  A
    negative id is a row without an adapter: act(base).  An id of
    ``adapters`` or more cannot be refused without waiting for the device:
    the row is NaN, and so is its gradient of x.

    scale: a number, or fp32 [adapters].  Gradients flow to base, x, a and
    b; an adapter that no row uses has a gradient of zero.  What is not
    finite in a row or an adapter stays within the rows and the gradients
    that depend on it (an infinity there may come out as NaN).
    """
    act = ACT_CODES[act] if isinstance(act, str) else act
    if act not in (ACT_NONE, ACT_RELU, ACT_SIGMOID):
        raise ValueError("unknown activation code %r" % (act,))
    tensors = (("base", base), ("x", x), ("a", a), ("b", b))
    for name, t in tensors:
        _check_float(name, t)
        if t.dtype != x.dtype or t.device != x.device:
            raise ValueError("%s is %s on %s and x %s on %s" % (
                name, t.dtype, t.device, x.dtype, x.device))
    if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] \
            or a.shape[1] != b.shape[2]:
        raise ValueError("a [adapters, rank, inputs] and b [adapters, "
                         "outputs, rank] do not fit: %s and %s"
                         % (tuple(a.shape), tuple(b.shape)))
    e, r, k = a.shape
    n = b.shape[1]
    if not 1 <= r <= _RANK_MAX or k < 1 or n < 1:
        raise ValueError("rank must be within 1 and %d, and inputs and "
                         "outputs at least 1: %s and %s"
                         % (_RANK_MAX, tuple(a.shape), tuple(b.shape)))
    groups = ids if isinstance(ids, AdapterGroups) else None
    lead = ids.shape
    if x.shape != lead + (k,) or base.shape != lead + (n,):
        raise ValueError("x %s and base %s do not fit ids %s and adapters "
                         "of %d inputs and %d outputs" % (
                             tuple(x.shape), tuple(base.shape), tuple(lead),
                             k, n))
    if ids.device != x.device:
        raise ValueError("x is on %s and ids on %s" % (x.device, ids.device))
    scales = None
    if isinstance(scale, torch.Tensor):
        if scale.requires_grad:
            raise ValueError("scale takes no gradient: detach it")
        if scale.shape != (e,) or scale.dtype != torch.float32 \
                or scale.device != x.device:
            raise ValueError("scale must be a number, or fp32 [%d] beside x"
                             % e)
        scales, scale = scale.contiguous(), 1.0
    else:
        scale = float(scale)
    plan = None
    if groups is None:
        _check_ids(ids, e)
        if ids.dtype != torch.int64:
            ids = ids.long()
    elif groups.adapters != e:
        raise ValueError("ids were grouped for %d adapters, not %d"
                         % (groups.adapters, e))
    else:
        ids, plan = groups.ids, groups.plan
    if ops.use_hip(x):
        return ops.hip.adapter_add_apply(base, x, a, b, scales, scale, ids,
                                         plan, act)
    return _AdapterAddCPU.apply(
        base.reshape(-1, n), x.reshape(-1, k), a, b, scales, scale,
        ids.reshape(-1), act).reshape(base.shape)


def argmax_rows(y: torch.Tensor) -> torch.Tensor:
    """Rowwise argmax prediction head (reference tf.argmax(out, 1))."""
    if ops.use_hip(y):
        return ops.hip.argmax_rows(y)
    return torch.argmax(y, dim=1).to(torch.float32)
