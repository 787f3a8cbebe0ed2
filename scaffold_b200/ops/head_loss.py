"""Cross entropy of a head with many classes, taken from the features in front of it.

``head_cross_entropy(features, weight, bias, labels)`` is the class-weighted mean cross entropy
(:func:`scaffold_b200.ops.loss.sharded_cross_entropy`) of ``features @ weight.T + bias``, with its gradients, without the
logits: a head of some hundred classes over a 128-cubed volume would keep gigabytes of them, several times over. The fused
segmentation loss keeps a voxel's classes in registers and ends at 32 classes; this one has no limit on the classes.

On CUDA with bf16 features (or under bf16 autocast) the kernels of ``csrc/head_loss.cu`` and ``csrc/head_wide.cu``
multiply features and weight tile by tile: once for the loss, and once more for both gradients together or, where one
kernel does not hold both, for each; other tensors take the PyTorch formula.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .layout import on_device, use_cuda_kernels

_P = C.c_void_p


_lib.register("sb_head_bytes", [C.c_int, C.c_longlong, C.c_int, C.c_int, C.c_int], C.c_longlong)
_lib.register("sb_head_forward", [_P, _P, _P, C.c_int, _P, C.c_int, C.c_int, C.c_longlong, _P, C.c_longlong, C.c_int,
                                  C.c_int, _P, _P, _P, _P, _P])
_lib.register("sb_head_total", [_P, _P, _P])
_lib.register("sb_head_backward", [_P, _P, _P, C.c_longlong, C.c_int, C.c_int, _P, _P, _P, _P, _P, C.c_int, _P, C.c_int,
                                   _P, _P])

_lib.register("sb_head_predict_bytes", [C.c_longlong, C.c_int, C.c_int], C.c_longlong)
_lib.register("sb_head_predict", [_P, _P, _P, C.c_int, C.c_longlong, C.c_int, C.c_int, _P, _P, _P, _P])

_LABEL_KIND = {torch.int16: 2, torch.int32: 4, torch.int64: 8}
_KIND = {torch.bfloat16: 0, torch.float32: 2}
MAX_WIDTH = 32768


def head_supported(width: int) -> bool:
    """Feature widths of the kernels."""
    return 8 <= width <= MAX_WIDTH and width % 8 == 0


@functools.lru_cache(maxsize=256)
def _bytes(v: int, k: int, c: int, weighted: bool):
    """Bytes of the state, of the forward pass's scratch and of the backward pass's: for one gradient, for both."""
    out = tuple(_lib.lib().sb_head_bytes(what, v, k, c, weighted) for what in range(4))
    if min(out) < 0:
        raise _lib.NativeError(f"sb_head_bytes refused {v} voxels, {k} classes, width {c}")
    return out


class _HeadLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, labels, cw, ignore, spatial):
        """x [V, C] bf16, weight [K, C], both contiguous."""
        dev = x.device
        w16 = weight if weight.dtype == torch.bfloat16 else weight.to(torch.bfloat16)
        v, c = x.shape
        k = w16.shape[0]
        n_state, n_scratch, *_ = _bytes(v, k, c, cw is not None)
        state = x.new_empty(n_state, dtype=torch.uint8)
        scratch = state.new_empty(n_scratch)
        loss = x.new_empty((), dtype=torch.float32)
        st = _lib.stream_ptr()
        _lib.check(_lib.lib().sb_head_forward(
            x.data_ptr(), w16.data_ptr(), _lib.ptr(bias), 0 if bias is None else _KIND[bias.dtype], labels.data_ptr(),
            _LABEL_KIND[labels.dtype], ignore is not None, ignore or 0, _lib.ptr(cw), v, k, c, state.data_ptr(),
            scratch.data_ptr(), loss.data_ptr(), _lib.status_tensor(dev).data_ptr(), st), "sb_head_forward")
        if spatial is not None and spatial.size > 1:
            spatial.all_reduce_sum(state[:16].view(torch.float64))
            _lib.check(_lib.lib().sb_head_total(state.data_ptr(), loss.data_ptr(), st), "sb_head_total")
        ctx.save_for_backward(x, w16, state, cw)
        ctx.types = weight.dtype, None if bias is None else bias.dtype
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, gout):
        x, w16, state, cw = ctx.saved_tensors
        dev = x.device
        v, c = x.shape
        k = w16.shape[0]
        w_type, b_type = ctx.types
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        gout = gout.float()
        with on_device(dev):
            dx = torch.empty_like(x) if want_x else None
            dw = torch.empty_like(w16, dtype=w_type) if want_w else None
            db = w16.new_empty(k, dtype=b_type) if want_b else None
            scratch = state.new_empty(_bytes(v, k, c, cw is not None)[3 if want_x and (want_w or want_b) else 2])
            _lib.check(_lib.lib().sb_head_backward(
                x.data_ptr(), w16.data_ptr(), _lib.ptr(cw), v, k, c, state.data_ptr(), scratch.data_ptr(), gout.data_ptr(),
                _lib.ptr(dx), _lib.ptr(dw), _KIND[w_type], _lib.ptr(db), _KIND[b_type] if want_b else 0,
                _lib.status_tensor(dev).data_ptr(), _lib.stream_ptr()), "sb_head_backward")
        return dx, dw, db, None, None, None, None


def head_cross_entropy(features: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], labels: torch.Tensor,
                       class_weights: Optional[torch.Tensor] = None, ignore_label: Optional[int] = None,
                       spatial=None) -> torch.Tensor:
    """The cross entropy of ``features @ weight.T + bias`` against ``labels``, as an fp32 scalar.

    ``features [..., C]`` (voxel-major, the classes' axis of the logits is the last), ``weight [K, C]`` (or the
    ``[K, C, 1, 1, 1]`` of a 1x1x1 convolution), ``bias [K]`` or None, ``labels [...]`` int16, int32 or int64.
    ``class_weights [K]`` (not negative) weigh the voxels by their label; the result is the sum of the weighted terms over
    the sum of the weights, over all shards with ``spatial``. Voxels of ``ignore_label`` and of a class whose weight is zero
    take no part; without any other voxel the loss and its gradients are zero. A bias of -inf turns its class off; a voxel
    that is labelled with it makes the loss +inf. A label outside the classes takes no part either and is reported by
    :func:`scaffold_b200.ops._lib.check_status`. Features of voxels that take no part have to be finite for the
    kernels: they reach the weight's gradient as ``0 * x``, as in any matrix product with rows of zeros.

    The kernels read bf16: an fp32 ``weight`` is rounded, its gradient comes back in fp32. Logits, log-sum-exp and all sums
    are fp32; the entries of ``softmax - onehot`` (and with ``class_weights`` the weighted features) are rounded to bf16 for
    the gradients' products, except in calls of few voxels, where one rounding could make up a result. A feature of a voxel
    that takes part which is infinite or NaN makes the loss NaN. Gradients: features in bf16,
    weight and bias in their own types; the class weights have none.
    """
    shape = features.shape
    if not shape or labels.shape != shape[:-1]:
        raise ValueError(f"features {tuple(shape)} need labels {tuple(shape[:-1])}; got {tuple(labels.shape)}")
    if labels.dtype not in _LABEL_KIND:
        raise TypeError(f"labels must be int16, int32 or int64; got {labels.dtype}")
    if ignore_label is not None and not -2 ** 63 <= ignore_label < 2 ** 63:
        raise ValueError(f"ignore_label {ignore_label} is no 64-bit number")
    weight = _check(features, weight, bias=bias, class_weights=class_weights, labels=labels)
    if not use_cuda_kernels(features):
        return _formula(features, weight, bias, labels, class_weights, ignore_label, spatial)
    x, weight = _operands(features, weight, bias)
    if labels.dim() != 1 or not labels.is_contiguous():
        labels = labels.reshape(-1).contiguous()
    if class_weights is not None and (class_weights.dtype != torch.float32 or class_weights.requires_grad
                                      or not class_weights.is_contiguous()):
        class_weights = class_weights.detach().float().contiguous()
    if x.shape[0] == 0:
        # a shard without voxels: its terms are zero, the other shards' sums are not, and are two fp64 numbers
        return _formula(x.double(), weight.double(), None if bias is None else bias.double(), labels, class_weights,
                        ignore_label, spatial).float()
    with on_device(x.device):
        return _HeadLossFn.apply(x, weight, None if bias is None else bias.contiguous(), labels, class_weights,
                                 ignore_label, spatial)


def head_predict(features: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The class of the largest of the logits ``features @ weight.T + bias`` (the lowest of several; a NaN is the
    largest), as int64 ``[...]``, without the logits. Arguments as for :func:`head_cross_entropy`; no gradients."""
    if not features.shape:
        raise ValueError("features need a channel axis")
    weight = _check(features, weight, bias=bias)
    with torch.no_grad():
        if not use_cuda_kernels(features):
            return _logits(features.reshape(-1, features.shape[-1]), weight, bias).argmax(1).view(features.shape[:-1])
        x, weight = _operands(features, weight, bias)
        out = torch.empty(features.shape[:-1], dtype=torch.int64, device=x.device)
        (v, c), k = x.shape, weight.shape[0]
        if v == 0:
            return out
        with on_device(x.device):
            w16 = weight.to(torch.bfloat16)
            bias = None if bias is None else bias.contiguous()
            scratch = torch.empty(_lib.lib().sb_head_predict_bytes(v, k, c), dtype=torch.uint8, device=x.device)
            _lib.check(_lib.lib().sb_head_predict(
                x.data_ptr(), w16.data_ptr(), _lib.ptr(bias), 0 if bias is None else _KIND[bias.dtype], v, k, c,
                scratch.data_ptr(), out.data_ptr(), _lib.status_tensor(x.device).data_ptr(), _lib.stream_ptr()),
                "sb_head_predict")
    return out


def _check(features, weight, **others) -> torch.Tensor:
    """The weight as [classes, channels], after checks of shapes and devices."""
    c, dev = features.shape[-1], features.device
    k = weight.shape[0] if weight.dim() else 0
    if weight.dim() < 2 or k < 1 or weight.shape[1] != c or weight.numel() != k * c:
        raise ValueError(f"weight must be [classes, {c}] (or [classes, {c}, 1, 1, 1]); got {tuple(weight.shape)}")
    if weight.device != dev:
        raise ValueError(f"weight is on {weight.device}, the features are on {dev}")
    for name, t in others.items():
        if t is not None and name != "labels" and t.shape != (k,):
            raise ValueError(f"{name} must be [{k}]; got {tuple(t.shape)}")
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, the features are on {dev}")
    return weight if weight.dim() == 2 else weight.reshape(k, c)


def _operands(features, weight, bias):
    """(features [V, C] in bf16, weight) as the kernels read them: contiguous, on 16 bytes (a tensor map starts there)."""
    c = features.shape[-1]
    if not head_supported(c):
        raise ValueError(f"the kernels read features of 8 to {MAX_WIDTH} channels in multiples of 8; got {c}")
    if weight.dtype not in _KIND or (bias is not None and bias.dtype not in _KIND):
        raise TypeError("weight and bias must be bf16 or fp32")
    n = features.numel() // c
    if n > 2 ** 31 - 1024:
        raise ValueError(f"{n} voxels are more than the kernels count")
    x = features if features.dtype == torch.bfloat16 else features.to(torch.bfloat16)
    if x.dim() != 2:
        x = x.reshape(n, c)
    if not x.is_contiguous() or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    if not weight.is_contiguous() or (weight.dtype == torch.bfloat16 and weight.data_ptr() % 16):
        weight = weight.clone(memory_format=torch.contiguous_format)
    return x, weight


def _logits(x, weight, bias):
    kind = torch.promote_types(torch.promote_types(x.dtype, weight.dtype), torch.float32)
    with torch.autocast(x.device.type, enabled=False):  # which would make a product of 16 bits of it
        logits = x.to(kind) @ weight.to(kind).T
    return logits if bias is None else logits + bias.to(kind)


def _formula(features, weight, bias, labels, class_weights, ignore_label, spatial):
    """The definition: the CPU path, and the oracle of the GPU tests in 64 bits."""
    from .loss import spatial_all_reduce
    k = weight.shape[0]
    y = labels.reshape(-1).long()
    live = (y >= 0) & (y < k)
    if ignore_label is not None:
        live &= y != ignore_label
    if class_weights is not None:
        class_weights = class_weights.detach()
        live &= class_weights[y.clamp(0, k - 1)] != 0
    x, y = features.reshape(-1, features.shape[-1])[live], y[live]
    logits = _logits(x, weight, bias)
    kind = logits.dtype
    u = torch.ones(len(y), dtype=kind, device=y.device) if class_weights is None else class_weights.to(kind)[y]
    nll = torch.logsumexp(logits, 1) - logits.gather(1, y[:, None])[:, 0]
    total = spatial_all_reduce(torch.stack([(u * nll).sum(), u.sum()]), spatial)
    return total[0] / total[1].detach().clamp_min(torch.finfo(torch.float32).eps)
