"""Activations kept in 8 bits between the forward and the backward pass.

``keep8(x)`` writes the 8-bit copy of a tensor, ``restore8(kept)`` reads it back: 1.0625 bytes per element instead of 2
(or 4). 16 elements that follow one another in memory share a power of two ``2^e``, the smallest one (``e`` at least
-126) with ``max |x| < 126.5 * 2^e``; each is kept as the whole number nearest to ``x / 2^e`` (a tie goes to the even
one), so a restored value is off by at most half a step: ``max |x| / 126`` of its block, or ``2^-127`` in blocks so small
that ``e`` is -126 (a block below that comes back as zeros). A block with an infinity or a NaN is restored as
NaN: an overflow shows. A value that would be restored beyond its type's largest number is kept as 63 steps, so what was
finite stays so; it is off by less than a step then.

A kept tensor is what a layer stores for its backward pass; no gradient flows through the copy. The layers of
:mod:`scaffold_b200.ops` use it when they are told to (``UNet.keep_activations(bits=8)``).

On CUDA the copy is made by ``csrc/kept8.cu`` on the current stream; on the CPU by the formula, with the same bits.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Tuple

import torch

from . import _lib
from .layout import on_device

_lib.register("sb_kept8_bytes", [C.c_longlong], C.c_longlong)
_lib.register("sb_keep8", [C.c_void_p, C.c_int, C.c_longlong, C.c_void_p, C.c_void_p])
_lib.register("sb_restore8", [C.c_void_p, C.c_int, C.c_longlong, C.c_void_p, C.c_void_p])

BLOCK = 16
KINDS = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class Kept8(NamedTuple):
    """An 8-bit copy: ``data`` (uint8, on the tensor's device) holds the whole numbers of all blocks, then one exponent
    byte per block; the rest says what :func:`restore8` makes of it."""

    data: torch.Tensor
    shape: Tuple[int, ...]
    stride: Tuple[int, ...]
    dtype: torch.dtype

    @property
    def device(self) -> torch.device:
        return self.data.device

    def numel(self) -> int:
        return math.prod(self.shape)


def kept_bytes(numel: int) -> int:
    """Bytes of the copy of ``numel`` elements."""
    return (numel + BLOCK - 1) // BLOCK * (BLOCK + 1)


def _dense(x: torch.Tensor) -> bool:
    """True when ``x`` covers one run of memory, every element once (channels-last tensors too)."""
    if x.is_contiguous() or (x.dim() == 5 and x.is_contiguous(memory_format=torch.channels_last_3d)):
        return True
    expected = 1
    for stride, size in sorted((st, s) for s, st in zip(x.shape, x.stride()) if s != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def keep8(x: torch.Tensor) -> Kept8:
    """The 8-bit copy of a bf16, fp16 or fp32 tensor of any shape. Blocks follow the tensor's memory; a tensor that does
    not cover one run of memory (a slice, an expanded view) is copied to one first, in the order of its indices."""
    dtype, shape = x.dtype, x.shape
    if dtype not in KINDS:
        raise TypeError(f"keep8 takes bf16, fp16 or fp32; got {dtype}")
    if x.layout != torch.strided or x.is_conj() or x.is_neg():
        raise TypeError("keep8 takes plain strided tensors")
    if not _dense(x):
        x = x.detach().contiguous()
    n = x.numel()
    if not x.is_cuda:
        return Kept8(_keep_formula(x.detach().as_strided((n,), (1,), x.storage_offset())), tuple(x.shape), x.stride(), x.dtype)
    dev = x.device
    with on_device(dev):
        data = x.new_empty(kept_bytes(n), dtype=torch.uint8)
        _lib.check(_lib.lib().sb_keep8(x.data_ptr(), KINDS[dtype], n, data.data_ptr(), _lib.stream_ptr()), "sb_keep8")
    return Kept8(data, tuple(shape), x.stride(), dtype)


def restore8(kept: Kept8) -> torch.Tensor:
    """The tensor that ``kept`` is a copy of, in its type, shape and memory format."""
    n = kept.numel()
    data = kept.data
    if kept.dtype not in KINDS:
        raise TypeError(f"restore8 makes bf16, fp16 or fp32; got {kept.dtype}")
    if data.dtype != torch.uint8 or data.numel() != kept_bytes(n) or not data.is_contiguous():
        raise ValueError(f"an 8-bit copy of {n} elements is {kept_bytes(n)} contiguous bytes; got "
                         f"{data.numel()} of {data.dtype}")
    dev = data.device
    y = torch.empty_strided(kept.shape, kept.stride, dtype=kept.dtype, device=dev)
    if not _dense(y):
        raise ValueError(f"strides {kept.stride} of shape {kept.shape} do not cover one run of memory")
    if not data.is_cuda:
        y.as_strided((n,), (1,)).copy_(_restore_formula(data, n, kept.dtype))
        return y
    with on_device(dev):
        _lib.check(_lib.lib().sb_restore8(data.data_ptr(), KINDS[kept.dtype], n, y.data_ptr(), _lib.stream_ptr()),
                   "sb_restore8")
    return y


# -- the formula (CPU, and the oracle of the GPU tests) -------------------------------------------------------------------
def block_steps(x: torch.Tensor, dtype: torch.dtype):
    """(exponent bytes, steps 2^e, largest whole numbers) of fp32 blocks ``[blocks, 16]`` of a tensor of ``dtype``."""
    most = x.abs().amax(1)  # a NaN stays one
    bad = ~torch.isfinite(most)
    m, k = torch.frexp(torch.where(bad, 0.0, most))
    e = torch.where(m * 128 < 126.5, k - 7, k - 6).clamp_min(-126)
    step = ((e + 127).int() << 23).view(torch.float32)
    cap = torch.where(64.0 * step.double() > torch.finfo(dtype).max, 63.0, 127.0)
    return torch.where(bad, 255, e + 127).to(torch.uint8), step, cap


def _keep_formula(flat: torch.Tensor) -> torch.Tensor:
    n, dtype = flat.numel(), flat.dtype
    blocks = (n + BLOCK - 1) // BLOCK
    x = torch.zeros(blocks * BLOCK, dtype=torch.float32, device=flat.device)
    x[:n] = flat
    x = x.view(blocks, BLOCK)
    exps, step, cap = block_steps(x, dtype)
    q = torch.round(x / step[:, None])
    q = torch.where((exps == 255)[:, None], 0.0, torch.minimum(torch.maximum(q, -cap[:, None]), cap[:, None]))
    return torch.cat([q.to(torch.int8).view(torch.uint8).reshape(-1), exps])


def _restore_formula(data: torch.Tensor, n: int, dtype: torch.dtype) -> torch.Tensor:
    blocks = (n + BLOCK - 1) // BLOCK
    q = data[:blocks * BLOCK].view(torch.int8).float().view(blocks, BLOCK)
    exps = data[blocks * BLOCK:].int()
    step = torch.where(exps == 255, float("inf"), (exps << 23).view(torch.float32))  # 0 * inf = NaN
    return (q * step[:, None]).reshape(-1)[:n].to(dtype)
