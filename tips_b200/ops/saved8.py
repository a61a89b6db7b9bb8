"""Activations kept for the backward pass in 8 bits (csrc/kernels/saved8.cu).

``pack8(x)`` stores a tensor in 33 bytes per 32 values and ``Packed8.unpack()`` reads it back.  The values of a block of 32
(of the flattened tensor) share a power-of-two step: the least one for which the block's largest magnitude rounds to at
most 127 of them.  A stored value is off by at most half a step, 1/127 of that magnitude; it is exact in fp32 and bf16.  A
value that is not finite comes back as NaN.

``linear(..., save8=True)`` (and ``Linear``, ``BertMLM``) keeps its input and, with GELU, its pre-activation that way instead of
in 16 bits: outputs and the input's gradient path are computed as before, the weight gradient from the stored input and the
activation's derivative from the stored pre-activation.

The reference keeps no activations of its own (it trains TensorFlow models).
"""
from __future__ import annotations

import torch

from . import base

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
BLOCK = 32  # values that share a step


def _check(dtype, what):
    if dtype not in _DTYPES:
        raise TypeError(f"{what} takes float32, bfloat16 or float16, got {dtype}")


def _aligned(x: torch.Tensor) -> torch.Tensor:
    """x, contiguous and starting on 16 bytes."""
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _pack_plain(x: torch.Tensor):
    n = x.numel()
    flat = torch.zeros(-(-n // BLOCK) * BLOCK, dtype=torch.float32)
    flat[:n] = x.reshape(-1)
    flat = flat.view(-1, BLOCK)
    finite = flat.isfinite()
    part, power = torch.frexp(torch.where(finite, flat, 0.0).abs().amax(1, keepdim=True))
    e = (power - 7 + (part * 128 >= 127.5)).clamp(-126, 121)
    e = torch.where(part == 0, torch.full_like(e, -126), e)
    step = ((e + 127) << 23).view(torch.float32)
    q = torch.where(finite, torch.round(flat / step).clamp(-127, 127), -128.0)
    return q.to(torch.int8).view(-1)[:n].clone(), e.to(torch.int8).view(-1)


def _unpack_plain(q: torch.Tensor, e: torch.Tensor, dtype) -> torch.Tensor:
    step = ((e.to(torch.int32) + 127) << 23).view(torch.float32).repeat_interleave(BLOCK)[:q.numel()]
    return torch.where(q == -128, float("nan"), q.float() * step).to(dtype)


def _pack(x: torch.Tensor):
    """(q, e) of a tensor: int8 values and step exponents, flat."""
    if not x.is_cuda:
        return _pack_plain(x)
    x = _aligned(x)
    n = x.numel()
    q = torch.empty(n, dtype=torch.int8, device=x.device)
    e = torch.empty(-(-n // BLOCK), dtype=torch.int8, device=x.device)
    if n:
        with torch.cuda.device(x.device):
            base.check(base.K().tipsk_pack8(x.data_ptr(), q.data_ptr(), e.data_ptr(), n, base.code(x), base.stream()), "pack8")
    return q, e


def _unpack(q: torch.Tensor, e: torch.Tensor, shape, dtype) -> torch.Tensor:
    if not q.is_cuda:
        return _unpack_plain(q, e, dtype).view(shape)
    y = torch.empty(shape, dtype=dtype, device=q.device)
    if y.numel():
        with torch.cuda.device(q.device):
            base.check(base.K().tipsk_unpack8(q.data_ptr(), e.data_ptr(), y.data_ptr(), y.numel(), base.code(y), base.stream()),
                       "unpack8")
    return y


class Packed8:
    """A tensor in 8 bits: `q` (int8, one per value, -128 for NaN), `e` (int8, one per block of 32: the step is 2**e),
    `shape` and `dtype` of what was packed."""

    __slots__ = ("q", "e", "shape", "dtype")

    def __init__(self, q, e, shape, dtype):
        self.q, self.e, self.shape, self.dtype = q, e, torch.Size(shape), dtype

    @property
    def nbytes(self) -> int:
        return self.q.numel() + self.e.numel()

    def unpack(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The stored values, in `dtype` (default: that of the packed tensor).  fp16 rounds values below 2**-14 once more,
        and values beyond its range become infinite."""
        dtype = self.dtype if dtype is None else dtype
        _check(dtype, "unpack")
        return _unpack(self.q, self.e, self.shape, dtype)


def pack8(x: torch.Tensor) -> Packed8:
    """The 8-bit form of a float32, bfloat16 or float16 tensor (any strides; no gradient flows through it)."""
    _check(x.dtype, "pack8")
    x = x.detach()
    return Packed8(*_pack(x), x.shape, x.dtype)


def act_bwd8(dy: torch.Tensor, q, e, bias_dtype=None):
    """(dz, column sums of dz or None) for dy [rows, cols], with dz = dy * gelu'(z) for z stored as (q, e), or dy without them."""
    rows, cols = dy.shape
    if q is None and bias_dtype is None:
        return dy, None
    if dy.is_cuda and cols % 8 == 0 and dy.dtype in _DTYPES and rows and cols:
        dy = _aligned(dy)
        lib = base.K()
        with torch.cuda.device(dy.device):
            dz = None if q is None else torch.empty_like(dy)
            db = part = None
            if bias_dtype is not None:
                db = torch.empty(cols, dtype=bias_dtype, device=dy.device)
                part = torch.empty(lib.tipsk_act_bwd8_parts(rows, cols), cols, dtype=torch.float32, device=dy.device)
                base.count_launches(1)
            base.check(lib.tipsk_act_bwd8(dy.data_ptr(), base.ptr(q), base.ptr(e), base.ptr(dz), base.ptr(db),
                                          0 if db is None else base.code(db), base.ptr(part), rows, cols, base.code(dy),
                                          base.stream()), "act_bwd8")
        return (dy if dz is None else dz), db
    dz = dy.float()
    if q is not None:
        z = _unpack(q, e, dy.shape, torch.float32)
        dz = dz * (0.5 * (1 + torch.erf(z * 0.7071067811865476)) + z * torch.exp(-0.5 * z * z) * 0.3989422804014327)
        dy = dz.to(dy.dtype)
    return dy, None if bias_dtype is None else dz.sum(0).to(bias_dtype)
