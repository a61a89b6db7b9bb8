"""Activations kept for the backward pass in 8 bits (csrc/kernels/saved8.cu).

``pack8(x)`` stores a tensor in 33 bytes per 32 values and ``Packed8.unpack()`` reads it back.  The values of a block of 32
(of the flattened tensor) share a power-of-two step: the least one for which the block's largest magnitude rounds to at
most 127 of them.  A stored value is off by at most half a step (a whole one where fp32's range ends), 1/127 of that
magnitude; it is exact in fp32 and bf16, and read back into the packed tensor's own type it is finite.  A value that is not
finite comes back as NaN.

``linear(..., save8=True)`` (and ``Linear``, ``BertMLM``) keeps its input and, with GELU, its pre-activation that way instead of
in 16 bits: outputs and the input's gradient path are computed as before, the weight gradient from the stored input and the
activation's derivative from the stored pre-activation.

The reference keeps no activations of its own (it trains TensorFlow models).
"""
from __future__ import annotations

import math

import torch

from . import base

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
BLOCK = 32  # values that share a step
_HALF_MAX = torch.finfo(torch.float16).max


def _check(dtype, what):
    if dtype not in _DTYPES:
        raise TypeError(f"{what} takes float32, bfloat16 or float16, got {dtype}")


def _aligned(x: torch.Tensor) -> torch.Tensor:
    """x, contiguous and starting on 16 bytes."""
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _exponents_at(n: int) -> int:
    """Where the exponents start in the buffer of n values: behind them, on 16 bytes."""
    return -(-n // 16) * 16


def _parts(buf: torch.Tensor, n: int):
    """The int8 values and step exponents in a buffer of n values."""
    at = _exponents_at(n)
    return buf[:n], buf[at:at - (-n // BLOCK)]


def _pack_plain(x: torch.Tensor, buf: torch.Tensor) -> None:
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
    values, exponents = _parts(buf, n)
    values.copy_(q.view(-1)[:n])
    exponents.copy_(e.view(-1))


def _unpack_plain(buf: torch.Tensor, n: int, dtype, from_half: bool) -> torch.Tensor:
    q, e = _parts(buf, n)
    step = ((e.to(torch.int32) + 127) << 23).view(torch.float32).repeat_interleave(BLOCK)[:n]
    x = torch.where(q == -128, float("nan"), q.float() * step)
    return (x.clamp(-_HALF_MAX, _HALF_MAX) if from_half and dtype == torch.float16 else x).to(dtype)


def _buffer(n: int, device) -> torch.Tensor:
    """An int8 buffer for the 8-bit form of n values."""
    return torch.empty(_exponents_at(n) - (-n // BLOCK), dtype=torch.int8, device=device)


def _pack(x: torch.Tensor) -> torch.Tensor:
    """The 8-bit form of a tensor as one int8 buffer: the values, and from _exponents_at on a step exponent per block."""
    n = x.numel()
    at = _exponents_at(n)
    buf = _buffer(n, x.device)
    if not x.is_cuda:
        _pack_plain(x, buf)
    elif n:
        x = _aligned(x)
        with base.device_of(x):
            q = buf.data_ptr()
            base.check(base.K().tipsk_pack8(x.data_ptr(), q, q + at, n, base.code(x), base.stream()), "pack8")
    return buf


def _unpack(buf: torch.Tensor, shape, dtype, packed) -> torch.Tensor:
    """The values of a buffer in `dtype`; `packed`: the type of the tensor that was packed.  The largest fp16 values may be stored as
    65536, which fp16 does not have: read back into it they are its largest number, which is within half a step of them as well."""
    from_half = packed == torch.float16
    if not buf.is_cuda:
        return _unpack_plain(buf, math.prod(shape), dtype, from_half).view(shape)
    y = torch.empty(shape, dtype=dtype, device=buf.device)
    n = y.numel()
    if n:
        with base.device_of(y):
            q = buf.data_ptr()
            base.check(base.K().tipsk_unpack8(q, q + _exponents_at(n), y.data_ptr(), n, base.code(y), int(from_half), base.stream()),
                       "unpack8")
    return y


class Packed8:
    """A tensor in 8 bits: `q` (int8, one per value, -128 for NaN), `e` (int8, one per block of 32: the step is 2**e),
    `shape` and `dtype` of what was packed."""

    __slots__ = ("buf", "shape", "dtype")

    def __init__(self, buf, shape, dtype):
        self.buf, self.shape, self.dtype = buf, torch.Size(shape), dtype

    @property
    def q(self) -> torch.Tensor:
        return _parts(self.buf, self.shape.numel())[0]

    @property
    def e(self) -> torch.Tensor:
        return _parts(self.buf, self.shape.numel())[1]

    @property
    def nbytes(self) -> int:
        return self.buf.numel()

    def unpack(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The stored values, in `dtype` (default: that of the packed tensor).  fp16 rounds values below 2**-14 once more; values
        beyond its range become infinite if another type was packed, and its largest number if it was fp16."""
        dtype = self.dtype if dtype is None else dtype
        _check(dtype, "unpack")
        return _unpack(self.buf, self.shape, dtype, self.dtype)


def pack8(x: torch.Tensor) -> Packed8:
    """The 8-bit form of a float32, bfloat16 or float16 tensor (any strides; no gradient flows through it)."""
    _check(x.dtype, "pack8")
    x = x.detach()
    return Packed8(_pack(x), x.shape, x.dtype)


def act_bwd8(dy: torch.Tensor, z: torch.Tensor | None, bias_dtype=None):
    """(dz, column sums of dz or None) for dy [rows, cols], with dz = dy * gelu'(z) for z in 8 bits (the buffer of `_pack`), or
    dy itself without it."""
    rows, cols = dy.shape
    if z is None and bias_dtype is None:
        return dy, None
    if bias_dtype not in (None, *_DTYPES):
        dz, db = act_bwd8(dy, z, torch.float32)
        return dz, db.to(bias_dtype)
    if dy.is_cuda and cols % 8 == 0 and dy.dtype in _DTYPES and rows and cols:
        dy = _aligned(dy)
        lib = base.K()
        with base.device_of(dy):
            dz = None if z is None else torch.empty_like(dy)
            db = part = None
            if bias_dtype is not None:
                db = torch.empty(cols, dtype=bias_dtype, device=dy.device)
                part = torch.empty(lib.tipsk_act_bwd8_parts(rows, cols) * cols, dtype=torch.float32, device=dy.device)
                base.count_launches(1)
            q = base.ptr(z)
            base.check(lib.tipsk_act_bwd8(dy.data_ptr(), q, None if q is None else q + _exponents_at(rows * cols), base.ptr(dz),
                                          base.ptr(db), 0 if db is None else base.code(db), base.ptr(part), rows, cols,
                                          base.code(dy), base.stream()), "act_bwd8")
        return (dy if dz is None else dz), db
    dz = dy.float()
    if z is not None:
        v = _unpack(z, dy.shape, torch.float32, dy.dtype)
        dz = dz * (0.5 * (1 + torch.erf(v * 0.7071067811865476)) + v * torch.exp(-0.5 * v * v) * 0.3989422804014327)
        dy = dz.to(dy.dtype)
    return dy, None if bias_dtype is None else dz.sum(0).to(bias_dtype)
