"""Linear layers on the tcgen05 GEMM (csrc/kernels/gemm_tcgen05.cu).

``gemm_tn(a, b)`` computes ``a @ b.T`` for bf16 row-major ``a [M,K]`` and ``b [N,K]`` with the bias
and activation fused into the epilogue.  ``Linear`` builds forward and backward from it:

    y  = act(x W^T + b)                      gemm_tn(x, W)
    dz = dy * act'(.) ; db = colsum(dz)      one pass (bias_act_bwd kernel)
    dx = dz W                                gemm_nn(dz, W): W is read in place as an MN-major operand
    dW = dz^T x                              the same GEMM with both operands MN-major (dz and x as they are); transposed
                                             copies only for feature counts that are not multiples of 64; fp32
                                             gradients come from the weight-gradient kernel of conv_tcgen05.cu

The reference has no GEMM or linear layer; this serves the CTR MLP and the BERT-shaped encoder.
CPU tensors (host-only tests) and shapes the kernel does not take (row strides that are not a
multiple of 16 bytes) use torch.matmul.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import base, saved8

_ACT = {None: 0, "none": 0, "relu": 1, "gelu": 2}


def _supported(a: torch.Tensor, b: torch.Tensor) -> bool:
    return (a.is_cuda and a.dtype == torch.bfloat16 and b.dtype == torch.bfloat16 and a.dim() == 2 and b.dim() == 2
            and a.stride(1) == 1 and b.stride(1) == 1 and a.stride(0) % 8 == 0 and b.stride(0) % 8 == 0
            and a.data_ptr() % 16 == 0 and b.data_ptr() % 16 == 0)


def _split(kind, a, b, c, bias, pre, m, n, k, act, accumulate) -> bool:
    """Run the product with its contraction split over idle SMs when it has few output tiles and a long K; False when
    the unsplit kernels are to take it.  The fp32 partial products live in a workspace of this call."""
    lib = base.K()
    splits = lib.tipsk_gemm_splits(m, n, k)
    if splits <= 1:
        return False
    partial = torch.empty(splits * m * n, dtype=torch.float32, device=c.device)
    base.check(lib.tipsk_gemm_bf16_split(kind, a.data_ptr(), b.data_ptr(), c.data_ptr(), base.ptr(bias), base.ptr(pre),
                                         partial.data_ptr(), splits, m, n, k, a.stride(0), b.stride(0), n, act,
                                         int(accumulate), base.stream()), "gemm_bf16_split")
    base.count_launches(1)
    return True


def gemm_tn(a, b, bias=None, act=None, want_pre=False):
    """act(a @ b.T + bias). Returns y, or (y, pre_activation) when want_pre."""
    code = _ACT[act]
    m, k = a.shape
    n = b.shape[0]
    assert b.shape[1] == k
    if not _supported(a, b):
        pre = a.float() @ b.float().t()
        if bias is not None:
            pre = pre + bias.float()
        y = F.relu(pre) if code == 1 else F.gelu(pre) if code == 2 else pre
        y = y.to(a.dtype)
        return (y, pre.to(a.dtype)) if want_pre else y
    c = torch.empty(m, n, dtype=torch.bfloat16, device=a.device)
    pre = torch.empty_like(c) if want_pre else None
    bb = None if bias is None else bias.to(torch.bfloat16).contiguous()
    if _split(0, a, b, c, bb, pre, m, n, k, code, False):
        return (c, pre) if want_pre else c
    base.check(base.K().tipsk_gemm_bf16(a.data_ptr(), b.data_ptr(), c.data_ptr(), base.ptr(bb), base.ptr(pre), m, n, k,
                                        a.stride(0), b.stride(0), n, code, base.stream()), "gemm_bf16")
    return (c, pre) if want_pre else c


def gemm_nn(a: torch.Tensor, b: torch.Tensor, into: torch.Tensor | None = None) -> torch.Tensor:
    """a @ b for bf16 row-major a [M,K] and b [K,N]: b is read in place as an MN-major operand.  With `into`
    (a contiguous [M,N] bf16 tensor) the product is added to it by the kernel's reduce-add stores."""
    m, k = a.shape
    n = b.shape[1]
    assert b.shape[0] == k
    if not (_supported(a, b) and n >= 64 and n % 8 == 0):
        c = gemm_tn(a, b.t().contiguous())
        return c if into is None else into.add_(c)
    if into is not None:
        assert into.shape == (m, n) and into.is_contiguous() and into.dtype == torch.bfloat16
        c = into
    else:
        c = torch.empty(m, n, dtype=torch.bfloat16, device=a.device)
    if _split(1, a, b, c, None, None, m, n, k, 0, into is not None):
        return c
    base.check(base.K().tipsk_gemm_bf16_nn(a.data_ptr(), b.data_ptr(), c.data_ptr(), m, n, k, a.stride(0), b.stride(0),
                                           n, 0 if into is None else 1, base.stream()), "gemm_bf16_nn")
    return c


def _weight_grad(dz: torch.Tensor, x2: torch.Tensor, dtype: torch.dtype | None = None) -> torch.Tensor:
    """dz^T @ x2 as [N, K], in fp32 or, with dtype=torch.bfloat16, rounded once from the fp32 accumulators.  Both
    operands are read in place (MN-major)."""
    m, n = dz.shape
    k = x2.shape[1]
    if (dz.is_cuda and dz.dtype == torch.bfloat16 and x2.dtype == torch.bfloat16 and n % 64 == 0 and k % 64 == 0
            and m >= 16 and dz.is_contiguous() and x2.is_contiguous()
            and dz.data_ptr() % 16 == 0 and x2.data_ptr() % 16 == 0):
        if dtype == torch.bfloat16 and base.K().tipsk_gemm_prefers_pair(2, n, k, m):
            dw = torch.empty(n, k, dtype=torch.bfloat16, device=dz.device)
            if not _split(2, dz, x2, dw, None, None, n, k, m, 0, False):
                base.check(base.K().tipsk_gemm_bf16_tt(dz.data_ptr(), x2.data_ptr(), dw.data_ptr(), n, k, m, n, k, k,
                                                       base.stream()), "gemm_bf16_tt")
            return dw
        # the convolution's weight-gradient kernel (a linear layer is a 1x1 convolution over "pixels" = rows)
        dw = torch.empty(n, k, dtype=torch.float32, device=dz.device)
        base.check(base.K().tipsk_conv2d_wgrad(x2.data_ptr(), dz.data_ptr(), dw.data_ptr(), 1, 1, m, k, n, 1, 1, 1, 0,
                                               base.stream()), "linear_wgrad")
        return dw
    return gemm_tn(dz.t().contiguous(), x2.t().contiguous())


def gemm_status() -> int:
    """0 when no GEMM launch since the last call reported a bounded-wait timeout (waits for all streams of the device)."""
    lib = base.K()
    return int(lib.tipsk_gemm_status()) or int(lib.tipsk_conv_status())  # the weight gradient runs on the conv kernels


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, act):
        x2 = x.reshape(-1, x.shape[-1])
        if not x2.is_contiguous():
            x2 = x2.contiguous()
        code = _ACT[act]
        if code == 2:
            y, pre = gemm_tn(x2, weight, bias, act, want_pre=True)
        else:
            y, pre = gemm_tn(x2, weight, bias, act), None
        ctx.save_for_backward(x2, weight, y if code == 1 else pre, bias)
        ctx.act = code
        ctx.in_shape = x.shape
        return y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    def backward(ctx, dy):
        return _linear_backward(ctx, dy, None)


def _linear8_fits(x2: torch.Tensor, weight: torch.Tensor) -> bool:
    """Whether the layer runs as one call per pass."""
    n, k = weight.shape
    return _supported(x2, weight) and n >= 64 and k >= 64 and n % 8 == 0 and k % 8 == 0 and x2.shape[0] > 0


def _linear8_forward(x2, weight, bias, act, want_x8, want_pre8):
    """(act(x2 @ weight.T + bias), x2 in 8 bits, the value before the activation in 8 bits) with None for what is not wanted."""
    m, k = x2.shape
    n = weight.shape[0]
    if not _linear8_fits(x2, weight):
        y = gemm_tn(x2, weight, bias, act, want_pre=want_pre8)
        y, pre8 = (y[0], saved8._pack(y[1])) if want_pre8 else (y, None)
        return y, saved8._pack(x2) if want_x8 else None, pre8
    lib = base.K()
    with base.device_of(x2):
        y = torch.empty(m, n, dtype=torch.bfloat16, device=x2.device)
        x8 = saved8._buffer(m * k, x2.device) if want_x8 else None
        pre8 = saved8._buffer(m * n, x2.device) if want_pre8 else None
        bb = None if bias is None else bias.to(torch.bfloat16).contiguous()
        need = lib.tipsk_linear8_fwd_ws(m, n, k, int(want_pre8))
        ws = torch.empty(need, dtype=torch.uint8, device=x2.device) if need else None
        base.check(lib.tipsk_linear8_fwd(x2.data_ptr(), weight.data_ptr(), base.ptr(bb), y.data_ptr(), base.ptr(x8), base.ptr(pre8),
                                         base.ptr(ws), m, n, k, weight.stride(0), _ACT[act], base.stream()), "linear8_fwd")
    base.count_launches(int(want_x8) + int(want_pre8))
    return y, x8, pre8


class _Linear8Fn(torch.autograd.Function):
    """linear(x) that keeps x and, with GELU, the value before the activation in 8 bits (ops/saved8.py).  `grad`: whether a backward
    pass can follow, which needs_input_grad does not tell (it is set for parameters without a grad mode as well)."""

    @staticmethod
    def forward(ctx, x, weight, bias, act, grad):
        x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
        if not x2.is_contiguous():
            x2 = x2.contiguous()
        need = [grad and n for n in ctx.needs_input_grad[:3]]
        y, x8, pre8 = _linear8_forward(x2, weight, bias, act, need[1], _ACT[act] == 2 and (need[0] or need[1] or need[2]))
        ctx.save_for_backward(weight, x8, pre8)
        ctx.x_dtype, ctx.bias_dtype = x.dtype, None if bias is None else bias.dtype
        ctx.in_shape = x.shape
        return y if x.dim() == 2 else y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @base.once_differentiable
    def backward(ctx, dy):
        return _linear8_backward(ctx, dy, None)


def _linear8_backward(ctx, dy, d_alias):
    weight, x8, pre8 = ctx.saved_tensors  # pre8: None without an activation
    n, k = weight.shape
    dz = dy if dy.dim() == 2 else dy.reshape(-1, n)
    if not dz.is_contiguous():
        dz = dz.contiguous()
    want_dx, want_dw = ctx.needs_input_grad[:2]
    want_db = ctx.bias_dtype if ctx.needs_input_grad[2] else None
    m = dz.shape[0]
    if not (_linear8_fits(dz, weight) and weight.dtype == ctx.x_dtype and want_db in (None, *saved8._DTYPES)):
        dz, db = saved8.act_bwd8(dz, pre8, want_db)
        dx = _input_grad(dz, weight, d_alias).view(ctx.in_shape) if want_dx else None
        dw = None
        if want_dw:
            dw = _weight_grad8(dz, saved8._unpack(x8, (m, k), ctx.x_dtype, ctx.x_dtype), weight.dtype).to(weight.dtype)
        return dx, dw, db, None, None
    lib = base.K()
    with base.device_of(dz):
        into = _accumulator(d_alias, k, dz) if want_dx else None
        dx = (torch.empty(m, k, dtype=torch.bfloat16, device=dz.device) if into is None else into) if want_dx else None
        dw = torch.empty(n, k, dtype=torch.bfloat16, device=dz.device) if want_dw else None
        db = torch.empty(n, dtype=want_db, device=dz.device) if want_db is not None else None
        need = lib.tipsk_linear8_bwd_ws(m, n, k, int(pre8 is not None), int(want_dw), int(db is not None))
        ws = torch.empty(need, dtype=torch.uint8, device=dz.device) if need else None
        base.check(lib.tipsk_linear8_bwd(dz.data_ptr(), weight.data_ptr(), base.ptr(x8), base.ptr(pre8), base.ptr(dx), base.ptr(dw),
                                         base.ptr(db), 0 if db is None else base.code(db), base.ptr(ws), m, n, k, weight.stride(0),
                                         int(into is not None), base.stream()), "linear8_bwd")
    base.count_launches(int(pre8 is not None or want_db is not None) + int(want_db is not None) + int(want_dx) + 2 * int(want_dw) - 1)
    return dx if dx is None or len(ctx.in_shape) == 2 else dx.view(ctx.in_shape), dw, db, None, None


class _Linear8PassFn(torch.autograd.Function):
    """_LinearPassFn with the activations in 8 bits."""

    @staticmethod
    def forward(ctx, x, weight, bias, act, grad):
        y = _Linear8Fn.forward(ctx, x, weight, bias, act, grad)
        return y, x.detach()

    @staticmethod
    @base.once_differentiable
    def backward(ctx, dy, d_alias):
        return _linear8_backward(ctx, dy, d_alias)


def _weight_grad8(dz: torch.Tensor, x2: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """dz^T @ x2 where the layer does not run as one call: `_weight_grad` where it reads both operands in place, and otherwise
    transposed copies, whose rows are filled up with zeros to the whole 16 bytes that the GEMM reads."""
    m, n = dz.shape
    k = x2.shape[1]
    if not (dz.is_cuda and dz.dtype == x2.dtype == torch.bfloat16 and m) or (n % 64 == 0 and k % 64 == 0 and m >= 16):
        return _weight_grad(dz, x2, dtype)
    pad = -m % 8
    return gemm_tn(F.pad(dz.t(), (0, pad)).contiguous(), F.pad(x2.t(), (0, pad)).contiguous())


def _accumulator(d_alias: torch.Tensor | None, k: int, dz: torch.Tensor) -> torch.Tensor | None:
    """The gradient of another consumer of a layer's input as a matrix that the GEMM can add to, while it reads dz."""
    if d_alias is None:
        return None
    into = d_alias.reshape(-1, k)
    # a sum of the layer's output and its input hands both the same gradient
    if not (into.is_contiguous() and into.data_ptr() % 16 == 0) or into.untyped_storage().data_ptr() == dz.untyped_storage().data_ptr():
        into = into.clone(memory_format=torch.contiguous_format)
    return into


def _input_grad(dz: torch.Tensor, weight: torch.Tensor, d_alias: torch.Tensor | None) -> torch.Tensor:
    """dz @ weight as [rows, k]; with `d_alias` (the gradient of another consumer of the input) added into it by the GEMM."""
    return gemm_nn(dz, weight, into=_accumulator(d_alias, weight.shape[1], dz))


def _linear_backward(ctx, dy, d_alias):
    """Gradients of the fused linear layer; `d_alias` (optional) is the gradient of another consumer of x, into
    which dx is accumulated inside the GEMM."""
    x2, weight, saved, bias = ctx.saved_tensors
    n = weight.shape[0]
    dy2 = dy.reshape(-1, n)
    if not dy2.is_contiguous():
        dy2 = dy2.contiguous()
    dbias = None
    vec_ok = (n * dy2.element_size()) % 16 == 0  # the fused kernel works on 16-byte column vectors
    if dy2.is_cuda and vec_ok:
        dz = dy2
        db = torch.empty(n, dtype=torch.float32, device=dy2.device) if bias is not None else None
        if ctx.act != 0 or db is not None:
            if ctx.act != 0:
                dz = torch.empty_like(dy2)
            # ReLU: the mask of y equals the mask of the pre-activation, so y stands in for it.
            base.check(base.K().tipsk_bias_act_bwd(dy2.data_ptr(), base.ptr(saved) if ctx.act != 0 else None, None,
                                                   dz.data_ptr() if ctx.act != 0 else None, base.ptr(db),
                                                   dy2.shape[0], n, ctx.act, base.code(dy2), base.stream()),
                       "bias_act_bwd")
        if db is not None:
            dbias = db.to(bias.dtype)
    else:
        if ctx.act == 1:
            dz = dy2 * (saved > 0).to(dy2.dtype)
        elif ctx.act == 2:
            s = saved.float()
            dz = (dy2.float() * (0.5 * (1 + torch.erf(s / math.sqrt(2))) + s * torch.exp(-0.5 * s * s) / math.sqrt(2 * math.pi))).to(dy2.dtype)
        else:
            dz = dy2
        if bias is not None:
            dbias = dz.float().sum(0).to(bias.dtype)
    dx = dw = None
    if ctx.needs_input_grad[0]:
        dx = _input_grad(dz, weight, d_alias).view(ctx.in_shape)
    if ctx.needs_input_grad[1]:
        dw = _weight_grad(dz, x2, weight.dtype).to(weight.dtype)
    return dx, dw, dbias, None


class _LinearPassFn(torch.autograd.Function):
    """linear(x) together with an alias of x for the other consumers of x (a residual connection): the backward pass
    adds dx into the gradient of that alias inside the GEMM (reduce-add stores) instead of leaving two tensors for
    autograd to sum.  The alias gradient is modified in place, so it must not be shared with another branch."""

    @staticmethod
    def forward(ctx, x, weight, bias, act):
        y = _LinearFn.forward(ctx, x, weight, bias, act)
        return y, x.detach()

    @staticmethod
    def backward(ctx, dy, d_alias):
        return _linear_backward(ctx, dy, d_alias)


def _check_save8(x, weight, bias, act):
    if _ACT[act] == 1:
        raise ValueError("save8 keeps the value before a GELU; a ReLU needs one bit per value, which it does not take")
    saved8._check(x.dtype, "save8")
    # one call runs the whole pass from addresses and sizes: they have to fit each other
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"weight must be [out_features, in_features] and x [..., in_features], got {tuple(weight.shape)} and {tuple(x.shape)}")
    if bias is not None and (bias.dim() != 1 or bias.shape[0] != weight.shape[0]):
        raise ValueError(f"bias must be [{weight.shape[0]}], got {tuple(bias.shape)}")
    if weight.device != x.device or (bias is not None and bias.device != x.device):
        raise ValueError(f"x is on {x.device}, weight on {weight.device}" + ("" if bias is None else f", bias on {bias.device}"))


def linear(x, weight, bias=None, act=None, save8=False):
    """act(x @ weight.T + bias) with the epilogue fused into the GEMM.

    `save8` (act None or "gelu"): what the backward pass needs of the activations is kept in 8 bits (see ops/saved8.py).  The
    output is the same; the weight's gradient is computed from the stored x, and with GELU all gradients from the stored
    pre-activation, which is rounded to x's type before it is stored.  Gradients of gradients are refused."""
    if save8:
        _check_save8(x, weight, bias, act)
        return _Linear8Fn.apply(x, weight, bias, act, torch.is_grad_enabled())
    return _LinearFn.apply(x, weight, bias, act)


def linear_passthrough(x, weight, bias=None, act=None, save8=False):
    """(linear(x), alias of x): use the alias for the residual branch; see _LinearPassFn."""
    if save8:
        _check_save8(x, weight, bias, act)
    if x.is_cuda and x.dtype == torch.bfloat16:
        if save8:
            return _Linear8PassFn.apply(x, weight, bias, act, torch.is_grad_enabled())
        return _LinearPassFn.apply(x, weight, bias, act)
    return linear(x, weight, bias, act, save8), x


class Linear(nn.Module):
    """`save8`: keep the activations for the backward pass in 8 bits (see `linear`)."""

    save8 = False

    def __init__(self, in_features, out_features, bias=True, act=None, save8=False):
        super().__init__()
        self.in_features, self.out_features, self.act, self.save8 = in_features, out_features, act, save8
        self.weight = nn.Parameter(torch.empty(out_features, in_features))
        self.bias = nn.Parameter(torch.zeros(out_features)) if bias else None
        nn.init.kaiming_uniform_(self.weight, a=math.sqrt(5))

    def forward(self, x, passthrough=False):
        if passthrough:
            return linear_passthrough(x, self.weight, self.bias, self.act, self.save8)
        return linear(x, self.weight, self.bias, self.act, self.save8)
