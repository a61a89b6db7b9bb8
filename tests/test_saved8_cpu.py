"""The 8-bit form of activations on CPU tensors, against its definition written out value by value, and its refusals."""
import math

import pytest
import torch

from tips_b200.ops.linear import Linear, linear, linear_passthrough
from tips_b200.ops.saved8 import Packed8, pack8


def by_definition(values):
    """The stored values of one block of at most 32 numbers, in Python's own arithmetic (64 bits, all steps exact)."""
    finite = [abs(x) for x in values if math.isfinite(x)]
    e = -126
    while e < 121 and round(max(finite, default=0.0) / 2.0 ** e) > 127:  # Python rounds ties to even, as rint does
        e += 1
    return [max(-127, min(127, round(x / 2.0 ** e))) * 2.0 ** e if math.isfinite(x) else math.nan for x in values]


def blocks_to_try():
    g = torch.Generator().manual_seed(0)
    out = [torch.randn(32, generator=g) * 10.0 ** (i - 8) for i in range(16)]
    out += [torch.zeros(32), torch.full((32,), 3.0e38), torch.full((32,), torch.finfo(torch.float32).max), torch.full((32,), 1.5e-45),
            torch.linspace(-1e-38, 1e-38, 32), torch.arange(32) * 0.5 - 8, torch.arange(32) + 96.5, torch.arange(32) + 96.0]
    for top in (127.5, 127.49999, 127.0, 63.75, 255.0, 128.0):  # around where the step doubles
        out.append(torch.cat([torch.tensor([top]), torch.arange(31) * 4.0 + 0.5]))
    bad = torch.randn(32, generator=g)
    bad[3], bad[4], bad[31] = math.inf, -math.inf, math.nan
    return torch.stack(out + [bad, torch.full((32,), math.nan), torch.full((32,), -math.inf)])


def test_definition():
    x = blocks_to_try()
    p = pack8(x)
    want = torch.tensor([by_definition(row.tolist()) for row in x], dtype=torch.float64)
    assert torch.equal(p.unpack().double().nan_to_num(nan=-12345.0), want.nan_to_num(nan=-12345.0))
    assert p.nbytes == x.numel() + x.shape[0] and p.q.dtype == p.e.dtype == torch.int8


@pytest.mark.parametrize("shape", [(1,), (31,), (32,), (33,), (3, 5, 7), (0,), (2, 0, 4), ()])
def test_shapes_and_the_last_block(shape):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(1))
    p = pack8(x)
    assert p.shape == x.shape and p.q.numel() == x.numel() and p.e.numel() == (x.numel() + 31) // 32
    assert x.numel() * 33 / 32 <= p.nbytes < x.numel() * 33 / 32 + 17
    y = p.unpack()
    assert y.shape == x.shape and y.dtype == x.dtype
    flat = x.reshape(-1).tolist()
    want = [v for i in range(0, len(flat), 32) for v in by_definition(flat[i:i + 32])]
    assert y.reshape(-1).tolist() == want


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_stored_values_are_exact_and_stay(dtype):
    x = (torch.randn(40, 96, generator=torch.Generator().manual_seed(2)) * 3).to(dtype)
    p = pack8(x)
    y = p.unpack()
    assert torch.equal(y.float(), p.unpack(torch.float32)) and torch.equal(p.unpack(torch.bfloat16).float(), y.float())
    assert torch.equal(pack8(y).unpack(), y)
    amax = x.float().view(-1, 32).abs().amax(1, keepdim=True)
    assert ((x.float() - y.float()).view(-1, 32).abs() <= amax / 127).all()
    assert torch.equal(pack8(x.t()).unpack(), pack8(x.t().contiguous()).unpack())


def test_refusals():
    for dtype in (torch.float64, torch.int8, torch.int32):
        with pytest.raises(TypeError):
            pack8(torch.zeros(4, dtype=dtype))
        with pytest.raises(TypeError):
            pack8(torch.zeros(4)).unpack(dtype)
    x, w = torch.zeros(2, 4), torch.zeros(3, 4)
    for fn in (linear, linear_passthrough):
        with pytest.raises(ValueError):
            fn(x, w, None, "relu", save8=True)
        with pytest.raises(TypeError):
            fn(x.double(), w.double(), save8=True)
    y = linear(x, w.requires_grad_(), save8=True)
    (g,) = torch.autograd.grad(y.square().sum(), w, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("bias", [True, False])
def test_linear_gradients(act, bias):
    g = torch.Generator().manual_seed(3)
    x, w, dy = (torch.randn(*s, generator=g) for s in ((2, 5, 24), (16, 24), (2, 5, 16)))
    b = torch.randn(16, generator=g) if bias else None
    leaves = [t.clone().requires_grad_() for t in (x, w) + ((b,) if bias else ())]
    y = linear(*leaves, *([] if bias else [None]), act, save8=True)
    assert torch.equal(y, linear(*leaves, *([] if bias else [None]), act))
    got = torch.autograd.grad(y, leaves, dy)
    x8 = pack8(x).unpack().double().view(10, 24)
    dz = dy.double().view(10, 16)
    if act:
        pre = x.view(10, 24) @ w.t() + (b if bias else 0)
        z = pack8(pre).unpack().double()
        dz = dz * (0.5 * (1 + torch.erf(z / math.sqrt(2))) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))
    want = [(dz @ w.double()).view(2, 5, 24), dz.t() @ x8, dz.sum(0)]
    for a, t in zip(got, want):
        assert torch.allclose(a.double(), t, rtol=1e-5, atol=1e-5)


def test_only_what_a_gradient_needs_is_kept():
    x, w = torch.randn(8, 32), torch.randn(4, 32)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.numel() * t.element_size()) or t, lambda t: t):
        linear(x, w.clone().requires_grad_(), None, "gelu", save8=True)
        assert sum(kept) == w.numel() * 4 + 8 * 32 + 8 + 8 * 4 + 1  # the weight, x and the pre-activation
        kept.clear()
        linear(x.clone().requires_grad_(), w, save8=True)
        assert sum(kept) == w.numel() * 4


def test_module():
    torch.manual_seed(0)
    a = Linear(24, 16, act="gelu", save8=True)
    b = Linear(24, 16, act="gelu")
    b.load_state_dict(a.state_dict())
    x = torch.randn(10, 24)
    assert torch.equal(a(x), b(x))
    y, alias = a(x, passthrough=True)
    assert torch.equal(y, b(x)) and torch.equal(alias, x)
    assert isinstance(pack8(x), Packed8)


def test_the_largest_fp16_values_stay_finite():
    """From 65024 on a value is stored as 64 * 2^10 = 65536, which fp16 does not have."""
    x = torch.tensor([65504.0, 65030.0, -65504.0, -65024.0, 64999.0, 1000.0, 3.0, math.inf], dtype=torch.float16)
    p = pack8(x)
    assert p.unpack(torch.float32).tolist()[:5] == [65536.0, 65536.0, -65536.0, -65536.0, 64512.0]
    y = p.unpack()
    assert y.tolist()[:7] == [65504.0, 65504.0, -65504.0, -65504.0, 64512.0, 1024.0, 0.0] and bool(y[7].isnan())
    assert bool(((y.double() - x.double())[:7].abs() <= 512).all())  # half a step
    # another type's values beyond fp16's range are as far beyond it as they were
    assert pack8(x.float()).unpack(torch.float16).tolist()[:2] == [math.inf, math.inf]


def test_fp16_weight_gradient_at_the_top_of_the_range():
    x = torch.full((4, 32), 1.0, dtype=torch.float16)
    x[0, :2], x[3, 1] = torch.tensor([65504.0, 65100.0]), -65504.0
    w = torch.zeros(8, 32, dtype=torch.float16, requires_grad=True)
    dy = torch.full((4, 8), 2.0 ** -10, dtype=torch.float16)
    dy[:, 3] = 0.0
    (dw,) = torch.autograd.grad(linear(x, w, save8=True), w, dy)
    want = dy.double().t() @ pack8(x).unpack().double()
    # a half step of the result; sums of four addends in 32 bits
    bound = 2.0 ** -11 * want.abs() + 4 * 2.0 ** -24 * (dy.double().t() @ x.double().abs())
    assert bool(((dw.double() - want).abs() <= bound).all()) and not dw[3].any()


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_nothing_is_packed_without_a_backward_pass_to_come(mode, monkeypatch):
    from tips_b200.ops import saved8
    packed = []
    pack = saved8._pack
    monkeypatch.setattr(saved8, "_pack", lambda t: packed.append(t.shape) or pack(t))
    x = torch.randn(10, 24)
    layer = Linear(24, 16, act="gelu", save8=True)
    with mode():
        y = layer(x)
        for t in linear_passthrough(x, layer.weight, layer.bias, "gelu", save8=True):
            assert not t.requires_grad
    assert packed == []
    assert torch.equal(layer(x), y) and len(packed) == 2


@pytest.mark.parametrize("fn", [linear, linear_passthrough])
def test_sizes_and_devices_that_do_not_fit_are_refused(fn):
    """A pass is one call with addresses and sizes, which would read beyond a weight with shorter rows or a shorter bias."""
    x, w, b = torch.zeros(2, 5, 64), torch.zeros(128, 64), torch.zeros(128)
    fn(x, w, b, save8=True)
    for bad in ((x, w[:, :56], b), (x, w[0], b), (x[..., :8], w, b), (x, w, b[:127]), (x, w, b[:1]), (x, w, b[None]), (x[0, 0, 0], w, b),
                (x, w.to("meta"), None), (x, w, b.to("meta"))):
        with pytest.raises(ValueError):
            fn(*bad, save8=True)
