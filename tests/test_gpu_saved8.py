"""The 8-bit kernels against the CPU form, bit by bit, and the linear layer's gradients against 64 bits."""
import math

import pytest
import torch

from test_saved8_cpu import blocks_to_try
from tips_b200.ops.linear import gemm_status, gemm_tn, linear, linear_passthrough
from tips_b200.ops.saved8 import act_bwd8, pack8

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def within(got, want, bound):
    """NaN where NaN is wanted (a pre-activation beyond fp16), and elsewhere within the bound."""
    nan = want.isnan()
    return bool((got.isnan() == nan).all() and (((got.double() - want).abs() <= bound) | nan).all())


def same(x):
    """pack8 on the GPU gives the CPU's bytes, and unpack its values in every type."""
    a, b = pack8(x), pack8(x.cpu())
    assert a.shape == b.shape and torch.equal(a.q.cpu(), b.q) and torch.equal(a.e.cpu(), b.e)
    for dtype in DTYPES:
        u, v = a.unpack(dtype).cpu(), b.unpack(dtype)
        assert u.dtype == v.dtype and torch.equal(u.nan_to_num(nan=-7.0), v.nan_to_num(nan=-7.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1,), (15,), (16,), (17,), (31,), (33,), (47,), (37, 101), (256, 512), (3, 7, 1000), (0,), ()])
def test_pack(shape, dtype):
    g = torch.Generator(device=DEV)
    g.manual_seed(len(shape))
    same((torch.randn(shape, generator=g, device=DEV) * 5).to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_special_values(dtype):
    same(blocks_to_try().to(dtype).to(DEV))
    ties = (torch.arange(-4096, 4096, device=DEV) * 0.25).to(dtype)  # many halves of a step
    same(ties)


def test_strides_and_alignment():
    x = torch.randn(64, 130, device=DEV).to(torch.bfloat16)
    for y in (x.t(), x[:, 1:], x[::2, 3:77], x.view(-1)[1:], x[:1].expand(5, 130)):
        same(y)


def test_long_tensor():
    """More values than the grid takes in one round."""
    x = torch.randn(148 * 8 * 256 * 16 + 77, device=DEV).to(torch.bfloat16)
    same(x)


@pytest.mark.parametrize("dtype", DTYPES)
# the largest take the slope from a table
@pytest.mark.parametrize("rows,cols", [(1, 8), (7, 24), (33, 264), (1000, 512), (4097, 40), (3, 4104), (5, 13), (40000, 72), (5000, 2048)])
def test_activation_backward(rows, cols, dtype):
    g = torch.Generator(device=DEV)
    g.manual_seed(rows)
    dy = torch.randn(rows, cols, generator=g, device=DEV).to(dtype)
    z = torch.randn(rows, cols, generator=g, device=DEV) * 2
    z[::3] *= torch.exp(torch.randn(z[::3].shape, generator=g, device=DEV) * 4)  # steps of any size
    p = pack8(z.to(dtype))
    z = p.unpack(torch.float32).double()
    want = dy.double() * (0.5 * (1 + torch.erf(z / math.sqrt(2))) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))
    u = torch.finfo(dtype).eps / 2
    # the derivative is computed in 32 bits, to 4e-6 at worst (erf by a rational approximation within 1.5e-7, approximate exp
    # and reciprocal at 2^-22 of factors up to 3); fp16's least half step is 2^-25
    slack = 4e-6 * dy.double().abs()
    for bias_dtype in DTYPES + [None]:
        dz, db = act_bwd8(dy, p.buf, bias_dtype)
        assert dz.dtype == dtype and within(dz, want, u * want.abs() + slack + 2.0 ** -25)
        if bias_dtype is None:
            assert db is None
            continue
        # sums of the unrounded values in 32 bits: 2^-24 per addition, at most rows of them in a row
        off = (slack + rows * 2.0 ** -24 * want.abs()).sum(0) + torch.finfo(bias_dtype).eps / 2 * want.sum(0).abs() + 2.0 ** -25
        assert db.dtype == bias_dtype and within(db, want.sum(0), off)
        assert torch.equal(db.nan_to_num(nan=-7.0), act_bwd8(dy, p.buf, bias_dtype)[1].nan_to_num(nan=-7.0))
    same_dy, db = act_bwd8(dy, None, torch.float32)
    assert same_dy.data_ptr() == dy.data_ptr()
    off = rows * 2.0 ** -24 * dy.double().abs().sum(0) + 2.0 ** -24 * dy.double().sum(0).abs()
    assert ((db.double() - dy.double().sum(0)).abs() <= off).all()


@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("rows,k,n", [(1, 64, 64), (100, 128, 512), (257, 520, 1096), (777, 72, 200), (2048, 1024, 4096),
                                      (4096, 512, 64), (64, 40, 13)])
def test_linear(rows, k, n, act):
    g = torch.Generator(device=DEV)
    g.manual_seed(rows + k)
    bf = torch.bfloat16
    x, dy = (torch.randn(rows, c, generator=g, device=DEV).to(bf) for c in (k, n))
    w = (torch.randn(n, k, generator=g, device=DEV) / math.sqrt(k)).to(bf)
    b = torch.randn(n, generator=g, device=DEV).to(bf)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = linear(*leaves, act, save8=True)
    assert torch.equal(y, linear(*leaves, act))
    got = torch.autograd.grad(y, leaves, dy)
    assert gemm_status() == 0
    u, slack = 2.0 ** -8, 2.0 ** -14
    dz = dy.double()
    if act:
        z = pack8(gemm_tn(x, w, b, act, want_pre=True)[1]).unpack().double()  # the value that the layer stores
        dz = dz * (0.5 * (1 + torch.erf(z / math.sqrt(2))) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))
        e = u * dz.abs() + 4e-6 * dy.double().abs()  # dz is rounded to bf16 as an operand
    else:
        e = torch.zeros_like(dz)
    x8, wd = pack8(x).unpack().double(), w.double()
    # products accumulate in 32 bits: slack times the sums of absolute values covers 2^-24 for each of up to 2^10 partial sums
    want = [dz @ wd, dz.t() @ x8, dz.sum(0)]
    mag = [dz.abs() @ wd.abs(), dz.abs().t() @ x8.abs(), dz.abs().sum(0)]
    off = [e @ wd.abs(), e.t() @ x8.abs(), 4e-6 * dy.double().abs().sum(0)]
    for a, t, m, o in zip(got, want, mag, off):
        assert a.dtype == bf and ((a.double() - t).abs() <= o + slack * m + u * t.abs()).all()


@pytest.mark.parametrize("m,n,k", [(16384, 4096, 1024), (9600, 4096, 64), (5000, 4128, 72), (16384, 1056, 256)])
def test_pre_activation_packed_by_the_gemm(m, n, k):
    """The bytes are those of packing the 16-bit pre-activation, with infinities and NaN among them; ragged rows and columns."""
    from tips_b200.ops import base
    from tips_b200.ops.linear import _linear8_forward
    from tips_b200.ops.saved8 import _pack, _parts
    g = torch.Generator(device=DEV)
    g.manual_seed(m + n)
    bf = torch.bfloat16
    a, b = torch.randn(m, k, generator=g, device=DEV).to(bf), torch.randn(n, k, generator=g, device=DEV).to(bf)
    bias = torch.randn(n, generator=g, device=DEV).to(bf)
    a[7, 3], a[m - 1, 0], b[n - 1, 1], bias[5] = math.inf, math.nan, -math.inf, 3e38
    a[100:200] *= 1e-30
    assert base.K().tipsk_gemm_pre8_fits(m, n, k)
    y, _, buf = _linear8_forward(a, b, bias, "gelu", False, True)
    want, pre = gemm_tn(a, b, bias, "gelu", want_pre=True)
    assert gemm_status() == 0
    assert torch.equal(y.nan_to_num(nan=-7.0), want.nan_to_num(nan=-7.0))
    for x, z in zip(_parts(buf, m * n), _parts(_pack(pre), m * n)):
        assert torch.equal(x, z)


def test_passthrough_and_dtypes():
    """The residual gradient is added into the input's; fp32 and fp16 layers take the same arguments."""
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    x, w, dy, da = (torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16) for s in ((300, 128), (256, 128), (300, 256), (300, 128)))
    x.requires_grad_()
    w.requires_grad_()
    y, alias = linear_passthrough(x, w, None, "gelu", save8=True)
    got = torch.autograd.grad((y, alias), (x, w), (dy, da.clone()))
    plain = torch.autograd.grad(linear(x, w, None, "gelu", save8=True), (x, w), dy)
    # dx is rounded to bf16 once in either; the sum once more
    assert ((got[0].double() - plain[0].double() - da.double()).abs()
            <= 2.0 ** -8 * (plain[0].double().abs() + got[0].double().abs()) + 2.0 ** -12).all()
    assert torch.equal(got[1], plain[1])
    for dtype in (torch.float32, torch.float16):
        a, b = x.detach().to(dtype).requires_grad_(), w.detach().to(dtype).requires_grad_()
        y = linear(a, b, None, "gelu", save8=True)
        got = torch.autograd.grad(y, (a, b), dy.to(dtype))
        for t, v in zip(got, plain):
            assert t.dtype == dtype and (t.double() - v.double()).norm() <= 2.0 ** -5 * v.double().norm()


@pytest.mark.parametrize("save8", [False, True])
def test_passthrough_of_a_sum_with_its_input(save8):
    """The layer's output and its input's alias get one and the same gradient, which the input's is added into."""
    g = torch.Generator(device=DEV)
    g.manual_seed(6)
    bf = torch.bfloat16
    x, w, dy = (torch.randn(*s, generator=g, device=DEV).to(bf) for s in ((700, 256), (256, 256), (700, 256)))
    x.requires_grad_()
    w.requires_grad_()
    y, alias = linear_passthrough(x, w, None, None, save8)
    got = torch.autograd.grad(y + alias, (x, w), dy)
    plain = torch.autograd.grad(linear(x, w, None, None, save8), (x, w), dy)
    assert ((got[0].double() - plain[0].double() - dy.double()).abs()
            <= 2.0 ** -8 * (plain[0].double().abs() + got[0].double().abs()) + 2.0 ** -12).all()
    if save8:
        assert torch.equal(got[1], plain[1])
    else:
        # without save8 the 700 products of an element are added in no fixed order, so that two runs may differ: each sum by
        # 700 * 2^-24 of the sum of absolute values, and by a half step of bf16, 2^-8, when it is rounded
        bound = 2.0 ** -8 * (got[1].double().abs() + plain[1].double().abs()) + 2 * 700 * 2.0 ** -24 * (dy.double().abs().t() @ x.detach().double().abs())
        assert ((got[1].double() - plain[1].double()).abs() <= bound).all()


def test_bias_of_another_type():
    x, w = torch.randn(64, 128, device=DEV).to(torch.bfloat16), torch.randn(256, 128, device=DEV).to(torch.bfloat16)
    dy = torch.randn(64, 256, device=DEV).to(torch.bfloat16)
    for dtype in (torch.float32, torch.float64, torch.float16):
        b = torch.randn(256, device=DEV).to(torch.bfloat16).to(dtype).requires_grad_()
        (db,) = torch.autograd.grad(linear(x, w, b, None, save8=True), b, dy)
        assert db.dtype == dtype
        # sums of 64 addends in 32 bits, rounded to the bias's type
        bound = 64 * 2.0 ** -24 * dy.double().abs().sum(0) + max(torch.finfo(dtype).eps, 2.0 ** -23) / 2 * dy.double().sum(0).abs()
        assert ((db.double() - dy.double().sum(0)).abs() <= bound).all()


def test_offsets_beyond_32_bits():
    """More than 2^31 values: the last ones keep their places."""
    n = 2 ** 31 + 2 ** 20 + 40
    x = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    tail = torch.randn(2 ** 20 + 40, device=DEV).to(torch.bfloat16)
    x[2 ** 31:] = tail
    p, small = pack8(x), pack8(tail)
    assert torch.equal(p.q[2 ** 31:], small.q) and torch.equal(p.e[2 ** 26:], small.e)
    y = p.unpack()
    assert torch.equal(y[2 ** 31:], small.unpack()) and not y[:2 ** 31:4097].any()


def test_graph_and_stream():
    x = torch.randn(513, 96, device=DEV).to(torch.bfloat16)
    want = pack8(x).unpack()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = pack8(x).unpack()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want)
    buf = torch.zeros_like(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = pack8(buf).unpack()
    buf.copy_(x)
    g.replay()
    assert torch.equal(y, want)


def test_encoder_keeps_less_and_trains_alike():
    """A padded batch through the small encoder with its linear layers at 8 bits: the loss is the same, the gradients are near
    those of the 16-bit form, and less is kept for the backward pass."""
    from tips_b200.models.bert import synthetic_mlm_batch, tiny_bert
    torch.manual_seed(0)
    a = tiny_bert()
    b = tiny_bert(save8=True)
    b.load_state_dict(a.state_dict())
    ids, pos, labels = (t.to(DEV) for t in synthetic_mlm_batch(8, 64, 1024, seed=3))
    n = torch.tensor([64, 20, 33, 64, 1, 50, 7, 64], device=DEV)
    pos = pos % n[:, None]
    kept, losses = [], []
    for m in (a, b):
        own = {p.data_ptr() for p in m.parameters()}
        seen = {}

        def keep(t):
            if t.data_ptr() not in own:
                seen[t.data_ptr()] = t.untyped_storage().nbytes()
            return t

        with torch.autograd.graph.saved_tensors_hooks(keep, lambda t: t):
            loss = m.loss(ids, pos, labels, lengths=n)
        kept.append(sum(seen.values()))
        loss.backward()
        losses.append(loss.detach())
    # the same logits; the loss kernel adds the 80 rows' terms, none negative, in any order: 2^-24 of the sum per addition
    assert torch.allclose(*losses, rtol=80 * 2.0 ** -24, atol=0)
    assert kept[1] < 0.8 * kept[0]
    for (name, p), q in zip(a.named_parameters(), b.parameters()):
        if p.grad is not None and float(p.grad.float().norm()) > 0 and "qkv.bias" not in name:
            # a stored value is off by 0.8 % of its block's root mean square; through two layers that stays within 10 %
            assert (p.grad.float() - q.grad.float()).norm() <= 0.1 * p.grad.float().norm(), name


def test_the_largest_fp16_values():
    x = torch.randn(9, 32, device=DEV).to(torch.float16)
    x[0, :3], x[4, 1], x[8, 30:] = torch.tensor([65504.0, 65030.0, -65024.0]), -65504.0, torch.tensor([65504.0, math.nan])
    for y in (x, x.view(-1)[:101], x.float() * 4):  # whole blocks, a last one of five values, values beyond fp16
        same(y)
    y = pack8(x).unpack()
    assert bool((y.isfinite() == x.isfinite()).all())
    w = torch.zeros(64, 32, device=DEV, dtype=torch.float16, requires_grad=True)
    dy = torch.full((9, 64), 2.0 ** -10, device=DEV, dtype=torch.float16)
    dy[:, 3] = 0.0
    (dw,) = torch.autograd.grad(linear(x[:8], w, save8=True), w, dy[:8])
    kept = y[:8].double()
    want = dy[:8].double().t() @ kept
    # a half step of the result; sums of eight addends in 32 bits
    bound = 2.0 ** -11 * want.abs() + 8 * 2.0 ** -24 * (dy[:8].double().t() @ kept.abs()) + 2.0 ** -25
    assert bool(((dw.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("act", [None, "gelu"])
def test_no_kernel_packs_without_a_backward_pass_to_come(act):
    """One launch, that of the product, and the same output."""
    from tips_b200.ops import base
    g = torch.Generator(device=DEV)
    g.manual_seed(7)
    x = torch.randn(300, 128, generator=g, device=DEV).to(torch.bfloat16)
    w = torch.randn(256, 128, generator=g, device=DEV).to(torch.bfloat16).requires_grad_()
    want = linear(x, w, None, act, save8=True)
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            for fn in (lambda: linear(x, w, None, act, save8=True), lambda: linear_passthrough(x, w, None, act, save8=True)[0]):
                before = base.launches()
                y = fn()
                assert base.launches() == before + 1 and torch.equal(y, want)
