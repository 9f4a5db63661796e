"""The row operators of a training step (normalisation, dropout, loss) against their definitions in 64 bits.

Tolerances count roundings.  ``U`` is half a step of the operator's sums (2^-24, for fp64 2^-53), ``half_step`` that of the
result's type; a sum of n terms whose longest chain is c has an error of at most c * U * sum|terms|."""
import math
import subprocess
import sys
import threading
from pathlib import Path

import numpy as np
import pytest
import torch

from compressgnn_b200 import runtime as rt
from compressgnn_b200.layer import CrossEntropy, Dropout, KPropagate, LayerNorm
from compressgnn_b200.model import GCN

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
TYPES = [F32, F64, BF16, F16]
IGNORED = -100


def unit(dtype):
    return 2.0**-53 if dtype == F64 else 2.0**-24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half the least positive value of a type: what a result near zero may be off by."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def within(got, want, bound, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[~finite & ~torch.isnan(want)],
                                                                           want[~finite & ~torch.isnan(want)]), what
    excess = ((got - want).abs() - bound)[finite]
    assert excess.numel() == 0 or excess.max() <= 0, f"{what}: over its bound by {excess.max():.3e}"


def rand(*shape, dtype=F32, seed=0, scale=1.0, offset=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=gen, dtype=F64) * scale + offset).to(dtype)


# ---------------------------------------------------------------------------------------------
# the random words
# ---------------------------------------------------------------------------------------------
def words(first, count, key):
    """Philox4x32 with 7 rounds, in whole numbers of 64 bits without a sign."""
    e = np.arange(first, first + count, dtype=np.uint64)
    block, low = e >> np.uint64(2), np.uint64(0xFFFFFFFF)
    c = [block & low, block >> np.uint64(32), np.full(count, 0x243F6A88, np.uint64), np.full(count, 0x85A308D3, np.uint64)]
    k = [key & 0xFFFFFFFF, (key >> 32) & 0xFFFFFFFF]
    for _ in range(7):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), p1 & low, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p0 & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.select([(e & np.uint64(3)) == np.uint64(i) for i in range(4)], c)


def kept(shape, p, key, first=0):
    n = int(np.prod(shape))
    bound = min(int(p * 2**32), 2**32 - 1)
    return torch.from_numpy(words(first, n, key & (2**64 - 1)) >= np.uint64(bound)).view(shape).cuda()


# ---------------------------------------------------------------------------------------------
# normalisation
# ---------------------------------------------------------------------------------------------
def norm_reference(x, weight, bias, eps, relu, p, key, z_sign):
    """The formulas in 64 bits, with the bound of each result.  ``z_sign``: what the operator takes z for where its sign
    decides (a value within its error of the border may lie on either side)."""
    dtype, width = x.dtype, x.size(-1)
    u = unit(dtype)
    wide = x.double()
    mean = wide.mean(-1, keepdim=True)
    rstd = (wide.var(-1, correction=0, keepdim=True) + eps).rsqrt()
    h = (wide - mean) * rstd
    w = weight.double() if weight is not None else torch.ones(width, dtype=F64, device="cuda")
    b = bias.double() if bias is not None else torch.zeros(width, dtype=F64, device="cuda")
    z = h * w + b
    mask = torch.ones_like(z, dtype=torch.bool) if not relu else z_sign > 0
    keep = kept(x.shape, p, key) if p else torch.ones_like(mask)
    factor = keep.double() / (1 - p if p else 1)
    y = torch.where(mask, z, 0.0) * factor
    # a lane adds up at most 64 terms, or width / 512, before the tree; the deviations' squares likewise
    chain = (64 + width / 512 + 16) * u
    h_bound = 4 * chain * (1 + wide.abs().amax(-1, keepdim=True) * rstd)
    y_bound = (h_bound * w.abs() + 4 * u * ((h * w).abs() + b.abs())) * factor + half_step(dtype) * y.abs() + least(dtype)

    def backward(grad):
        g = torch.where(mask, grad.double() * factor, 0.0)
        v = g * w
        c0, c1 = v.mean(-1, keepdim=True), (v * h).mean(-1, keepdim=True)
        dx = rstd * (v - c0 - h * c1)
        most = v.abs().amax(-1, keepdim=True)
        dx_bound = rstd * most * (1 + h.abs()) * 4 * (chain + h_bound) + half_step(dtype) * dx.abs() + least(dtype)
        parts = (g * h).reshape(-1, width), g.reshape(-1, width)
        bounds = ((g.abs() * h_bound).reshape(-1, width).sum(0) + 640 * u * parts[0].abs().sum(0), 640 * u * parts[1].abs().sum(0))
        kind = weight.dtype if weight is not None else bias.dtype if bias is not None else dtype
        sums = [part.sum(0) for part in parts]
        return dx, dx_bound, [(s, bound + half_step(kind) * s.abs() + least(kind)) for s, bound in zip(sums, bounds)]

    return y, y_bound, backward


def check_norm(x, weight, bias, relu=False, p=0.0, key=1234567890123, eps=1e-5, what=""):
    leaves = [t for t in (x, weight, bias) if t is not None]
    for t in leaves:
        t.requires_grad_()
    with torch.no_grad():
        sign = rt.layer_norm(x, weight, bias, eps)
    y = rt.layer_norm(x, weight, bias, eps, "relu" if relu else None, p, key)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    want, bound, backward = norm_reference(x.detach(), *(t if t is None else t.detach() for t in (weight, bias)), eps, relu, p, key,
                                           sign)
    within(y.detach(), want, bound, f"{what} y")
    grad = rand(*x.shape, dtype=x.dtype, seed=9)
    grads = torch.autograd.grad(y, leaves, grad)
    dx, dx_bound, params = backward(grad)
    within(grads[0], dx, dx_bound, f"{what} dx")
    rest = list(grads[1:])
    for t, (s, s_bound) in zip((weight, bias), params):
        if t is not None:
            got = rest.pop(0)
            assert got.dtype == t.dtype and got.shape == t.shape
            within(got, s, s_bound, f"{what} parameter")


WIDTHS = [1, 2, 3, 4, 7, 8, 16, 31, 47, 64, 100, 128, 255, 256, 301, 512, 602, 1000, 1024, 2048, 2050, 4096, 4100, 8192, 10001, 16384,
          20000]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_norm_widths(width, dtype):
    rows = 37 if width <= 4096 else 5
    check_norm(rand(rows, width, dtype=dtype, offset=0.3), rand(width, dtype=dtype, seed=1, scale=0.3, offset=1.0),
               rand(width, dtype=dtype, seed=2, scale=0.3), relu=True, p=0.3, what=f"{dtype} {width}")


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("p", [0.0, 0.5])
@pytest.mark.parametrize("params", ["both", "weight", "bias", "none"])
def test_norm_parts(params, p, relu):
    for dtype, kind in ((F32, F32), (F64, F64), (BF16, F32), (BF16, BF16), (F16, F32), (F16, F16)):
        for rows, width in ((1, 64), (3, 33), (1000, 24), (300, 5000)):
            weight = rand(width, dtype=kind, seed=1, offset=1.0) if params in ("both", "weight") else None
            bias = rand(width, dtype=kind, seed=2) if params in ("both", "bias") else None
            check_norm(rand(rows, width, dtype=dtype), weight, bias, relu, p, what=f"{dtype} {kind} {rows}x{width}")


@pytest.mark.parametrize("rows", [1, 2, 31, 592, 5000, 40000])
@pytest.mark.parametrize("width", [6, 64, 129])
def test_norm_rows(rows, width):
    check_norm(rand(rows, width), rand(width, seed=1, offset=1.0), rand(width, seed=2), p=0.1, what=f"{rows}x{width}")


@pytest.mark.parametrize("dtype,rows,width", [(F64, 1500, 601), (F64, 700, 4098), (F32, 1100, 8200), (F32, 1537, 8193), (BF16, 1100, 8193),
                                              (F16, 1025, 8200)])
def test_norm_parameters_of_many_long_rows(dtype, rows, width):
    """Rows that no team holds, more of them than one block of the parameters' sums takes, in shares of unequal size."""
    for relu, p in ((False, 0.0), (True, 0.3)):
        check_norm(rand(rows, width, dtype=dtype, offset=0.3), rand(width, dtype=dtype, seed=1, scale=0.3, offset=1.0),
                   rand(width, dtype=dtype, seed=2, scale=0.3), relu, p, what=f"{dtype} {rows}x{width}")


def test_norm_of_rows_far_from_zero():
    """Deviations are squared, not squares subtracted: a mean of a thousand deviations leaves the result exact to its bound."""
    for dtype in (F32, F64):
        check_norm(rand(50, 128, dtype=dtype, offset=1000.0), rand(128, dtype=dtype, seed=1), None, what=str(dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_layouts(dtype):
    base = rand(40, 300, dtype=dtype)
    weight, bias = rand(64, dtype=dtype, seed=1), rand(64, dtype=dtype, seed=2)
    for x in (base[:, 8:72], base[:, 5:69], base[::2, :64], base[:, :128:2], base.t()[:40, :].t()[:, :40][:, :64], base[:1].expand(7, 300)[:, :64]):
        w, b = weight[:x.size(1)], bias[:x.size(1)]
        check_norm(x.detach(), w.detach().clone(), b.detach().clone(), relu=True, what=str(x.stride()))
    # parameters that begin anywhere and lie apart
    for w, b in ((rand(65, dtype=dtype, seed=1)[1:], rand(67, dtype=dtype, seed=2)[3:]), (rand(128, dtype=dtype, seed=1)[::2], rand(64, dtype=dtype, seed=2))):
        check_norm(base[:, :64].detach().clone(), w.detach(), b.detach(), relu=True)
    flat = rand(40 * 64 + 1, dtype=dtype)
    check_norm(flat[1:].view(40, 64).detach(), weight.detach(), bias.detach(), relu=True, p=0.2, what="off a vector's boundary")
    x = rand(3, 5, 2, 24, dtype=dtype)
    check_norm(x, None, None, relu=True, p=0.2, what="four dimensions")
    check_norm(rand(24, dtype=dtype), None, None, what="one dimension")
    check_norm(x.detach().transpose(0, 2), None, None, what="dimensions in another order")


def test_norm_of_nothing():
    for shape in ((0, 8), (4, 0), (0, 0)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        w, b = torch.ones(shape[1], device="cuda", requires_grad=True), torch.zeros(shape[1], device="cuda", requires_grad=True)
        y = rt.layer_norm(x, w, b, dropout=0.5)
        assert y.shape == shape
        for g, t in zip(torch.autograd.grad(y, (x, w, b), torch.ones_like(y)), (x, w, b)):
            assert g.shape == t.shape and not g.any()


def test_norm_of_values_that_are_no_numbers():
    x = rand(6, 64)
    x[1, 3], x[2, 5] = float("nan"), float("inf")
    y = rt.layer_norm(x, activation="relu")
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all() and torch.isfinite(y[[0, 3, 4, 5]]).all()
    constant = rt.layer_norm(torch.full((3, 64), 7.0, device="cuda"), None, torch.ones(64, device="cuda"))
    assert torch.equal(constant, torch.ones_like(constant))
    # a dropped element is zero whatever it was, its gradient too
    key = 77
    keep = kept((6, 64), 0.5, key)
    y = rt.layer_norm(x, dropout=0.5, seed=key)
    assert not y[~keep].any() and torch.isnan(y[1][keep[1]]).all()
    x = rand(6, 64).requires_grad_()
    w = torch.ones(64, device="cuda", requires_grad=True)
    grad = torch.where(keep, 1.0, float("inf"))
    dx, dw = torch.autograd.grad(rt.layer_norm(x, w, dropout=0.5, seed=key), (x, w), grad)
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all()


def test_norm_gradients_against_differences():
    for shape in ((5, 7), (3, 33), (2, 2600)):
        x, w, b = (rand(*s, dtype=F64, seed=i).requires_grad_() for i, s in enumerate((shape, shape[1:], shape[1:])))
        fast = shape[1] > 100
        assert torch.autograd.gradcheck(lambda *a: rt.layer_norm(*a, dropout=0.3, seed=5), (x, w, b), eps=1e-6, atol=1e-6, rtol=1e-4,
                                        fast_mode=fast)
        assert torch.autograd.gradcheck(lambda *a: rt.layer_norm(*a, activation="relu"), (x, w, b), eps=1e-7, atol=1e-5, rtol=1e-3,
                                        fast_mode=fast)


@pytest.mark.parametrize("wanted", ["x", "weight", "bias"])
def test_norm_gradient_of_one_input_alone(wanted):
    for width in (64, 5000):
        inputs = {"x": rand(20, width), "weight": rand(width, seed=1), "bias": rand(width, seed=2)}
        whole = [t.clone().requires_grad_() for t in inputs.values()]
        grad = rand(20, width, seed=3)
        want = dict(zip(inputs, torch.autograd.grad(rt.layer_norm(*whole, activation="relu"), whole, grad)))[wanted]
        inputs[wanted].requires_grad_()
        got, = torch.autograd.grad(rt.layer_norm(*inputs.values(), activation="relu"), inputs[wanted], grad)
        assert torch.equal(got, want)


def test_norm_refusals():
    x, w = rand(4, 8), rand(8, seed=1)
    for call, message in ((lambda: rt.layer_norm(x.int()), "float32"), (lambda: rt.layer_norm(x, w[:7]), "vectors"),
                          (lambda: rt.layer_norm(x, w.double()), "type"), (lambda: rt.layer_norm(x, w.bfloat16()), "type"),
                          (lambda: rt.layer_norm(x.bfloat16(), w.half()), "type"), (lambda: rt.layer_norm(x, w, w.double()), "one type"),
                          (lambda: rt.layer_norm(x, w.cpu()), "device"), (lambda: rt.layer_norm(x, w[None]), "vectors"),
                          (lambda: rt.layer_norm(x, dropout=1.0), "probability"), (lambda: rt.layer_norm(x, dropout=-0.1), "probability"),
                          (lambda: rt.layer_norm(x, eps=-1.0), "eps"), (lambda: rt.layer_norm(x.sum()), "dimension"),
                          (lambda: rt.layer_norm(x, dropout=0.5, seed=torch.zeros(1, dtype=torch.int64)), "seed"),
                          (lambda: rt.layer_norm(x, dropout=0.5, seed=torch.zeros(2, dtype=torch.int64, device="cuda")), "seed"),
                          (lambda: rt.layer_norm(x, dropout=0.5, seed=torch.zeros(1, device="cuda")), "seed")):
        with pytest.raises(RuntimeError, match=message):
            call()


# ---------------------------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [0, 1, 3, 4, 7, 8, 100, 4097, 123457])
def test_dropout(n, dtype):
    for p, key in ((0.3, 2**64 - 5), (0.999, 17), (2.0**-31, 3), (0.0, 3)):
        x, residual, grad = (rand(n, dtype=dtype, seed=i).requires_grad_() for i in range(3))
        keep = kept((n,), p, key)
        factor = keep.double() / (1 - p)
        y = rt.dropout(x, p, residual, key)
        assert y.dtype == dtype and y.shape == (n,)
        want = x.detach().double() * factor + residual.detach().double()
        # one rounding of 1 / (1 - p), one of the product, one of the sum, one to the type
        bound = 4 * unit(dtype) * ((x.detach().double() * factor).abs() + want.abs()) + half_step(dtype) * want.abs() + least(dtype)
        within(y.detach(), want, bound, f"{dtype} {n} {p}")
        dx, dresidual = torch.autograd.grad(y, (x, residual), grad.detach())
        within(dx, grad.detach().double() * factor, 2 * unit(dtype) * (grad.detach().double() * factor).abs() +
               half_step(dtype) * (grad.detach().double() * factor).abs() + least(dtype), "dx")
        assert torch.equal(dresidual, grad.detach())
        assert not rt.dropout(x, p, None, key)[~keep].any()


def test_dropout_has_the_mask_of_the_reconstruction():
    for rows, width in ((100, 64), (33, 47), (7, 6)):
        ones = torch.ones(1, width, device="cuda")
        index = torch.zeros(rows, dtype=torch.int64, device="cuda")
        for key in (0, 9, 2**63 + 11):
            assert torch.equal(rt.dropout(torch.ones(rows, width, device="cuda"), 0.3, seed=key),
                               rt.cluster_reconstruct(ones, index, None, True, 0.3, key))


@pytest.mark.parametrize("dtype", [F32, F16])
def test_dropout_layouts(dtype):
    flat = rand(4003, dtype=dtype)
    for x in (flat[1:], flat[3:1000], flat[::2], flat[:4000].view(40, 100).t(), flat[:1].expand(300)):
        assert torch.equal(rt.dropout(x, 0.3, seed=4), rt.dropout(x.contiguous().clone(), 0.3, seed=4))
        assert torch.equal(rt.dropout(x, 0.3, x, seed=4), rt.dropout(x.contiguous().clone(), 0.3, x.contiguous().clone(), seed=4))


def test_dropout_of_values_that_are_no_numbers():
    keep = kept((1000,), 0.5, 3)
    x = torch.full((1000,), float("nan"), device="cuda", requires_grad=True)
    y = rt.dropout(x, 0.5, seed=3)
    assert not y[~keep].any() and torch.isnan(y[keep]).all()
    dx, = torch.autograd.grad(y, x, torch.where(keep, 1.0, float("inf")))
    assert torch.equal(dx, torch.where(keep, 2.0, 0.0))


def test_dropout_keys():
    x = torch.ones(10000, device="cuda")
    torch.manual_seed(3)
    a, b = rt.dropout(x, 0.5), rt.dropout(x, 0.5)
    torch.manual_seed(3)
    keys = [int(torch.randint(0, 2**63 - 1, (1,))) for _ in range(2)]
    assert not torch.equal(a, b)
    for got, key in zip((a, b), keys):
        assert torch.equal(got, rt.dropout(x, 0.5, seed=key))
        on_device = torch.tensor([key], device="cuda")
        assert torch.equal(got, rt.dropout(x, 0.5, seed=on_device))
        assert torch.equal(got, rt.layer_norm(torch.zeros(10, 1000, device="cuda"), None, torch.ones(1000, device="cuda"), dropout=0.5,
                                              seed=on_device).view(-1))
    # a binomial of 10000: five standard deviations are 250
    assert all(abs(int((t == 0).sum()) - 5000) < 250 for t in (a, b))
    on_device = torch.tensor([5], device="cuda")
    leaf = x.clone().requires_grad_()
    y = rt.dropout(leaf, 0.5, seed=on_device)
    on_device += 1
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


def test_dropout_refusals():
    x = rand(4, 8)
    for call, message in ((lambda: rt.dropout(x, 1.0), "probability"), (lambda: rt.dropout(x, float("nan")), "probability"),
                          (lambda: rt.dropout(x.long(), 0.5), "float32"), (lambda: rt.dropout(x, 0.5, x[:1]), "shape"),
                          (lambda: rt.dropout(x, 0.5, x.double()), "type"), (lambda: rt.dropout(x, 0.5, x.cpu()), "device"),
                          (lambda: rt.dropout(x, 0.5, seed=torch.zeros(2, dtype=torch.int64, device="cuda")), "seed")):
        with pytest.raises(RuntimeError, match=message):
            call()


def test_dropout_beyond_32_bits():
    n, p, key = 2**32 + 4097, 0.25, 21
    x = torch.ones(n, dtype=F16, device="cuda")
    y = rt.dropout(x, p, seed=key)
    for first in (2**31 - 64, 2**32 - 64, n - 4096):
        assert torch.equal(y[first:first + 4096] != 0, kept((min(4096, n - first),), p, key, first))


# ---------------------------------------------------------------------------------------------
# loss
# ---------------------------------------------------------------------------------------------
def loss_case(rows, classes, dtype=F32, seed=0, scale=3.0, ignored=0.3):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    logits = rand(rows, classes, dtype=dtype, seed=seed, scale=scale)
    target = torch.randint(0, classes, (rows,), device="cuda", generator=gen)
    if rows > 1:
        target[torch.rand(rows, device="cuda", generator=gen) < ignored] = IGNORED
        target[0] = classes - 1
    return logits, target


def check_loss(logits, target, reduction, upstream=None, ignore_index=IGNORED, what=""):
    """Bounds: exp() is good to 2 + 1.2 d steps (of 2 U) at a distance d from the row's largest score, where it is at most
    e^-d, and the sum of a row is at least 1, so both are off by at most 64 U together; a chain of classes / 256 + 64
    additions; one rounding each of the score's distance, the logarithm, the difference and the product."""
    dtype, classes, rows = logits.dtype, logits.size(1), logits.size(0)
    u = unit(dtype)
    z = logits.detach().double()
    labelled = (target != ignore_index) & (target >= 0) & (target < classes)
    at = torch.where(labelled, target, 0)[:, None]
    log_p = z.log_softmax(1)
    each = torch.where(labelled, -log_p.gather(1, at).view(-1), 0.0)
    chain = (classes / 256 + 64 + 64) * u
    distance = (z.amax(1) - z.gather(1, at).view(-1)).abs()
    distance = torch.where(labelled & torch.isfinite(distance), distance, 0.0)
    each_bound = 2 * chain + 4 * u * (each.abs() + distance)
    each_bound = torch.where(torch.isfinite(each_bound), each_bound, 0.0)
    count = int(labelled.sum())
    kind = F64 if dtype == F64 else F32
    divide = count if reduction == "mean" else 1
    if reduction == "none":
        want, bound = each, each_bound
    else:
        want = each.sum() / divide if divide else torch.tensor(math.nan, device="cuda", dtype=F64)
        bound = each_bound.sum() / max(divide, 1) + half_step(kind) * 4 * want.abs()
    logits.requires_grad_()
    loss = rt.cross_entropy(logits, target, ignore_index, reduction)
    assert loss.dtype == kind and loss.shape == want.shape
    within(loss.detach(), want, bound, f"{what} loss")
    with torch.no_grad():
        assert torch.equal(rt.cross_entropy(logits, target, ignore_index, reduction).nan_to_num(-1), loss.detach().nan_to_num(-1))
    up = torch.ones_like(loss) if upstream is None else upstream.to(loss.dtype)
    share = torch.where(labelled, up.double().expand(rows) / max(divide, 1), 0.0)[:, None]
    p = log_p.exp()
    onehot = torch.zeros_like(p).scatter_(1, at, 1.0)
    grad = torch.where(labelled[:, None], (p - onehot) * share, 0.0)
    grad_bound = share.abs() * (2 * chain * p + 4 * u) + half_step(dtype) * grad.abs() + least(dtype)
    for _ in range(2):  # the second pass over the retained graph has nothing of the first
        got, = torch.autograd.grad(loss, logits, up, retain_graph=True)
        assert got.dtype == dtype and got.shape == logits.shape
        within(got, grad, torch.where(labelled[:, None], grad_bound, 0.0).nan_to_num(0.0), f"{what} gradient")
        got.fill_(7.0)
    return loss


CLASSES = [1, 2, 3, 4, 7, 8, 16, 17, 32, 47, 48, 64, 100, 128, 172, 349, 500, 512, 513, 1000, 1024, 1025, 5000, 16384, 50001]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", CLASSES)
def test_loss_classes(classes, dtype):
    rows = 70 if classes <= 5000 else 9
    for reduction in ("mean", "sum", "none"):
        logits, target = loss_case(rows, classes, dtype)
        check_loss(logits, target, reduction, what=f"{dtype} {classes} {reduction}")
    assert rt.device_status() == 0


@pytest.mark.parametrize("rows", [1, 2, 33, 1025, 4096, 4097, 20000, 200001])
def test_loss_rows(rows):
    for classes in (2, 7, 47):
        for reduction in ("mean", "sum", "none"):
            logits, target = loss_case(rows, classes)
            check_loss(logits, target, reduction, what=f"{rows}x{classes} {reduction}")


@pytest.mark.parametrize("classes", [5, 40, 90, 172, 380, 600, 1000, 4000, 20000, 60000, 130000])
def test_loss_around_the_sizes_of_one_cluster(classes):
    """Calls that one cluster does alone, those just too large for it, and the same losses as rows of a larger call."""
    for dtype in (F32, BF16, F64):
        for rows in (1, 8, 9, 33) if classes > 768 else (1, 8, 9, 250, 300, 1100, 4096, 4100):
            if rows * classes > 3_000_000:
                continue
            logits, target = loss_case(rows, classes, dtype)
            for reduction in ("mean", "sum"):
                check_loss(logits.detach(), target, reduction, what=f"{dtype} {rows}x{classes} {reduction}")


@pytest.mark.parametrize("dtype", [F32, F16])
def test_loss_with_an_incoming_gradient(dtype):
    for classes in (7, 47, 64, 2000):
        logits, target = loss_case(50, classes, dtype)
        for reduction in ("mean", "sum"):
            for up in (1.0, 1024.0, -0.5, 0.0):
                check_loss(logits.detach(), target, reduction, torch.tensor(up, device="cuda"), what=f"{classes} {reduction} {up}")
        check_loss(logits.detach(), target, "none", rand(50, seed=4), what=f"{classes} none")


def test_loss_layouts():
    base = rand(60, 400, seed=3, scale=2.0)
    target = torch.randint(0, 20, (60,), device="cuda")
    for x in (base[:, 8:56], base[:, 3:50], base[:, 1:385], base[:, 16:400], base[:, ::2], base.t()[:60].t(), base[:1].expand(60, 400)):
        for reduction in ("mean", "none"):
            check_loss(x.detach(), target[:x.size(0)], reduction, what=str(x.stride()))
    flat = rand(60 * 48 + 1, seed=3)
    check_loss(flat[1:].view(60, 48).detach(), target, "mean", what="off a vector's boundary")
    logits = base[:, :48].detach().clone()
    apart = torch.stack([target, target], 1)[:, 0]
    assert torch.equal(rt.cross_entropy(logits, apart), rt.cross_entropy(logits, target))


@pytest.mark.parametrize("classes", [7, 64, 3000])
def test_loss_of_masked_classes(classes):
    """Scores of minus infinity, or of the type's lowest value: classes that cannot be."""
    for low in (-math.inf, torch.finfo(F32).min):
        logits, target = loss_case(40, classes)
        masked = torch.rand(40, classes, device="cuda") < 0.5
        masked[torch.arange(40, device="cuda"), target.clamp_min(0)] = False
        logits[masked] = low
        check_loss(logits, target, "mean")
        check_loss(logits.detach(), target, "none")
    # a row with nothing left: fine without a label, not a number with one
    logits, target = loss_case(40, classes)
    logits[3] = -math.inf
    target[3] = IGNORED
    check_loss(logits, target, "mean")
    target[3] = 0
    each = rt.cross_entropy(logits, target, reduction="none")
    assert torch.isnan(each[3]) and torch.isfinite(each[torch.arange(40, device="cuda") != 3]).all()
    # the label's own score masked: an infinite loss, a finite gradient
    logits, target = loss_case(40, classes, ignored=0.0)
    logits[5, target[5]] = -math.inf
    check_loss(logits, target, "none")
    # whatever stands in a row without a label is not looked at
    logits, target = loss_case(40, classes)
    target[4] = IGNORED
    want = rt.cross_entropy(logits, target)
    logits[4] = math.nan
    leaf = logits.requires_grad_()
    loss = rt.cross_entropy(leaf, target)
    assert torch.equal(loss, want)
    got, = torch.autograd.grad(loss, leaf)
    assert torch.isfinite(got).all() and not got[4].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [7, 47, 384, 768, 769, 1000, 1025, 5000, 50001, 130000])
def test_loss_of_a_score_that_is_no_number(classes, dtype):
    """A NaN makes its row's loss and gradient NaN wherever it stands: among ordinary scores, and as the one class beside
    the label that is not masked.  The other rows keep their values."""
    for place in (0, 3, classes // 2, classes - 1):
        for masked in (False, True):
            logits, target = loss_case(6, classes, dtype, seed=place)
            target[1], target[4] = (place + classes // 3) % classes, place
            for row in (1, 4):
                if masked:
                    label = logits[row, target[row]].item()
                    logits[row] = -math.inf
                    logits[row, target[row]] = label
                logits[row, place] = math.nan
            for reduction in ("none", "sum", "mean"):
                check_loss(logits.detach().clone(), target, reduction, what=f"{dtype} {classes} {place} {masked} {reduction}")
            each = rt.cross_entropy(logits, target, reduction="none")
            assert each.isnan().tolist() == [False, True, False, False, True, False]


def test_loss_of_large_scores():
    for scale in (100.0, 1e4):
        for classes in (7, 1000, 3000):
            logits, target = loss_case(40, classes, scale=scale)
            check_loss(logits, target, "mean", what=f"{scale} {classes}")


@pytest.mark.parametrize("rising", [False, True])
@pytest.mark.parametrize("classes", [47, 768, 769, 1000, 1025, 4097, 50001, 130000])
def test_loss_of_scores_far_from_zero(classes, rising):
    """An offset that all scores of a row share, which changes neither the loss nor the gradient of a row's scores as they are
    stored; rising ones give a thread a larger score in every step.  The bounds are those of any scores: a distance from the
    row's largest score is exact to the type's rounding whatever the two have in common."""
    for dtype, offsets in ((F32, (3e3, -3e3, 1e5, 3e5, -3e5, 9e5, 2e6)), (F16, (3e2, -3e3)), (F64, (3e5,)), (BF16, (3e2,))):
        for offset in offsets:
            logits, target = loss_case(5, classes, dtype, seed=7)
            logits = (logits.double() + offset).to(dtype)
            if rising:
                logits = logits.sort(1).values
            target[1] = classes // 2
            for reduction in ("mean", "none"):
                check_loss(logits.detach().clone(), target, reduction, what=f"{dtype} {classes} {offset} {reduction}")


def test_loss_without_labels():
    logits, target = loss_case(40, 7)
    target[:] = IGNORED
    for reduction in ("mean", "sum", "none"):
        check_loss(logits.detach(), target, reduction)
    empty = torch.empty(0, 7, device="cuda", requires_grad=True)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert torch.isnan(rt.cross_entropy(empty, none)) and rt.cross_entropy(empty, none, reduction="sum") == 0
    assert rt.cross_entropy(empty, none, reduction="none").shape == (0,)
    assert torch.autograd.grad(rt.cross_entropy(empty, none), empty)[0].shape == (0, 7)


def test_loss_of_labels_that_are_no_classes():
    for classes in (7, 3000):
        logits, target = loss_case(40, classes)
        target[2], target[7], target[9] = classes, -1, 2**40
        for reduction in ("mean", "sum", "none"):
            assert rt.device_status() == 0
            check_loss(logits.detach(), target, reduction)
            assert rt.device_status() == 1
        target[2] = target[7] = target[9] = 3
        check_loss(logits.detach(), target, "mean", ignore_index=3)  # a class may be the one that is left out
        assert rt.device_status() == (1 if (target == IGNORED).any() else 0)


def test_a_copy_that_is_given_up():
    """Every wait of the loss for a copy given up at once: the blocks meet all the same, the call's results are NaN and the
    status says so; the next call is as ever."""
    from compressgnn_b200 import _lib
    for rows, classes in ((40, 7), (500, 47), (4000, 500), (100001, 7), (60000, 47), (9000, 768)):
        logits, target = loss_case(rows, classes)
        logits.requires_grad_()
        up = rand(rows, seed=1)

        def results():
            out = []
            for reduction in ("mean", "sum", "none"):
                loss = rt.cross_entropy(logits, target, reduction=reduction)
                for factor in (1.0, 2.0):
                    incoming = up if reduction == "none" else torch.full_like(loss, factor)
                    out += [loss.detach(), torch.autograd.grad(loss, logits, incoming, retain_graph=True)[0]]
            return out

        want = results()
        assert _lib.lib().cgnn_cross_entropy_wait_limit(0) == 2**20
        try:
            got = results()
            torch.cuda.synchronize()
        finally:
            assert _lib.lib().cgnn_cross_entropy_wait_limit(-1) == 0
        assert all(t.isnan().all() for t in got), (rows, classes)
        assert rt.device_status() == 2 and rt.device_status() == 0
        assert all(torch.equal(a, b) for a, b in zip(results(), want))
    assert _lib.lib().cgnn_cross_entropy_wait_limit(-1) == 2**20


def test_loss_gradients_against_differences():
    for classes in (5, 48, 1300):
        logits, target = loss_case(6, classes, F64)
        for reduction in ("mean", "sum", "none"):
            assert torch.autograd.gradcheck(lambda z: rt.cross_entropy(z, target, reduction=reduction), (logits.detach().requires_grad_(),),
                                            eps=1e-6, atol=1e-6, rtol=1e-4, fast_mode=classes > 100)


def test_loss_refusals():
    x, t = rand(4, 8), torch.zeros(4, dtype=torch.int64, device="cuda")
    for call, message in ((lambda: rt.cross_entropy(x.int(), t), "float32"), (lambda: rt.cross_entropy(x, t.int()), "int64"),
                          (lambda: rt.cross_entropy(x, t[:3]), "per row"), (lambda: rt.cross_entropy(x, t.cpu()), "device"),
                          (lambda: rt.cross_entropy(x[0], t), "matrix"), (lambda: rt.cross_entropy(x[:, :0], t), "matrix"),
                          (lambda: rt.cross_entropy(x, t[:, None]), "per row")):
        with pytest.raises(RuntimeError, match=message):
            call()


def test_rows_beyond_32_bits():
    """Offsets of elements that 32 bits do not hold, in the normalisation and in the loss."""
    rows, width = 2**20 + 3, 4104
    x = torch.empty(rows, width, dtype=F16, device="cuda").normal_()
    w, b = rand(width, dtype=F16, seed=1), rand(width, dtype=F16, seed=2)
    last = slice(rows - 5, rows)
    y = rt.layer_norm(x, w, b, activation="relu")
    assert torch.equal(y[last], rt.layer_norm(x[last].clone(), w, b, activation="relu"))
    del y
    y = rt.layer_norm(x, w, b, dropout=0.5, seed=8)
    assert torch.equal(y[last] == 0, ~kept((5, width), 0.5, 8, (rows - 5) * width))
    del y
    leaf = x[last].clone().requires_grad_()
    dx, = torch.autograd.grad(rt.layer_norm(leaf, w, b), leaf, leaf.detach())
    x.requires_grad_()
    assert torch.equal(torch.autograd.grad(rt.layer_norm(x, w, b), x, x.detach())[0][last], dx)
    x = x.detach()
    target = torch.arange(rows, device="cuda") % width
    each = rt.cross_entropy(x, target, reduction="none")
    assert torch.equal(each[last], rt.cross_entropy(x[last].clone(), target[last], reduction="none"))
    leaf = x[last].clone().requires_grad_()
    want, = torch.autograd.grad(rt.cross_entropy(leaf, target[last], reduction="sum"), leaf)
    x.requires_grad_()
    assert torch.equal(torch.autograd.grad(rt.cross_entropy(x, target, reduction="sum"), x)[0][last], want)


# ---------------------------------------------------------------------------------------------
# autograd
# ---------------------------------------------------------------------------------------------
def operators():
    """Each operator as a function of its matrix, first derivative only."""
    w, b = rand(12, seed=1), rand(12, seed=2)
    target = torch.arange(9, device="cuda") % 12
    return [lambda x: rt.layer_norm(x, w, b, activation="relu", dropout=0.3, seed=1), lambda x: rt.dropout(x, 0.3, x, seed=1),
            lambda x: rt.cross_entropy(x, target), lambda x: rt.cross_entropy(x, target, reduction="none")]


@pytest.mark.parametrize("which", range(4))
def test_nodes(which):
    f = operators()[which]
    x = rand(9, 12, seed=5).requires_grad_()
    # twice over a retained graph, then no more
    out = f(x)
    up = torch.ones_like(out)
    first, = torch.autograd.grad(out, x, up, retain_graph=True)
    first = first.clone()
    second, = torch.autograd.grad(out, x, up)
    assert torch.equal(first, second)
    if which != 1:  # (a dropout keeps nothing that could be gone)
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(out, x, up)
    # not twice differentiable
    grad, = torch.autograd.grad(f(x), x, up.clone().requires_grad_(), create_graph=True)
    assert torch.equal(grad, first)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grad.sum().backward()
    # an input that changed is refused (the dropout keeps none)
    changed = x.detach().clone().requires_grad_()
    inner = changed * 1
    out = f(inner)
    inner += 0
    if which == 1:
        torch.autograd.grad(out, changed, up)
    else:
        with pytest.raises(RuntimeError, match="inplace"):
            torch.autograd.grad(out, changed, up)
    # no forward-mode derivative
    import torch.autograd.forward_ad as ad
    with ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(ad.make_dual(x.detach(), torch.ones_like(x)))
    # a consumer that returns no gradient
    class Nothing(torch.autograd.Function):
        @staticmethod
        def forward(ctx, t):
            return t.clone()

        @staticmethod
        def backward(ctx, g):
            return None

    leaf = x.detach().clone().requires_grad_()
    Nothing.apply(f(leaf)).sum().backward()
    assert leaf.grad is not None and not leaf.grad.any()
    # without gradients there is no node
    with torch.no_grad():
        assert f(x).grad_fn is None
    # accumulation into a leaf's gradient, which is the leaf's own afterwards
    leaf = x.detach().clone().requires_grad_()
    for _ in range(2):
        out = f(leaf)
        out.backward(torch.ones_like(out))
    assert torch.equal(leaf.grad, first + first)


def test_traced_operators_replay():
    w, b = rand(12, seed=1), rand(12, seed=2)
    target = torch.arange(9, device="cuda") % 12
    for f in (lambda x: rt.layer_norm(x, w, b, activation="relu"), lambda x: rt.dropout(x, 0.3, seed=4),
              lambda x: rt.cross_entropy(x, target)):
        traced = torch.jit.trace(f, rand(9, 12, seed=5), check_trace=False)
        other = rand(9, 12, seed=6)
        assert torch.equal(traced(other), f(other))


# ---------------------------------------------------------------------------------------------
# streams, threads, graphs
# ---------------------------------------------------------------------------------------------
def step(x, w, b, target, key):
    h = rt.layer_norm(x, w, b, activation="relu", dropout=0.3, seed=key)
    loss = rt.cross_entropy(rt.dropout(h, 0.2, x, key), target)
    return [loss.detach()] + list(torch.autograd.grad(loss, (x, w, b)))


def step_inputs(rows=3000, width=40, seed=0):
    x, w, b = rand(rows, width, seed=seed).requires_grad_(), rand(width, seed=seed + 1).requires_grad_(), rand(width, seed=seed + 2).requires_grad_()
    return x, w, b, torch.arange(rows, device="cuda") % width


def test_steps_have_the_same_bits_each_time():
    for rows, width in ((3000, 40), (50, 3001), (40000, 128)):
        inputs = step_inputs(rows, width)
        want = step(*inputs, 7)
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(step(*inputs, 7), want))


def test_steps_on_streams_and_threads():
    inputs = [step_inputs(seed=10 * i) for i in range(4)]
    want = [step(*one, 7) for one in inputs]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = step(*inputs[i], 7)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_calls_of_several_threads_with_rows_of_several_lengths():
    """Calls whose kernels are one and the same and take different amounts of shared memory, from two threads at once."""
    for dtype, lengths in ((BF16, (30000, 50001)), (F32, (720, 768)), (F32, (13000, 25000))):
        cases = []
        for classes in lengths:
            logits, target = loss_case(40, classes, dtype)
            cases.append((logits, target, rt.cross_entropy(logits, target)))
        torch.cuda.synchronize()
        failures = []

        def work(logits, target, want):
            try:
                with torch.cuda.stream(torch.cuda.Stream()):
                    for _ in range(1500):
                        got = rt.cross_entropy(logits, target)
                    assert torch.equal(got, want)
            except Exception as e:  # (an assertion in a thread ends the thread alone)
                failures.append(e)

        threads = [threading.Thread(target=work, args=case) for case in cases]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not failures, failures


def test_captured_steps():
    """A step captured twice, replayed in turn, each time with another key and other features."""
    graphs = []
    side = torch.cuda.Stream()
    for seed in (0, 50):
        x, w, b, target = step_inputs(seed=seed)
        key = torch.tensor([3], device="cuda")
        with torch.cuda.stream(side):
            step(x, w, b, target, key)
        torch.cuda.synchronize()
        recorded = torch.cuda.CUDAGraph()
        with torch.cuda.graph(recorded, stream=side):
            out = step(x, w, b, target, key)
        graphs.append((recorded, out, (x, w, b, target), key))
    for k in range(4):
        for recorded, out, inputs, key in graphs:
            with torch.no_grad():
                key.fill_(100 + k)
                inputs[0].mul_(1.01)
        for recorded, *_ in graphs:
            recorded.replay()
        torch.cuda.synchronize()
        for recorded, out, inputs, key in graphs:
            # (a captured loss computes its gradient from the saved statistics, with the same arithmetic)
            assert all(torch.equal(a, b) for a, b in zip(out, step(*inputs, 100 + k)))
            recorded.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, step(*inputs, key)))


def test_a_captured_backward_pass_may_be_replayed_alone():
    logits, target = loss_case(100, 47)
    logits.requires_grad_()
    up = torch.ones((), device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.autograd.grad(rt.cross_entropy(logits, target), logits, up)
    torch.cuda.synchronize()
    forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(forward, stream=side):
        loss = rt.cross_entropy(logits, target)
    with torch.cuda.graph(backward, stream=side, pool=forward.pool()):
        grad, = torch.autograd.grad(loss, logits, up)
    forward.replay()
    for value in (1.0, 4.0, 4.0, 1.0):
        up.fill_(value)
        backward.replay()
        torch.cuda.synchronize()
        leaf = logits.detach().clone().requires_grad_()
        unit, = torch.autograd.grad(rt.cross_entropy(leaf, target), leaf, torch.tensor(value, device="cuda"))
        assert torch.equal(grad, unit)
        grad.fill_(0.0)


def test_fresh_keys_inside_a_capture():
    x = torch.ones(5000, device="cuda", requires_grad=True)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    recorded = torch.cuda.CUDAGraph()
    with torch.cuda.graph(recorded, stream=side):
        y = rt.dropout(x, 0.5)
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        z = rt.layer_norm(torch.zeros(5, 1000, device="cuda"), None, torch.ones(1000, device="cuda"), dropout=0.5)
    seen = []
    for _ in range(3):
        recorded.replay()
        torch.cuda.synchronize()
        assert torch.equal(dx, y.detach()) and abs(int((y == 0).sum()) - 2500) < 200
        seen += [y.detach().clone(), z.view(-1).clone()]
    assert all(not torch.equal(a, b) for i, a in enumerate(seen) for b in seen[:i])


def test_a_capture_over_leaves_of_a_living_eager_graph_is_refused():
    x, w, b, target = step_inputs()
    living = rt.layer_norm(x, w, b)  # holds the leaves' accumulators, on the default stream
    for f in (lambda: rt.layer_norm(x, w, b), lambda: rt.dropout(x, 0.5, seed=1), lambda: rt.cross_entropy(x, target)):
        recorded = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="still lives"):
            with torch.cuda.graph(recorded, stream=torch.cuda.Stream()):
                keep_something_recorded = torch.zeros(1, device="cuda")
                f()
        torch.cuda.synchronize()
    del living
    recorded = torch.cuda.CUDAGraph()
    with torch.cuda.graph(recorded):
        out = step(x, w, b, target, 5)
    recorded.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(out, step(x, w, b, target, 5)))


FIRST_CALLS_IN_A_CAPTURE = """
import torch
from compressgnn_b200 import runtime as rt
x = torch.randn(300, 130, device="cuda", dtype=torch.float64, requires_grad=True)
target = torch.arange(300, device="cuda") % 130
side = torch.cuda.Stream()
torch.cuda.synchronize()
recorded = torch.cuda.CUDAGraph()
with torch.cuda.graph(recorded, stream=side):
    loss = rt.cross_entropy(rt.dropout(rt.layer_norm(x, dropout=0.2, seed=3), 0.1, seed=4), target)
    dx, = torch.autograd.grad(loss, x)
recorded.replay()
torch.cuda.synchronize()
again = rt.cross_entropy(rt.dropout(rt.layer_norm(x, dropout=0.2, seed=3), 0.1, seed=4), target)
assert torch.equal(again, loss) and torch.equal(torch.autograd.grad(again, x)[0], dx)
print("same")
"""


def test_first_calls_of_a_process_inside_a_capture():
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS_IN_A_CAPTURE], cwd=Path(__file__).resolve().parents[1],
                          capture_output=True, text=True, timeout=240)
    assert done.returncode == 0 and done.stdout.strip() == "same", done.stderr[-2000:]


def test_masks_beyond_the_lower_half_of_the_counter():
    """Blocks of four words beyond 2^32 of them, and a row that lies on both sides: 2^34 elements (32 GiB of fp16 out, the
    rows in share their memory)."""
    p, key, width = 0.5, 2**40 + 9, 4100
    rows = 2**34 // width + 3
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    x = rand(1, width, dtype=F16).expand(rows, width)
    y = rt.layer_norm(x, None, torch.full((width,), 30.0, dtype=F16, device="cuda"), dropout=p, seed=key)
    for r in (0, 2**34 // width - 1, 2**34 // width, rows - 1):
        assert torch.equal(y[r] != 0, kept((width,), p, key, r * width)), r


# ---------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------
def graph_data(n=600, width=24):
    from compressgnn_b200 import offline as off
    from compressgnn_b200.loader import CompressgnnData
    v, e = off.generate_copy_graph(n, 2.1, 4.0, 200, 0.7, 32, 8, seed=3)
    x = np.random.default_rng(3).standard_normal((n, width)).astype(np.float32)
    mask = np.ones(n, bool)
    data = CompressgnnData(x, (v, e), np.zeros(n, np.int64), mask, mask, mask, min_pair_frequency=3, threshold=1, min_edge=10)
    data.to("cuda")
    return data


@pytest.mark.parametrize("transformation", [False, True])
def test_a_model_of_them(transformation):
    """Three layers with normalisation, dropout and residual connections in fp64, against the same model of torch's
    operators: the chain amplifies roundings (2^-53 a step) by far less than 10^6, so 10^-9 of a gradient's size is theirs."""
    data = graph_data()
    torch.manual_seed(1)
    model = GCN(24, 7, hidden_features=24, dropout=0.3, use_transformation=transformation, param_H=8, num_layers=3, norm="layer",
                residual=True).cuda().double()
    x = data.x.double()
    target = torch.arange(data.vertex_cnt, device="cuda") % 7
    target[::3] = IGNORED
    torch.manual_seed(5)
    loss = model.loss(x, data.edge_index, target)
    parameters = list(model.parameters())
    grads = torch.autograd.grad(loss, parameters)
    torch.manual_seed(5)
    h, propagate = x, KPropagate()
    for i, layer in enumerate(model.layers):
        out = propagate(h, data.edge_index)
        if transformation:
            kept_assignment = layer.cluster.assignment(out)
            index, counts = kept_assignment.index, kept_assignment.counts
            sums = torch.zeros(counts.numel(), out.size(1), dtype=F64, device="cuda").index_add(0, index, out)
            out = (sums / counts.clamp_min(1).double()[:, None])[index]
        out = torch.nn.functional.linear(out, layer.lin.weight, layer.lin.bias)
        if i < 2:
            mean, var = out.mean(1, keepdim=True), out.var(1, correction=0, keepdim=True)
            out = torch.relu((out - mean) / torch.sqrt(var + layer.norm.eps) * layer.norm.weight + layer.norm.bias)
            key = int(torch.randint(0, 2**63 - 1, (1,)))
            h = h + torch.where(kept(out.shape, 0.3, key), out / 0.7, 0.0)
        else:
            h = out
    want = torch.nn.functional.nll_loss(h.log_softmax(1), target, ignore_index=IGNORED)
    assert abs(float(loss - want)) <= 1e-12 * abs(float(want))
    for (name, _), got, ref in zip(model.named_parameters(), grads, torch.autograd.grad(want, parameters)):
        assert (got - ref).abs().max() <= 1e-9 * ref.abs().max() + 1e-15, name
    model.eval()
    scores = model(x, data.edge_index)
    assert torch.equal(scores, model.inference(x, data.edge_index))
    assert torch.allclose(model.loss(x, data.edge_index, target),
                          torch.nn.functional.nll_loss(scores, target, ignore_index=IGNORED), rtol=1e-12)


def test_modules():
    x = rand(50, 32, seed=1).requires_grad_()
    norm, drop, loss = LayerNorm(32, activation="relu").cuda(), Dropout(0.4), CrossEntropy(reduction="sum")
    target = torch.arange(50, device="cuda") % 32
    torch.manual_seed(2)
    got = loss(drop(norm(x, dropout=0.1), residual=x), target)
    torch.manual_seed(2)
    keys = [int(torch.randint(0, 2**63 - 1, (1,))) for _ in range(2)]
    h = rt.layer_norm(x, norm.weight, norm.bias, activation="relu", dropout=0.1, seed=keys[0])
    assert torch.equal(got, rt.cross_entropy(rt.dropout(h, 0.4, x, seed=keys[1]), target, reduction="sum"))
    got.backward()
    assert all(p.grad is not None for p in norm.parameters()) and x.grad is not None
    # a layer's hooks run once, with a residual stream too
    from compressgnn_b200.model import GNNLayer
    data, seen = graph_data(), []
    layer = GNNLayer(24, 24, activation="relu", norm="layer").cuda()
    layer.register_forward_hook(lambda module, given, out: seen.append(out))
    out = layer(data.x, data.edge_index, residual=data.x)
    assert len(seen) == 1 and torch.equal(out, layer(data.x, data.edge_index) + data.x)
    drop.eval()
    assert torch.equal(drop(h, residual=x), h + x) and LayerNorm(8, bias=False).bias is None


@pytest.mark.parametrize("training", [False, True])
def test_a_residual_of_another_shape_or_type(training):
    """What may be added outside of training may be added in training, with the same shape and type: the residual is
    broadcast and promoted as torch does."""
    from compressgnn_b200.model import GNNLayer
    data = graph_data()
    layer = GNNLayer(24, 24, activation="relu", norm="layer").cuda()
    drop = Dropout(0.4).train(training)
    x = rand(data.vertex_cnt, 24, seed=1)
    half = x.half()
    for value, residual in ((x, rand(1, 24, seed=2)), (x, rand(24, seed=2)), (x, rand(2, *x.shape, seed=2)), (x, rand(*x.shape, dtype=F64, seed=2)),
                            (half, rand(*x.shape, seed=2)), (x, half)):
        residual.requires_grad_()
        leaf = value.clone().requires_grad_()
        y = drop(leaf, residual=residual, seed=9)
        dropped = rt.dropout(value, 0.4, seed=9) if training else value
        want = dropped + residual.detach()
        assert y.dtype == want.dtype and torch.equal(y.detach(), want)
        dx, dr = torch.autograd.grad(y, (leaf, residual), torch.ones_like(y))
        times = y.numel() // value.numel()
        assert torch.equal(dx, (rt.dropout(torch.ones_like(value), 0.4, seed=9) if training else torch.ones_like(value)) * times)
        assert dr.shape == residual.shape and (dr == y.numel() // residual.numel()).all()
        if value is x and residual.dim() < 3:
            torch.manual_seed(4)
            out = layer(x, data.edge_index, dropout=0.4 if training else 0.0, residual=residual.detach())
            torch.manual_seed(4)
            plain = layer(x, data.edge_index)
            want = (rt.dropout(plain, 0.4) if training else plain) + residual.detach()
            # (in one pass the sum is rounded once, from a product that is not: one rounding of the product apart)
            assert out.dtype == want.dtype and (out - want).abs().max() <= 2.0**-24 * 2 * want.abs().max()


def test_a_training_loop_runs():
    """The training loop of the example in the documents runs, and every parameter gets a gradient."""
    data = graph_data()
    model = GCN(24, 7, hidden_features=32, num_layers=4, norm="layer", residual=True).cuda()
    opt = torch.optim.Adam(model.parameters(), lr=1e-3)
    target = torch.arange(data.vertex_cnt, device="cuda") % 7
    for _ in range(3):
        opt.zero_grad()
        loss = model.loss(data.x, data.edge_index, target)
        loss.backward()
        assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
        opt.step()
    assert torch.isfinite(loss)
    rt.raise_on_device_status()
