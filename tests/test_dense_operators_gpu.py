"""The dense layer and the optimiser step against their definitions in 64 bits.

Tolerances count roundings, from ``U``, half a step of the sums (2^-24; for fp64 2^-53), and ``half_step``, that of a result's type.

A product of ``n`` terms is off by at most ``(n + 32) U sum|a b|``: an fp32 sum one after the other makes n roundings.  A tensor
core's: fp32 operands go in as three bf16 numbers whose remainder is at most 2^-24 of them, the products left out are at
most 2 * 2^-24 of the term, and every 16 terms are added to their sum with a truncation of at most 2 U for the alignment of
each of 17 summands: 34 / 16 a term (the parts of lower order add 2^-8 of that).  So those sums count ``3 n``."""
import copy
import math
import subprocess
import sys
import threading
from pathlib import Path

import numpy as np
import pytest
import torch

from compressgnn_b200 import optim
from compressgnn_b200 import runtime as rt
from compressgnn_b200.layer import Linear
from compressgnn_b200.model import GCN

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
TYPES = [F32, F64, BF16, F16]
E4M3 = torch.float8_e4m3fn


def unit(dtype):
    return 2.0**-53 if dtype == F64 else 2.0**-24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
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


def kept(shape, p, key):
    n = int(np.prod(shape))
    bound = min(int(p * 2**32), 2**32 - 1)
    return torch.from_numpy(words(0, n, key & (2**64 - 1)) >= np.uint64(bound)).view(shape).cuda()


# ---------------------------------------------------------------------------------------------
# dense layer
# ---------------------------------------------------------------------------------------------
def terms(n, u):
    return (3 * n + 32) * u


def check_linear(x, weight, bias=None, relu=False, p=0.0, residual=None, key=987654321, what=""):
    dtype = x.dtype
    u, h = unit(dtype), half_step(dtype)
    leaves = [t for t in (x, weight, bias, residual) if t is not None]
    for t in leaves:
        t.requires_grad_()
    with torch.no_grad():
        positive = rt.linear(x, weight, bias, "relu") > 0
    y = rt.linear(x, weight, bias, "relu" if relu else None, p, residual, key)
    inner, outer = weight.size(1), weight.size(0)
    assert y.shape == (*x.shape[:-1], outer) and y.dtype == dtype and y.is_contiguous()
    grad = rand(*y.shape, dtype=dtype, seed=9, scale=0.1)
    grads = torch.autograd.grad(y, leaves, grad)
    with torch.no_grad():
        wide, w = x.double().reshape(-1, inner), weight.double()
        z, size = wide @ w.t(), wide.abs() @ w.abs().t()
        if bias is not None:
            z, size = z + bias.double(), size + bias.double().abs()
        z, size = z.view(y.shape), size.view(y.shape)
        factor = torch.ones_like(z) if not relu else positive.double()
        if p:
            factor = factor * kept(y.shape, p, key).double() / (1 - p)
        added = residual.double() if residual is not None else torch.zeros_like(z)
        want = z * factor + added
        error = terms(inner, u) * size * factor
        within(y.detach(), want, error + 2 * u * (z * factor).abs() + u * added.abs() + (h + u) * (want.abs() + error) + least(dtype),
               f"{what} y")
        g = (grad.double() * factor).reshape(-1, outer)
        rows = g.size(0)
        rest = list(grads)

        def one(want, size, n, name):
            got = rest.pop(0)
            assert got.dtype == dtype and got.is_contiguous(), name
            error = terms(n, u) * size
            within(got, want.view(got.shape), (error + (h + u) * (want.abs() + error) + least(dtype)).view(got.shape), f"{what} {name}")

        one(g @ w, g.abs() @ w.abs(), outer, "dx")
        one(g.t() @ wide, g.abs().t() @ wide.abs(), rows, "dweight")
        if bias is not None:
            one(g.sum(0), g.abs().sum(0), rows, "dbias")
        if residual is not None:
            assert torch.equal(rest.pop(0), grad), f"{what} dresidual"


SIZES = [(1, 1, 1), (1, 64, 64), (2, 3, 5), (5, 1000, 3), (17, 31, 1), (33, 64, 47), (64, 8, 130), (127, 129, 128), (128, 128, 128),
         (129, 65, 130), (300, 301, 173), (1000, 64, 7), (2708, 64, 47), (4097, 256, 128), (513, 1100, 260), (20001, 96, 64),
         (9000, 7, 9), (3000, 500, 16), (700, 2048, 1), (40000, 128, 256)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, inner, outer", SIZES)
def test_linear_at_sizes(dtype, rows, inner, outer):
    x = rand(rows, inner, dtype=dtype, seed=1, offset=0.2)
    weight = rand(outer, inner, dtype=dtype, seed=2, scale=inner**-0.5)
    bias = rand(outer, dtype=dtype, seed=3, scale=0.1)
    check_linear(x, weight, bias, what=f"{rows}x{inner}x{outer}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, inner, outer", [(7, 5, 3), (129, 65, 130), (513, 48, 257), (5000, 64, 128), (20001, 96, 61)])
@pytest.mark.parametrize("relu, p, added", [(True, 0.0, False), (False, 0.3, False), (True, 0.5, True), (False, 0.0, True)])
def test_linear_with_what_follows(dtype, rows, inner, outer, relu, p, added):
    x, weight = rand(rows, inner, dtype=dtype, seed=1), rand(outer, inner, dtype=dtype, seed=2, scale=inner**-0.5)
    residual = rand(rows, outer, dtype=dtype, seed=4) if added else None
    check_linear(x, weight, rand(outer, dtype=dtype, seed=3), relu, p, residual, what=f"relu {relu} p {p}")


# Calls that go to the tensor cores: their edges in rows and both widths, contractions of one chunk and of several segments, more
# tiles than multiprocessors, and weight gradients of few and of many splits.
TILE_SIZES = [(40000, 64, 72), (9001, 257, 129), (130, 1024, 1024), (129, 2051, 33), (1, 2048, 2056), (20000, 40, 136), (70001, 33, 47),
              (3000, 1030, 17), (5000, 300, 300), (150000, 16, 24), (19000, 128, 256), (300000, 8, 24), (2500, 512, 1000)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows, inner, outer", TILE_SIZES)
@pytest.mark.parametrize("relu, p, added", [(False, 0.0, False), (True, 0.3, True)])
def test_linear_on_tiles(dtype, rows, inner, outer, relu, p, added):
    x = rand(rows, inner, dtype=dtype, seed=1, offset=0.2)
    weight = rand(outer, inner, dtype=dtype, seed=2, scale=inner**-0.5)
    check_linear(x, weight, rand(outer, dtype=dtype, seed=3, scale=0.1), relu, p,
                 rand(rows, outer, dtype=dtype, seed=4) if added else None, what=f"{rows}x{inner}x{outer}")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_linear_on_tiles_strides(dtype):
    rows, weight, bias = 40000, rand(72, 64, dtype=dtype, seed=2, scale=0.1), rand(72, dtype=dtype, seed=3)
    base = rand(rows, 104, dtype=dtype, seed=1)
    # rows on vectors, on vectors of other lengths, between vectors, far apart, backwards in memory, on one place
    for x in (base[:, 8:72], base[:, 4:68], base[:, 3:67], rand(rows, 100, dtype=dtype, seed=4)[:, :64], base[::3, :64].repeat(3, 1),
              rand(64, rows, dtype=dtype, seed=5).t(), rand(1, 64, dtype=dtype, seed=6).expand(rows, 64), base[1:, 32:96]):
        check_linear(x.detach(), weight.detach(), bias.detach(), True, 0.25, what=str(x.stride()))
    # rows on vectors that end inside one
    check_linear(base[:, 8:68].detach(), weight[:, :60].contiguous().detach(), bias.detach(), True, 0.25, what="60 of 104")
    odd = rand(rows * 64 + 1, dtype=dtype, seed=7)[1:].view(rows, 64)
    oddly = rand(72 * 64 + 1, dtype=dtype, seed=8, scale=0.1)[1:].view(72, 64)
    check_linear(odd, oddly, bias.detach(), True, residual=rand(rows * 72 + 1, dtype=dtype, seed=9)[1:].view(rows, 72), what="odd addresses")
    check_linear(base[:, :64].detach().clone(), rand(64, 72, dtype=dtype, seed=10, scale=0.1).t().detach(), what="transposed weight")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("polls", [0, 1])
def test_linear_waits_that_run_out(dtype, polls):
    """A kernel that gives up a wait leaves NaN for what it has not computed and says so; the next one is as ever."""
    x, w, b = (t.requires_grad_() for t in (rand(30000, 96, dtype=dtype, seed=1), rand(128, 96, dtype=dtype, seed=2, scale=0.1),
                                             rand(128, dtype=dtype, seed=3)))
    grad = rand(30000, 128, dtype=dtype, seed=4)

    def both():
        y = rt.linear(x, w, b, "relu")  # (a dropped element would be a zero all the same)
        return [y.detach(), *torch.autograd.grad(y, (x, w, b), grad)]
    want = both()
    assert rt.device_status() == 0
    before = rt.lib().cgnn_linear_wait_limit(polls)
    try:
        got = both()
        torch.cuda.synchronize()
    finally:
        rt.lib().cgnn_linear_wait_limit(before)
    assert rt.device_status() == 2
    lost = [torch.isnan(g) for g in got]
    assert any(nan.any() for nan in lost)
    for g, v, nan in zip(got, want, lost):
        assert nan.all() if polls == 0 else torch.equal(g[~nan], v[~nan])
    for g, v in zip(both(), want):
        assert torch.equal(g, v)
    assert rt.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [40, 6000])
def test_linear_strides_and_dimensions(dtype, rows):
    base = rand(rows, 100, dtype=dtype, seed=1)
    weight = rand(33, 64, dtype=dtype, seed=2, scale=0.1)
    bias = rand(33, dtype=dtype, seed=3)
    for x in (base[:, 3:67], base[:, 32:96], base[::2, :64], rand(64, rows, dtype=dtype, seed=5).t(), base[1:, :64]):
        check_linear(x.detach(), weight.detach(), bias.detach(), True, 0.2, what=str(x.stride()))
    wide = rand(64, 33, dtype=dtype, seed=6).t()  # columns first
    check_linear(base[:, :64].detach().clone(), wide.detach(), None, what="transposed weight")
    check_linear(rand(3, rows // 8, 64, dtype=dtype, seed=7), weight.detach(), bias.detach(), True, 0.1,
                 rand(3, rows // 8, 33, dtype=dtype, seed=8), what="three dimensions")
    check_linear(rand(64, dtype=dtype, seed=9), weight.detach(), bias.detach(), what="one dimension")
    # every row the same one
    check_linear(rand(1, 64, dtype=dtype, seed=10).expand(rows, 64).detach(), weight.detach(), bias.detach(), what="rows on one place")
    # memory that begins between vectors
    odd = rand(rows * 64 + 1, dtype=dtype, seed=11)[1:].view(rows, 64)
    oddly = rand(33 * 64 + 1, dtype=dtype, seed=12, scale=0.1)[1:].view(33, 64)
    check_linear(odd, oddly, bias.detach(), True, what="odd addresses")


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_of_nothing(dtype):
    for rows, inner, outer in ((0, 8, 4), (5, 0, 4), (5, 8, 0), (0, 0, 0)):
        x, w, b = rand(rows, inner, dtype=dtype), rand(outer, inner, dtype=dtype), rand(outer, dtype=dtype)
        for t in (x, w, b):
            t.requires_grad_()
        y = rt.linear(x, w, b, "relu", 0.25, seed=3)
        assert y.shape == (rows, outer)
        if rows and outer:
            want = b.detach().double().clamp(min=0) * kept(y.shape, 0.25, 3) / 0.75
            within(y.detach(), want, 3 * half_step(dtype) * want.abs() + least(dtype), "the bias alone")
        dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
        assert dx.shape == x.shape and dw.shape == w.shape and db.shape == b.shape
        if not rows:
            assert not dw.any() and not db.any()
        if not outer:
            assert not dx.any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [300, 40000])
def test_linear_infinities_and_nan(dtype, rows):
    """They reach the outputs that they have a part in, as the formula says, and no others."""
    x, w = rand(rows, 70, dtype=dtype, seed=1), rand(50, 70, dtype=dtype, seed=2)
    w[:, 0] = 1.0  # exact in every type: an infinity times the rest of a split would be no number
    w[7, 1] = 0.0
    x[3, 0], x[5, 1], x[rows - 1, 69], x[8, 2] = math.inf, -math.inf, math.nan, torch.finfo(dtype).max
    w[8, 2] = 1.0
    w[20, 5] = math.inf
    x[11, 5] = 0.0
    got, want = rt.linear(x, w), x.double() @ w.double().t()
    narrowed = want.to(dtype)
    assert torch.equal(torch.isnan(got), torch.isnan(narrowed))
    special = ~torch.isfinite(narrowed) & ~torch.isnan(narrowed)
    sure = special & ~torch.isfinite(want)  # (a large finite sum may lie on either side of the type's end)
    assert torch.equal(got[sure], narrowed[sure])
    ordinary = torch.isfinite(want) & (want.abs() < torch.finfo(dtype).max / 4)
    size = torch.nan_to_num(x.double(), 0.0, 0.0, 0.0).abs() @ torch.nan_to_num(w.double(), 0.0, 0.0, 0.0).abs().t()
    bound = terms(70, unit(dtype)) * size + half_step(dtype) * want.abs() + least(dtype)
    assert ((got.double() - want).abs() <= bound)[ordinary].all()
    assert torch.equal(rt.linear(x, w, None, "relu").isnan(), narrowed.isnan())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_products_of_any_magnitude(dtype):
    """Terms far apart, and very large and very small ones: the split of an fp32 number spans its whole range."""
    for scale_x, scale_w in ((1e18, 1e-18), (1e-15, 1e-15), (1e15, 1e15), (1e-3, 1e4)):
        x, w = rand(5000, 130, dtype=dtype, seed=1, scale=scale_x), rand(64, 130, dtype=dtype, seed=2, scale=scale_w)
        check_linear(x, w, what=f"{scale_x} {scale_w}")
    x = rand(5000, 130, dtype=dtype, seed=1)
    x[:, ::3] *= 1e6
    check_linear(x, rand(64, 130, dtype=dtype, seed=2), what="columns far apart")
    # sums of one sign, where truncations would add up
    check_linear(rand(20000, 1000, dtype=dtype, seed=3).abs(), rand(64, 1000, dtype=dtype, seed=4).abs(), what="one sign")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_linear_is_deterministic_and_rows_do_not_touch_each_other(dtype):
    x, w, b = rand(30001, 136, dtype=dtype, seed=1), rand(72, 136, dtype=dtype, seed=2), rand(72, dtype=dtype, seed=3)
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    grad = rand(30001, 72, dtype=dtype, seed=4)

    def once():
        y = rt.linear(x, w, b, "relu", 0.3, seed=5)
        return [y.detach(), *torch.autograd.grad(y, (x, w, b), grad)]
    for a, c in zip(once(), once()):
        assert torch.equal(a, c)
    with torch.no_grad():
        y = rt.linear(x, w, b)
        other = x.clone()
        other[:30000] = math.nan
        assert torch.equal(rt.linear(other, w, b)[30000:], y[30000:])


def test_linear_beyond_32_bits():
    """More elements than 32 bits count, in the output, its mask and gradient, and in the input."""
    rows, last = 2_200_000, slice(2_199_900, None)
    x = torch.ones(rows, 16, dtype=BF16, device="cuda")
    x[last] = rand(100, 16, dtype=BF16, seed=1)
    w = rand(1000, 16, dtype=BF16, seed=2)
    x.requires_grad_()
    y = rt.linear(x, w, None, "relu")
    assert y.numel() > 2**31
    with torch.no_grad():
        z = x[last].double() @ w.double().t()
        within(y[last].detach(), z.clamp(min=0), terms(16, 2.0**-24) * (x[last].double().abs() @ w.double().abs().t()) +
               half_step(BF16) * z.abs() + least(BF16), "the last rows")
        assert torch.equal(y[1000], y[0]) and torch.equal(y[2_000_000], y[0])
    dx, = torch.autograd.grad(y.sum(), x)
    want = (y[last].detach() > 0).double() @ w.double()
    within(dx[last], want, terms(1000, 2.0**-24) * w.double().abs().sum(0) + half_step(BF16) * want.abs() + least(BF16), "dx")
    del y, dx
    wide = torch.zeros(rows, 1000, dtype=BF16, device="cuda")
    wide[-1], wide[0] = 2.0, 1.0
    v = rand(16, 1000, dtype=BF16, seed=3).requires_grad_()
    y = rt.linear(wide, v)
    with torch.no_grad():
        assert torch.equal(y[1], torch.zeros_like(y[1]))
        within(y[-1], 2 * v.double().sum(1), terms(1000, 2.0**-24) * 2 * v.double().abs().sum(1) + half_step(BF16) * y[-1].double().abs() +
               least(BF16), "wide")
    dv, = torch.autograd.grad(y, v, torch.ones_like(y))
    assert torch.equal(dv, torch.full_like(dv, 3.0))


def test_linear_dropout_is_the_dropout_operators():
    for shape, outer in (((300, 40), 31), ((20000, 64), 128), ((20000, 64), 47)):
        x, w = rand(*shape, seed=1), rand(outer, shape[1], seed=2)
        dropped = rt.linear(x, w, dropout=0.4, seed=77) == 0
        assert torch.equal(dropped, rt.dropout(torch.ones(shape[0], outer, device="cuda"), 0.4, seed=77) == 0)
    for rows in (50, 20000):  # a probability that drops nothing
        a, b = (rand(rows, 64, seed=3).requires_grad_() for _ in range(2))
        y, z = rt.linear(a, w, dropout=1e-12), rt.linear(b, w)
        assert torch.equal(y, z) and torch.equal(torch.autograd.grad(y.sum(), a)[0], torch.autograd.grad(z.sum(), b)[0])
    key = torch.tensor([77], device="cuda")
    assert torch.equal(rt.linear(x, w, dropout=0.4, seed=key), rt.linear(x, w, dropout=0.4, seed=77))
    torch.manual_seed(3)
    a = rt.linear(x, w, dropout=0.4)
    b = rt.linear(x, w, dropout=0.4)
    torch.manual_seed(3)
    assert torch.equal(a, rt.linear(x, w, dropout=0.4)) and not torch.equal(a, b)


@pytest.mark.parametrize("rows, inner, outer", [(6, 5, 4), (40, 70, 33)])
def test_linear_gradients_against_differences(rows, inner, outer):
    x, w, b, r = (rand(*s, dtype=F64, seed=i).requires_grad_() for i, s in
                  enumerate(((rows, inner), (outer, inner), (outer,), (rows, outer))))
    assert torch.autograd.gradcheck(lambda *a: rt.linear(a[0], a[1], a[2], None, 0.3, a[3], 5), (x, w, b, r))
    with torch.no_grad():  # away from the border of the ReLU
        z = x @ w.t() + b
        b += 0.0
        keep = (z.abs() > 1e-3).all(1)
    x = x.detach()[keep].requires_grad_()
    assert torch.autograd.gradcheck(lambda a, v, c: rt.linear(a, v, c, "relu"), (x, w, b))


def test_linear_only_what_is_asked_for():
    x, w, b = rand(5000, 64, seed=1), rand(48, 64, seed=2), rand(48, seed=3)
    for which in ((0,), (1,), (2,), (0, 2), (1, 2), (0, 1, 2)):
        leaves = [t.clone().requires_grad_(i in which) for i, t in enumerate((x, w, b))]
        every = [t.clone().requires_grad_() for t in (x, w, b)]
        asked = torch.autograd.grad(rt.linear(*leaves, "relu", 0.2, seed=4).square().sum(), [leaves[i] for i in which])
        full = torch.autograd.grad(rt.linear(*every, "relu", 0.2, seed=4).square().sum(), every)
        for g, i in zip(asked, which):
            within(g, full[i], 1e-6 * full[i].abs() + 1e-5 * full[i].abs().max(), f"{which}")
    # a broadcast incoming gradient, and a graph that is kept
    y = rt.linear(*every)
    first = torch.autograd.grad(y.sum(), every, retain_graph=True)
    again = torch.autograd.grad(y, every, torch.ones_like(y))
    assert all(torch.equal(a, c) for a, c in zip(first, again))
    # in place between forward and backward
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    y = rt.linear(*leaves)
    with torch.no_grad():
        leaves[1].add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_linear_replayed_and_on_other_streams():
    x, w, b = rand(20000, 128, seed=1), rand(96, 128, seed=2, scale=0.1), rand(96, seed=3)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    key = torch.tensor([5], device="cuda")
    grad = rand(20000, 96, seed=4)

    def both():
        y = rt.linear(x, w, b, "relu", 0.3, seed=key)
        return [y.detach(), *torch.autograd.grad(y, leaves, grad)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = both()
        graphs.append((graph, out))
    with torch.no_grad():
        x.copy_(rand(20000, 128, seed=11))
        key.fill_(9)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    want = both()
    for _, out in graphs:
        for a, c in zip(out, want):
            assert torch.equal(a, c)
    results = {}

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            results[i] = both()
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for got in results.values():
        assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_linear_traced():
    w, b = rand(72, 64, seed=2), rand(72, seed=3)
    traced = torch.jit.trace(lambda a: rt.linear(a, w, b, "relu"), (rand(2000, 64, seed=1),))
    x = rand(3000, 64, seed=4).requires_grad_()
    y = traced(x)
    assert torch.equal(y, rt.linear(x, w, b, "relu"))
    grads = [torch.autograd.grad(f(x).square().sum(), x)[0] for f in (traced, lambda a: rt.linear(a, w, b, "relu"))]
    assert torch.equal(*grads)


FIRST = """
import sys, torch
sys.path.insert(0, {root!r})
from compressgnn_b200 import runtime as rt
x, w, b = (torch.randn(*s, device="cuda").requires_grad_() for s in ((30000, 64), (72, 64), (72,)))
p, g, m, v = (torch.randn(5000, device="cuda") for _ in range(4))
v.square_()
steps = [torch.zeros((), dtype=torch.int64, device="cuda")]
grad, before = torch.randn(30000, 72, device="cuda"), p.clone()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = rt.linear(x, w, b, "relu", 0.0)
    grads = torch.autograd.grad(y, (x, w, b), grad)
    rt.adamw_step([p], [g], [m], [v], steps, max_norm=1.0)
graph.replay()
torch.cuda.synchronize()
y = y.detach().clone()
assert torch.equal(y, rt.linear(x, w, b, "relu").detach()) and int(steps[0]) == 1 and not torch.equal(p, before)
z = rt.linear(x, w, b, "relu")
assert all(torch.equal(a, c) for a, c in zip(grads, torch.autograd.grad(z, (x, w, b), grad)))
"""


def test_first_calls_inside_a_capture():
    root = Path(__file__).resolve().parents[1]
    done = subprocess.run([sys.executable, "-c", FIRST.format(root=str(root))], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_linear_refuses():
    x, w, b = rand(4, 8), rand(3, 8), rand(3)
    wrong = [(x, w.t(), b, None, "weight"), (x, w.half(), b, None, "weight"), (x, w.cpu(), b, None, "weight"), (x, w, b[:2], None, "bias"),
             (x, w, b.half(), None, "bias"), (x, w, b.cpu(), None, "bias"), (x, w, b, rand(4, 8), "residual"),
             (x, w, b, rand(4, 3).half(), "residual"), (x, w, b, rand(3), "residual"), (x.int(), w, b, None, "only float32"),
             (x, w[0], b, None, "weight"), (torch.tensor(1.0, device="cuda"), w, b, None, "dimension")]
    for a, c, d, r, message in wrong:
        with pytest.raises(RuntimeError, match=message):
            rt.linear(a, c, d, residual=r)
    for p in (1.0, -0.1, math.nan):
        with pytest.raises(RuntimeError, match="probability"):
            rt.linear(x, w, b, dropout=p)
    with pytest.raises(RuntimeError, match="seed"):
        rt.linear(x, w, b, dropout=0.5, seed=torch.tensor([1.0], device="cuda"))
    with pytest.raises(RuntimeError, match="twice"):
        leaf = x.clone().requires_grad_()
        g, = torch.autograd.grad(rt.linear(leaf, w).square().sum(), leaf, create_graph=True)
        g.sum().backward()


def test_linear_beside_an_eager_graph_of_its_leaves():
    """A capture over leaves whose eager graph still lives on another stream is refused before anything is recorded."""
    w = rand(5, 8).requires_grad_()
    x = rand(4, 8)
    y = rt.linear(x, w)
    y.sum().backward(retain_graph=True)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(graph):
            rt.linear(x, w)
    del y


def test_linear_module_adds_any_residual():
    layer = Linear(16, 8, activation="relu").cuda()
    x = rand(30, 16)
    for residual in (rand(30, 8), rand(8), rand(30, 8, dtype=F64)):
        got = layer(x, residual=residual)
        want = torch.relu(torch.nn.functional.linear(x.double(), layer.weight.double(), layer.bias.double())) + residual.double()
        assert got.dtype == torch.result_type(x, residual)
        within(got.detach(), want.detach(), 1e-5 * (1 + want.detach().abs()), "module")


# ---------------------------------------------------------------------------------------------
# optimiser step
# ---------------------------------------------------------------------------------------------
B1, B2 = 0.9, 0.999
TENSOR_KEY, STEP_KEY = 0x9E3779B97F4A7C15, 0xD1342543DE82EF95


def tensors(shapes, dtype, seed=0, scale=1.0):
    return [rand(*s, dtype=dtype, seed=seed + i, scale=scale) for i, s in enumerate(shapes)]


def step_count(n, done):
    return list(torch.full((n,), done, dtype=torch.int64, device="cuda").unbind())


def check_step(params, grads, done=3, lr=1e-2, eps=1e-8, decay=0.1, max_norm=None):
    """Moments of full width against the formulas."""
    wide = [F64 if p.dtype == F64 else F32 for p in params]
    first = [rand(*p.shape, dtype=w, seed=50 + i, scale=0.1) for i, (p, w) in enumerate(zip(params, wide))]
    second = [rand(*p.shape, dtype=w, seed=80 + i, scale=0.1).square() for i, (p, w) in enumerate(zip(params, wide))]
    before = [[t.to(F64, copy=True) for t in ts] for ts in (params, grads, first, second)]  # (the step writes in place)
    steps = step_count(len(params), done)
    norm = rt.adamw_step(params, grads, first, second, steps, lr, (B1, B2), eps, decay, max_norm)
    t, clip, clip_off = done + 1, 1.0, 0.0
    if max_norm is not None:
        exact = math.sqrt(sum(float(g.square().sum()) for g in before[1]))
        assert abs(float(norm) - exact) <= 2 * 2.0**-24 * exact
        clip, clip_off = min(1.0, max_norm / (exact + 1e-6)), 4.0
    else:
        assert norm is None
    for i, (p, g, m, v) in enumerate(zip(*before)):
        u, h = unit(params[i].dtype), half_step(params[i].dtype)
        g = g * clip
        m1, m_size = B1 * m + (1 - B1) * g, B1 * m.abs() + (1 - B1) * g.abs()
        v1 = B2 * v + (1 - B2) * g * g
        # a constant, a product and a sum are rounded, a clipped gradient twice more
        within(first[i], m1, (4 + clip_off) * u * m_size + 1e-45, f"m {i}")
        within(second[i], v1, (6 + 2 * clip_off) * u * v1 + 1e-45, f"v {i}")
        # (1 - B2**t would lose its digits: a power near one is rounded by U, 250 U of the difference at t = 4)
        c1, c2 = -math.expm1(t * math.log(B1)), -math.expm1(t * math.log(B2))
        update = lr / c1 * m1 / ((v1 / c2).sqrt() + eps)
        off = lr / c1 * m_size / ((v1 / c2).sqrt() + eps) * (24 + 2 * clip_off) * u
        want = p * (1 - lr * decay) - update
        within(params[i], want, 4 * u * (p.abs() + update.abs()) + off + (h + u) * want.abs() + least(params[i].dtype), f"p {i}")
        assert int(steps[i]) == t


SHAPES = [(7,), (1,), (300, 41), (256,), (64, 64), (5000, 33), (2048,), (0,), (2049,), (3, 5, 7)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("max_norm", [None, 1.0, 1e9])
def test_step_against_the_formulas(dtype, max_norm):
    check_step(tensors(SHAPES, dtype), tensors(SHAPES, dtype, 30, 0.3), max_norm=max_norm)
    check_step(tensors(SHAPES, dtype), tensors(SHAPES, dtype, 30, 0.3), done=0, decay=0.0, max_norm=max_norm)
    check_step(tensors(SHAPES, dtype), tensors(SHAPES, dtype, 30, 0.3), done=10**6, max_norm=max_norm)


def test_step_of_many_and_mixed_tensors():
    shapes = [(1 + (i * 37) % 300,) for i in range(650)]
    check_step(tensors(shapes, F32), tensors(shapes, F32, 1000), max_norm=5.0)
    mixed = [(shape, TYPES[i % 4]) for i, shape in enumerate(SHAPES + SHAPES)]
    check_step([rand(*s, dtype=d, seed=i) for i, (s, d) in enumerate(mixed)], [rand(*s, dtype=d, seed=99 + i) for i, (s, d) in enumerate(mixed)],
               max_norm=3.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_step_on_odd_addresses(dtype):
    def odd(n, seed):
        return rand(n + 1, dtype=dtype, seed=seed)[1:]
    check_step([odd(1000, 1), odd(4096, 2), rand(4096, dtype=dtype)], [odd(1000, 3), odd(4096, 4), odd(4096, 5)], max_norm=1.0)
    around = rand(5000, dtype=dtype, seed=6)  # what lies beside a parameter stays
    whole = around.clone()
    p = around[1000:3333]
    check_step([p], [rand(2333, dtype=dtype, seed=7)])
    assert torch.equal(around[:1000], whole[:1000]) and torch.equal(around[3333:], whole[3333:]) and not torch.equal(p, whole[1000:3333])


def test_step_rates_of_their_own():
    shapes = [(500,), (3000,), (64, 65)]
    rates, decays = [1e-2, torch.tensor([2e-2], device="cuda"), 0.0], [0.0, 0.1, 0.2]
    params, grads = tensors(shapes, F32), tensors(shapes, F32, 9)
    together = [p.clone() for p in params]
    state = [tensors(shapes, F32, 20), [t.square() for t in tensors(shapes, F32, 40)]]
    rt.adamw_step(together, grads, [t.clone() for t in state[0]], [t.clone() for t in state[1]], step_count(3, 4), rates,
                  weight_decay=decays)
    for i, p in enumerate(params):
        rt.adamw_step([p], [grads[i]], [state[0][i].clone()], [state[1][i].clone()], step_count(1, 4),
                      float(rates[i]) if i != 1 else 0.02, weight_decay=decays[i])
        within(together[i], p, 2.0**-22 * p.abs().double(), f"{i}")  # (a rate of 0.02 in 32 bits)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_step_with_gradients_that_are_no_numbers(bad):
    grads = tensors([(300,), (10,)], F32, 5)
    grads[0][7] = bad
    params = tensors([(300,), (10,)], F32)
    ours = [p.clone() for p in params]
    first, second = ([torch.zeros_like(p) for p in params] for _ in range(2))
    rt.adamw_step(ours, grads, first, second, step_count(2, 0))
    assert torch.isnan(ours[0][7]) and int((~torch.isfinite(ours[0])).sum()) == 1 and torch.isfinite(ours[1]).all()
    clipped = [p.clone() for p in params]
    norm = rt.adamw_step(clipped, grads, [torch.zeros_like(p) for p in params], [torch.zeros_like(p) for p in params],
                         step_count(2, 0), max_norm=1.0)
    assert not torch.isfinite(norm)
    if math.isnan(bad):  # as every gradient times a factor that is no number
        assert all(torch.isnan(p).all() for p in clipped)
    eight, scales = ([torch.zeros(300, dtype=torch.uint8, device="cuda").view(E4M3)] for _ in range(2)), None
    first, second = eight
    scales = [[torch.ones(2, device="cuda")], [torch.ones(2, device="cuda")]]
    rt.adamw_step([params[0]], [grads[0]], first, second, step_count(1, 0), exp_avg_scales=scales[0], exp_avg_sq_scales=scales[1])
    for t in (first[0], second[0]):  # the others of its block are what they were
        assert torch.isnan(t.float()[7]) and int(torch.isnan(t.float()).sum()) == 1 and (t.float()[:7] != 0).any()


def exponents(blocks):
    fraction, exponent = torch.frexp(blocks.abs().amax(1))
    return torch.where(fraction == 0, -117, (exponent - 9 + (fraction > 0.875)).clamp(min=-117))


def rounded(values, random16, root):
    """Stochastic rounding to e4m3 in units of the block's scale, from 64-bit arithmetic on the fp32 values."""
    n = values.numel()
    blocks = torch.nn.functional.pad(values.reshape(-1), (0, -n % 256)).view(-1, 256)
    scale = torch.exp2(exponents(blocks).double())
    size = (blocks.double().abs() / scale[:, None]).view(-1)[:n]
    step = torch.exp2(torch.floor(torch.log2(size.clamp(min=2.0**-20))).clamp(min=-6) - 3)
    code = torch.floor(size / step + torch.from_numpy(random16.astype(np.float64)).cuda() / 65536) * step
    if root:
        code = torch.where((size > 0) & (code == 0), 2.0**-9, code)
    return torch.copysign(code, values.reshape(-1).double()).view(values.shape), scale


def spread(codes, scale):
    return (codes.float().reshape(-1) * scale.repeat_interleave(256)[:codes.numel()]).view(codes.shape)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_step_with_moments_of_8_bits(dtype):
    """Codes and scales to the bit: the moments in fp32 are products and sums rounded one by one."""
    shapes = [(300, 41), (256,), (1,), (5000,), (0,), (2047,), (17, 129)]
    params = tensors(shapes, dtype)
    first, second = ([torch.zeros(s, dtype=torch.uint8, device="cuda").view(E4M3) for s in shapes] for _ in range(2))
    scales = [[torch.ones((p.numel() + 255) // 256, device="cuda") for p in params] for _ in range(2)]
    steps = step_count(len(shapes), 0)
    for done in range(4):
        grads = tensors(shapes, dtype, 100 + 31 * done, 0.02)
        if done == 2:
            grads[0][:13] = 0  # whole blocks without a gradient
            grads[3][100:4000] *= 1e-3
        old = [[spread(c, s) for c, s in zip(codes, sc)] for codes, sc in ((first, scales[0]), (second, scales[1]))]
        before = [p.double() for p in params]
        rt.adamw_step(params, grads, first, second, steps, 1e-2, exp_avg_scales=scales[0], exp_avg_sq_scales=scales[1], seed=2**63 + 5,
                      weight_decay=0.0)
        for i, g in enumerate(grads):
            g = g.float()
            c1, c2 = (torch.tensor(1.0 - b, dtype=F64).float().cuda() for b in (B1, B2))
            m = old[0][i] * torch.tensor(B1).cuda() + g * c1
            v = old[1][i] * old[1][i] * torch.tensor(B2).cuda() + g * g * c2
            key = (2**63 + 5 + i * TENSOR_KEY + done * STEP_KEY) % 2**64
            w = words(0, g.numel(), key).astype(np.uint32)
            for got, scale, values, bits, root in ((first[i], scales[0][i], m, w & 0xFFFF, False), (second[i], scales[1][i], v.sqrt(), w >> 16, True)):
                code, want_scale = rounded(values, bits, root)
                assert torch.equal(scale.double(), want_scale), (done, i, root)
                assert torch.equal(got.double(), code), (done, i, root)
            t = done + 1
            want = before[i] - 1e-2 / (1 - B1**t) * m.double() / ((v.double() / (1 - B2**t)).sqrt() + 1e-8)
            within(params[i], want, 24 * 2.0**-24 * (before[i].abs() + 1e-2 / (1 - B1**t) * 4) + half_step(dtype) * want.abs() +
                   least(dtype), f"p {i}")
            assert int(steps[i]) == t


def test_rounding_of_8_bits_has_the_right_mean():
    """Over many keys a moment's mean is the moment: 2^16 draws of a step s leave the mean within 5 s / 2 / 256 of it."""
    n = 65536
    values = torch.tensor([0.7, -0.33, 0.0101, 0.9, 1.0, -0.77, 0.05, 0.002], device="cuda").repeat(n // 8)
    first, second = (torch.zeros(n, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
    scales = [[torch.ones(n // 256, device="cuda")] for _ in range(2)]
    rt.adamw_step([torch.zeros(n, device="cuda")], [values], [first], [second], step_count(1, 0), exp_avg_scales=scales[0],
                  exp_avg_sq_scales=scales[1], seed=11)
    for codes, scale, exact in ((first, scales[0][0], values * (1 - B1)), (second, scales[1][0], values.abs() * (1 - B2)**0.5)):
        got = spread(codes, scale).double().view(-1, 8).mean(0)
        want = exact[:8].double()
        step = want.abs() / 8 + 2.0**-9 * float(scale[0])
        assert ((got - want).abs() <= 5 * step / 2 / (n / 8)**0.5 + 1e-6 * want.abs()).all()


def test_step_replayed_and_on_other_streams():
    shapes = [(3000, 17), (40,), (9000,)]
    for bits in (32, 8):
        params = [torch.nn.Parameter(t) for t in tensors(shapes, F32)]
        copies = [torch.nn.Parameter(p.detach().clone()) for p in params]
        for ps in (params, copies):
            for p, g in zip(ps, tensors(shapes, F32, 9)):
                p.grad = g
        opt, eager = (optim.AdamW(ps, lr=1e-2, max_norm=1.0, state_bits=bits) for ps in (params, copies))
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="outside of the capture"):
            with torch.cuda.graph(graph):
                opt.step()
        opt.step(), eager.step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
        for i in range(3):
            for ps in (params, copies):
                for p, g in zip(ps, tensors(shapes, F32, 70 + i)):
                    p.grad.copy_(g)
            graph.replay()
            eager.step()
        for p, q in zip(params, copies):
            assert torch.equal(p, q) and int(opt.state[p]["step"]) == 4
            assert torch.equal(opt.state[p]["exp_avg"].view(torch.uint8), eager.state[q]["exp_avg"].view(torch.uint8))
        assert torch.equal(opt.grad_norm, eager.grad_norm)


@pytest.mark.parametrize("eight", [False, True])
def test_step_beyond_32_bits(eight):
    n, tail = 2**31 + 5000, 4096
    p, g = (torch.full((n,), v, dtype=BF16, device="cuda") for v in (0.5, 0.01))
    p[-tail:], g[-tail:] = rand(tail, dtype=BF16, seed=1), rand(tail, dtype=BF16, seed=2, scale=0.01)
    part = p[-tail:].clone()
    if eight:
        first, second = (torch.zeros(n, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
        scales = [[torch.ones((n + 255) // 256, device="cuda")] for _ in range(2)]
    else:
        first, second = (torch.zeros(n, device="cuda") for _ in range(2))
        scales = [None, None]
    rt.adamw_step([p], [g], [first], [second], step_count(1, 0), exp_avg_scales=scales[0], exp_avg_sq_scales=scales[1])
    one = [torch.zeros(tail, device="cuda") for _ in range(2)]
    rt.adamw_step([part], [g[-tail:].clone()], [one[0]], [one[1]], step_count(1, 0))
    assert torch.equal(p[-tail:], part) and bool((p[:-tail] == p[0]).all())
    if not eight:
        assert torch.equal(first[-tail:], one[0]) and torch.equal(second[-tail:], one[1])


def test_steps_beside_each_other():
    """Two models stepped on two streams at once are what they are one after the other."""
    results = []
    for concurrent in (False, True):
        models = []
        for k in range(2):
            ps = [torch.nn.Parameter(t) for t in tensors([(4000, 33), (77,)], F32, 10 * k)]
            for p, g in zip(ps, tensors([(4000, 33), (77,)], F32, 100 + k)):
                p.grad = g
            models.append((ps, optim.AdamW(ps, max_norm=0.5, state_bits=8)))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in models] if concurrent else [torch.cuda.current_stream()] * 2
        for _ in range(5):
            for (ps, opt), stream in zip(models, streams):
                with torch.cuda.stream(stream):
                    opt.step()
        torch.cuda.synchronize()
        results.append([p.detach() for ps, _ in models for p in ps])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_step_refuses():
    p, g, m, v = (rand(10, seed=i) for i in range(4))
    t = step_count(1, 0)

    def call(params=[p], grads=[g], first=[m], second=[v], steps=t, **more):
        return rt.adamw_step(params, grads, first, second, steps, **more)
    eight, scale = torch.zeros(10, dtype=torch.uint8, device="cuda").view(E4M3), torch.ones(1, device="cuda")
    other = torch.zeros(10, dtype=torch.uint8, device="cuda").view(E4M3)
    refused = [
        (dict(grads=[]), "as many"), (dict(grads=[g[:5]]), "gradient"), (dict(grads=[g.half()]), "gradient"), (dict(grads=[g.cpu()]), "one device"),
        (dict(params=[p[::2]], grads=[g[::2]]), "contiguous"), (dict(grads=[rand(20)[::2]]), "contiguous"), (dict(first=[m.half()]), "moments"),
        (dict(first=[m[:3]]), "moments"), (dict(steps=[torch.tensor([0.0], device="cuda")]), "int64"),
        (dict(params=[p, p], grads=[g, g], first=[m, m + 0], second=[v, v + 0], steps=step_count(2, 0)), "share memory"),
        (dict(params=[p, g + 0], grads=[g, g], first=[m, m + 0], second=[v, v + 0], steps=t + t), "share memory"),
        (dict(first=[p]), "share memory"), (dict(betas=(1.0, 0.9)), "betas"), (dict(betas=(0.9, -0.1)), "betas"), (dict(lr=-1.0), "negative"),
        (dict(lr=math.nan), "negative"), (dict(eps=-1.0), "negative"), (dict(weight_decay=-1.0), "negative"), (dict(max_norm=-1.0), "negative"),
        (dict(max_norm=math.nan), "negative"), (dict(lr=torch.tensor([1.0], device="cuda", dtype=F64)), "float32"),
        (dict(lr=torch.tensor([1.0])), "float32"), (dict(lr=[0.1, 0.1]), "as many"), (dict(first=[eight], second=[other]), "scales"),
        (dict(exp_avg_scales=[scale], exp_avg_sq_scales=[scale + 0]), "scales"), (dict(first=[eight], second=[other], exp_avg_scales=[scale]), "scales"),
        (dict(first=[eight], second=[other], exp_avg_scales=[scale], exp_avg_sq_scales=[torch.ones(2, device="cuda")]), "256"),
        (dict(first=[eight], second=[eight], exp_avg_scales=[scale], exp_avg_sq_scales=[scale + 0]), "share memory"),
        (dict(params=[p.int()], grads=[g.int()]), "only float32"), (dict(params=[p.cpu()], grads=[g.cpu()], first=[m.cpu()], second=[v.cpu()],
                                                                         steps=[torch.tensor(0)]), "CUDA"),
        (dict(params=[p.double()], grads=[g.double()], first=[eight], second=[other], exp_avg_scales=[scale], exp_avg_sq_scales=[scale + 0]),
         "moments"),
    ]
    kept_ = [x.clone() for x in (p, g, m, v)]
    for wrong, message in refused:
        with pytest.raises(RuntimeError, match=message):
            call(**wrong)
    assert all(torch.equal(a, b) for a, b in zip(kept_, (p, g, m, v))) and int(t[0]) == 0
    assert rt.adamw_step([], [], [], [], []) is None


# ---------------------------------------------------------------------------------------------
# the optimiser
# ---------------------------------------------------------------------------------------------
def small_model(seed=0, dtype=F32):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(20, 300), torch.nn.ReLU(), torch.nn.Linear(300, 5)).cuda().to(dtype)


def gradients(model, seed):
    for i, p in enumerate(model.parameters()):
        p.grad = rand(*p.shape, dtype=p.dtype, seed=seed + i, scale=0.1)


@pytest.mark.parametrize("dtype", [F32, F64])
def test_optimiser_is_torchs(dtype):
    ours, theirs = small_model(dtype=dtype), small_model(dtype=dtype)
    a = optim.AdamW([dict(params=ours[0].parameters(), lr=1e-2), dict(params=ours[2].parameters(), weight_decay=0.0)], lr=1e-3)
    b = torch.optim.AdamW([dict(params=theirs[0].parameters(), lr=1e-2), dict(params=theirs[2].parameters(), weight_decay=0.0)], lr=1e-3)
    schedules = [torch.optim.lr_scheduler.StepLR(o, 3, 0.5) for o in (a, b)]
    for i in range(12):
        for model in (ours, theirs):
            gradients(model, 100 * i)
        if i in (4, 5):  # without a gradient a parameter and its count stay
            ours[2].bias.grad = theirs[2].bias.grad = None
        a.step(), b.step()
        [s.step() for s in schedules]
    for p, q in zip(ours.parameters(), theirs.parameters()):
        # 12 steps of at most 2 lr, each off by some 30 roundings
        within(p.detach(), q.detach(), 12 * 2e-2 * 30 * unit(dtype) + 24 * unit(dtype) * q.detach().abs().double(), "parameter")
    assert int(a.state[ours[2].bias]["step"]) == 10 and int(a.state[ours[0].bias]["step"]) == 12


def test_optimiser_clips_like_torch():
    ours, theirs = small_model(), small_model()
    a, b = optim.AdamW(ours.parameters(), max_norm=0.1), torch.optim.AdamW(theirs.parameters())
    for i in range(5):
        for model in (ours, theirs):
            gradients(model, 100 * i)
        norm = torch.nn.utils.clip_grad_norm_(theirs.parameters(), 0.1)
        a.step(), b.step()
        within(a.grad_norm, norm, 1e-5 * norm, "norm")
    for p, q in zip(ours.parameters(), theirs.parameters()):
        within(p.detach(), q.detach(), 5 * 2e-3 * 1e-4 + 1e-6 * q.detach().abs().double(), "parameter")


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_optimiser_state_is_saved_and_loaded(bits, dtype, tmp_path):
    model = small_model(dtype=dtype)
    opt = optim.AdamW(model.parameters(), state_bits=bits, least_8bit=1000, seed=4)
    for i in range(3):
        gradients(model, i)
        opt.step()
    kinds = [opt.state[p]["exp_avg"].dtype for p in model.parameters()]
    assert kinds == ([E4M3, F32, E4M3, F32] if bits == 8 else [F32] * 4)
    torch.save([model.state_dict(), opt.state_dict()], tmp_path / "saved")
    weights, state = torch.load(tmp_path / "saved")
    other = small_model(1, dtype)
    other.load_state_dict(weights)
    opt2 = optim.AdamW(other.parameters(), state_bits=bits, least_8bit=1000, seed=4)
    opt2.load_state_dict(state)
    for m, o in ((model, opt), (other, opt2)):
        gradients(m, 50)
        o.step()
    for p, q in zip(model.parameters(), other.parameters()):
        assert torch.equal(p, q) and int(opt2.state[q]["step"]) == 4
        assert opt2.state[q]["exp_avg"].dtype == opt.state[p]["exp_avg"].dtype


def test_optimiser_is_copied_whole():
    model = small_model()
    opt = optim.AdamW(model.parameters(), max_norm=0.5, state_bits=8, least_8bit=100, seed=7)
    gradients(model, 3)
    opt.step()
    other = copy.deepcopy((model, opt))
    for m, o in ((model, opt), other):
        gradients(m, 20)
        o.step()
    for p, q in zip(model.parameters(), other[0].parameters()):
        assert torch.equal(p, q)
    assert torch.equal(opt.grad_norm, other[1].grad_norm)
    for p in model.parameters():
        p.grad = None
    opt.step()
    assert opt.grad_norm is None


def test_optimiser_with_8_bits_follows_the_one_with_32():
    """The same gradients for 200 steps: random roundings of at most an eighth each, over a mean of 1 / (1 - beta) steps."""
    models = [small_model() for _ in range(2)]
    opts = [optim.AdamW(models[0].parameters(), lr=1e-3, state_bits=8, least_8bit=0), optim.AdamW(models[1].parameters(), lr=1e-3)]
    start = [p.detach().clone() for p in models[0].parameters()]
    for i in range(200):
        for model, opt in zip(models, opts):
            gradients(model, 10 * i)
            for p, s in zip(model.parameters(), start):
                p.grad += 0.05 * s.sign()
            opt.step()
    for p, q, s in zip(models[0].parameters(), models[1].parameters(), start):
        moved = (q - s).detach().norm()
        assert (p - q).detach().norm() < 0.2 * moved


def test_optimiser_refuses():
    p = torch.nn.Parameter(rand(4))
    for wrong, message in ((dict(lr=-1.0), "lr"), (dict(betas=(0.9, 1.0)), "betas"), (dict(eps=-1.0), "eps"), (dict(weight_decay=-1.0), "weight_decay"),
                           (dict(max_norm=-1.0), "max_norm"), (dict(state_bits=4), "state_bits")):
        with pytest.raises(ValueError, match=message):
            optim.AdamW([p], **wrong)
    table = torch.nn.Embedding(5, 3, sparse=True).cuda()
    table(torch.tensor([1], device="cuda")).sum().backward()
    with pytest.raises(RuntimeError, match="sparse"):
        optim.AdamW(table.parameters()).step()
    q = torch.nn.Parameter(rand(4))
    p.grad, q.grad = rand(4), rand(4)
    with pytest.raises(RuntimeError, match="share betas"):
        optim.AdamW([dict(params=[p]), dict(params=[q], betas=(0.5, 0.9))], max_norm=1.0).step()
    optim.AdamW([dict(params=[p]), dict(params=[q], betas=(0.5, 0.9))]).step()


# ---------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------
def propagated(monkeypatch):
    """Models without a graph: every vertex keeps its features."""
    from compressgnn_b200.layer import KPropagate
    monkeypatch.setattr(KPropagate, "forward", lambda self, x, *a, **k: x)


@pytest.mark.parametrize("norm, residual", [(None, False), (None, True), ("layer", True)])
def test_a_model_with_fused_layers(norm, residual, monkeypatch):
    propagated(monkeypatch)
    torch.manual_seed(1)
    fused = GCN(64, 7, hidden_features=64, num_layers=3, dropout=0.0, norm=norm, residual=residual, linear="fused").cuda()
    plain = GCN(64, 7, hidden_features=64, num_layers=3, dropout=0.0, norm=norm, residual=residual).cuda()
    plain.load_state_dict(fused.state_dict())
    plain = plain.double()
    x, target = rand(3000, 64, seed=3), torch.randint(0, 7, (3000,), device="cuda")
    got, want = fused(x, None), plain(x.double(), None)
    assert (got.double() - want).abs().max() < 1e-5
    a = torch.autograd.grad(fused.loss(x, None, target), fused.parameters())
    b = torch.autograd.grad(plain.loss(x.double(), None, target), plain.parameters())
    for p, q in zip(a, b):
        assert (p.double() - q).norm() <= 1e-4 * q.norm() + 1e-9
    assert torch.equal(fused.inference(x, None), fused.eval()(x, None))


def test_a_training_run(monkeypatch):
    """Layers, loss and optimiser as a user runs them, the whole step captured and replayed beside the same steps run eagerly."""
    propagated(monkeypatch)
    results = []
    for captured in (False, True):
        torch.manual_seed(1)
        model = GCN(48, 7, hidden_features=96, num_layers=3, dropout=0.0, residual=True, linear="fused").cuda()
        opt = optim.AdamW(model.parameters(), lr=3e-3, max_norm=1.0, state_bits=8, least_8bit=512)
        x, target = rand(5000, 48, seed=3), torch.randint(0, 7, (5000,), device="cuda", generator=torch.Generator("cuda").manual_seed(2))
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())

        def step():
            opt.zero_grad(set_to_none=True)
            loss = model.loss(x, None, target)
            loss.backward()
            opt.step()
            return loss.detach()
        with torch.cuda.stream(stream):
            step(), step()
        torch.cuda.current_stream().wait_stream(stream)
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                loss = step()
            for _ in range(3):
                graph.replay()
        else:
            with torch.cuda.stream(stream):
                for _ in range(3):
                    loss = step()
        torch.cuda.synchronize()
        results.append([loss.clone(), opt.grad_norm.clone(), *(p.detach().clone() for p in model.parameters())])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert rt.device_status() == 0
