"""What the dense layer and the optimiser step promise where ordinary data does not show it: numbers that have to come out to the
bit, calls that want a part of the gradients only, operands at the ends of their type's range.

Whole numbers small enough that every sum of them is exact need no tolerance; where one is used its derivation stands beside it."""
import ctypes

import pytest
import torch

from compressgnn_b200 import runtime as rt

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
TYPES = [F32, F64, BF16, F16]
CODES = {F32: 0, F64: 1, BF16: 2, F16: 3}


def rand(*shape, dtype=F32, seed=0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=gen, dtype=F64) * scale).to(dtype)


def whole(*shape, dtype=F32, seed=0, largest=2):
    """Whole numbers of -largest .. largest."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-largest, largest + 1, shape, device="cuda", generator=gen).to(dtype)


def address(t):
    return None if t is None else t.data_ptr()


def backward(x, weight, mask, grad, p=0.0, dx=None, dweight=None, dbias=None, inner=0):
    """The C entry, whose pointers may be null."""
    lib = rt.lib()
    rows, outer = grad.shape
    room = lib.cgnn_linear_backward_scratch_bytes(CODES[grad.dtype], rows, inner, outer)
    scratch = torch.empty(room, dtype=torch.uint8, device="cuda")
    rc = lib.cgnn_linear_backward(CODES[grad.dtype], rows, inner, outer, inner, address(x), address(weight), address(mask), address(grad),
                                  p, address(dx), address(dweight), address(dbias), address(scratch), room,
                                  ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0, lib.cgnn_last_error()


def random_mask(rows, outer, seed):
    """A mask as the forward pass writes it (rows of whole 64-bit words, nothing behind their ends), and its bits."""
    words = (outer + 63) // 64
    gen = torch.Generator(device="cuda").manual_seed(seed)
    bits = torch.randint(0, 2, (rows, words * 64), device="cuda", generator=gen, dtype=torch.uint8)
    bits[:, outer:] = 0
    weights = 2 ** torch.arange(8, device="cuda", dtype=torch.uint8)
    return (bits.view(rows, words * 8, 8) * weights).sum(2, dtype=torch.uint8).contiguous(), bits[:, :outer].bool()


# ---------------------------------------------------------------------------------------------
# a part of the gradients
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, inner, outer", [(1, 5, 3), (63, 8, 33), (40000, 64, 72), (40000, 1030, 47), (9001, 257, 129), (3, 8, 40000)])
@pytest.mark.parametrize("masked", [False, True])
def test_bias_gradient_alone_looks_at_the_incoming_one_only(dtype, rows, inner, outer, masked):
    """Neither the input nor the weight is there."""
    grad = whole(rows, outer, dtype=dtype, seed=1)
    mask, bits = random_mask(rows, outer, 2) if masked else (None, torch.ones_like(grad, dtype=torch.bool))
    dbias = torch.empty(outer, dtype=dtype, device="cuda")
    backward(None, None, mask, grad, 0.5 if masked else 0.0, dbias=dbias, inner=inner)
    want = torch.where(bits, grad, 0).double().sum(0) * (2 if masked else 1)
    assert torch.equal(dbias, want.to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, outer", [(1, 8), (7, 16), (64, 24), (65, 136), (5000, 264), (100000, 16), (30011, 1032)])
@pytest.mark.parametrize("masked", [False, True])
def test_bias_gradient_alone_of_rows_on_any_address(dtype, rows, outer, masked):
    """Rows of whole vectors, on their boundary and an element behind it."""
    mask, bits = random_mask(rows, outer, 2) if masked else (None, torch.ones(rows, outer, dtype=torch.bool, device="cuda"))
    for ahead in (0, 1):
        held = whole(rows * outer + ahead, dtype=dtype, seed=1)
        grad = held[ahead:].view(rows, outer)
        dbias = torch.empty(outer, dtype=dtype, device="cuda")
        backward(None, None, mask, grad, 0.5 if masked else 0.0, dbias=dbias, inner=3)
        want = torch.where(bits, grad, 0).double().sum(0) * (2 if masked else 1)
        assert torch.equal(dbias, want.to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [50, 40000])
def test_gradients_with_a_frozen_weight(dtype, rows):
    x, w, b = whole(rows, 64, dtype=dtype, seed=1), whole(72, 64, dtype=dtype, seed=2), whole(72, dtype=dtype, seed=3)
    grad = whole(rows, 72, dtype=dtype, seed=4)
    b.requires_grad_()
    alone, = torch.autograd.grad(rt.linear(x, w, b), b, grad)
    x.requires_grad_()
    dx, beside = torch.autograd.grad(rt.linear(x, w, b), (x, b), grad)
    assert torch.equal(alone, grad.double().sum(0).to(dtype)) and torch.equal(alone, beside)
    assert torch.equal(dx, (grad.double() @ w.double()).to(dtype))


@pytest.mark.parametrize("activation, p", [(None, 0.0), ("relu", 0.25)])
def test_what_no_gradient_needs_is_not_kept(activation, p):
    """The input is there for the weight's gradient and the weight for the input's, as torch's layer has it: otherwise they may be
    changed, or given back, in front of the backward pass."""
    def tensors_():
        return [rand(*shape, seed=i) for i, shape in enumerate([(300, 7, 64), (48, 64), (48,)])]
    grad = rand(300, 7, 48, seed=5)
    for which in ((0,), (1,), (2,), (0, 2), (1, 2)):
        leaves = [t.requires_grad_(i in which) for i, t in enumerate(tensors_())]
        every = [t.requires_grad_() for t in tensors_()]
        want = torch.autograd.grad(rt.linear(*every, activation, p, seed=4), every, grad)
        y = rt.linear(*leaves, activation, p, seed=4)
        with torch.no_grad():
            if 0 not in which:
                leaves[1].fill_(7.0)
            if 1 not in which:
                leaves[0].fill_(7.0)
        got = torch.autograd.grad(y, [leaves[i] for i in which], grad)
        assert all(torch.equal(g, want[i]) for g, i in zip(got, which))
    # what is needed is kept, and a change of it refused
    for changed, wanted in ((0, 1), (1, 0)):
        leaves = [t.requires_grad_(i == wanted) for i, t in enumerate(tensors_())]
        y = rt.linear(*leaves, activation, p, seed=4)
        with torch.no_grad():
            leaves[changed].add_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    # nor does a frozen layer hold its input's memory
    x, w, b = tensors_()
    b.requires_grad_()
    inner = torch.zeros(1 << 20, 64, device="cuda")
    y = rt.linear(inner, w, b, activation, p, seed=4)
    held = torch.cuda.memory_allocated()
    inner = None
    assert held - torch.cuda.memory_allocated() >= 256 << 20
    assert torch.autograd.grad(y, b, torch.ones_like(y))[0].shape == b.shape


# ---------------------------------------------------------------------------------------------
# infinities and NaN
# ---------------------------------------------------------------------------------------------
def terms(n, dtype=F32):
    """Half steps of an fp32 sum of n terms on the tensor cores, of the sum of their sizes: n roundings of a sum, and 2 n for the
    truncations of every sixteen and the parts left out of fp32's three."""
    return (3 * n + 32) * (2.0**-53 if dtype == F64 else 2.0**-24)


def compare(got, want, bound, what):
    """64-bit results with what fp32 makes of them: NaN and infinities in their places, the others within their bound."""
    narrowed = want.float()
    assert torch.equal(torch.isnan(got), torch.isnan(narrowed)), f"{what}: NaN"
    sure = torch.isinf(want)  # (a large finite sum may lie on either side of the type's end)
    assert torch.equal(got[sure], narrowed[sure]), f"{what}: infinities"
    ordinary = torch.isfinite(want) & (want.abs() < 2.0**126)
    excess = ((got.double() - want).abs() - bound)[ordinary]
    assert excess.numel() == 0 or excess.max() <= 0, f"{what}: over its bound by {excess.max():.3e}"


def finite(t):
    return torch.nan_to_num(t.double(), 0.0, 0.0, 0.0).abs()


BAD = [float("inf"), float("-inf"), float("nan"), torch.finfo(F32).max]


@pytest.mark.parametrize("which", ["grad", "x", "weight"])
@pytest.mark.parametrize("rows, inner, outer", [(20000, 256, 4096), (300000, 72, 136), (3001, 1030, 301)])
@pytest.mark.parametrize("relu", [False, True])
def test_gradients_with_numbers_that_are_not_finite(which, rows, inner, outer, relu):
    """They reach the elements that they have a part in and no others, whatever a multiprocessor's further tiles wait for meanwhile."""
    x, w, b = rand(rows, inner, seed=1), rand(outer, inner, seed=2, scale=inner**-0.5), rand(outer, seed=3)
    grad = rand(rows, outer, seed=4)
    activation = "relu" if relu else None

    def both():
        leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)]
        y = rt.linear(*leaves, activation)
        return [y.detach(), *torch.autograd.grad(y, leaves, grad)]
    clean = both()
    held = {"grad": grad, "x": x, "weight": w}[which]
    places = [(held.size(0) // 2 + 3 * i, held.size(1) - 1 - 37 * i) for i in range(len(BAD))]
    for place, bad in zip(places, BAD):
        held[place] = bad
    assert rt.device_status() == 0
    y, dx, dw, db = both()
    assert rt.device_status() == 0
    z = x.double() @ w.double().t() + b.double()
    sizes = finite(x) @ finite(w).t() + b.double().abs()
    got_z = rt.linear(x, w, b)
    compare(got_z, z, (terms(inner) + 2.0**-24) * sizes + 2.0**-149, "z")
    assert torch.equal(y, torch.where(got_z <= 0, 0.0, got_z) if relu else got_z) or \
        torch.equal(torch.isnan(y), torch.isnan(got_z)) and torch.equal(y[~torch.isnan(y)], torch.where(got_z <= 0, 0.0, got_z)[~torch.isnan(y)]
                                                                        if relu else got_z[~torch.isnan(y)])
    g = torch.where(got_z <= 0, 0.0, grad.double()) if relu else grad.double()
    del z, sizes
    compare(dx, g @ w.double(), terms(outer) * (finite(g) @ finite(w)) + 2.0**-149, "dx")
    compare(dw, g.t() @ x.double(), terms(rows) * (finite(g).t() @ finite(x)) + 2.0**-149, "dweight")
    compare(db, g.sum(0), terms(rows) * finite(g).sum(0) + 2.0**-149, "dbias")
    # what has no part in them is what it was, to the bit
    rows_of, columns_of = (torch.ones(held.size(d), dtype=torch.bool, device="cuda") for d in (0, 1))
    for r, c in places:
        rows_of[r] = columns_of[c] = False
    if which == "grad":
        assert torch.equal(dx[rows_of], clean[1][rows_of]) and torch.equal(dw[columns_of], clean[2][columns_of])
        assert torch.equal(db[columns_of], clean[3][columns_of]) and torch.equal(y, clean[0])
    elif which == "x":
        assert torch.equal(y[rows_of], clean[0][rows_of]) and torch.equal(dx[rows_of], clean[1][rows_of])


@pytest.mark.parametrize("columns", [128, 131])
@pytest.mark.parametrize("p, added", [(0.0, False), (0.25, True)])
def test_forward_with_numbers_that_are_not_finite_and_what_follows(columns, p, added):
    x, w, b = rand(40000, 96, seed=1), rand(columns, 96, seed=2, scale=0.1), rand(columns, seed=3)
    residual = rand(40000, columns, seed=5) if added else None
    x[5, 0], x[20000, 95], x[39999, 50], x[39998, 50] = BAD
    y = rt.linear(x, w, b, "relu", p, residual, seed=7)
    z = rt.linear(x, w, b)
    want = torch.where(z <= 0, 0.0, z)
    if p:
        kept = rt.dropout(torch.ones_like(z), p, seed=7) != 0
        want = torch.where(kept, want * (1 / (1 - p)), 0.0)
    if added:
        want = want + residual
    assert torch.equal(y.isnan(), want.isnan())
    assert torch.equal(y[~y.isnan()], want[~y.isnan()])
    # the mask, by the gradient of a constant: what the ReLU and the dropout let through
    one = torch.zeros(columns, device="cuda", requires_grad=True)
    g = rand(40000, columns, seed=6)
    db, = torch.autograd.grad(rt.linear(x, w, b + one, "relu", p, residual, seed=7), one, g)
    passed = ~(z <= 0) & (kept if p else True)
    exact = torch.where(passed, g, 0.0).double().sum(0) / (1 - p)
    assert ((db.double() - exact).abs() <= terms(40000) * g.double().abs().sum(0)).all()
    assert rt.device_status() == 0


def test_waits_go_on_while_elements_are_computed_again():
    """A row of 4096 sums over 20,000 nodes by lanes takes milliseconds, a wait of 2^14 polls some tenths of one: the tiles behind the
    row's wait for as long as it takes."""
    x, grad = rand(20000, 4096, seed=1), rand(20000, 4096, seed=2)
    w = torch.zeros(4096, 4096, device="cuda", requires_grad=True)
    before = rt.lib().cgnn_linear_wait_limit(1 << 14)
    try:
        clean, = torch.autograd.grad(rt.linear(x, w), w, grad)
        assert rt.device_status() == 0
        grad[777, 1000] = float("inf")
        got, = torch.autograd.grad(rt.linear(x, w), w, grad)
        assert rt.device_status() == 0
    finally:
        rt.lib().cgnn_linear_wait_limit(before)
    others = torch.arange(4096, device="cuda") != 1000
    assert torch.equal(got[others], clean[others])
    assert torch.equal(got[1000], torch.copysign(torch.full_like(got[1000], float("inf")), x[777]))


# ---------------------------------------------------------------------------------------------
# long contractions of 16-bit operands
# ---------------------------------------------------------------------------------------------
def positive(*shape, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.rand(*shape, device="cuda", generator=gen).mul_(0.2).add_(0.1).to(dtype)


def within_one_rounding(got, want, what):
    """One rounding of the result.  In front of it an accumulator takes up to 8192 terms in 512 additions, each off by at most two steps
    of 2^-23 of a sum that is half of the last on average (together 2^-14), and no more than 64 such sums are added."""
    relative = ((got.double() - want) / want).abs().max()
    assert relative <= torch.finfo(got.dtype).eps / 2 + 2.0**-14 + 64 * 2.0**-24, f"{what}: {relative:.3e}"


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows, inner, outer", [(300000, 2048, 1280), (300001, 2045, 1277), (700000, 64, 128), (9000, 2048, 1280)])
def test_weight_gradients_of_one_sign_over_many_rows(dtype, rows, inner, outer):
    """In one split and in many: sums that only grow keep their last digits."""
    x, grad = positive(rows, inner, dtype=dtype, seed=1), positive(rows, outer, dtype=dtype, seed=2)
    w = torch.zeros(outer, inner, dtype=dtype, device="cuda", requires_grad=True)
    b = torch.zeros(outer, dtype=dtype, device="cuda", requires_grad=True)
    dw, db = torch.autograd.grad(rt.linear(x, w, b), (w, b), grad)
    some = torch.arange(0, inner, max(1, inner // 61), device="cuda")
    within_one_rounding(dw[:, some], grad.double().t() @ x[:, some].double(), "dweight")
    if dtype == BF16 or rows < 300000:  # (fp16 ends at 65504)
        within_one_rounding(db, grad.double().sum(0), "dbias")
    assert rt.device_status() == 0


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows, terms_, columns", [(256, 400000, 128), (300, 100001, 131), (20000, 8200, 40)])
def test_products_of_one_sign_and_many_terms(dtype, rows, terms_, columns):
    x, w = positive(rows, terms_, dtype=dtype, seed=1), positive(columns, terms_, dtype=dtype, seed=2)
    b, residual = positive(columns, dtype=dtype, seed=3), positive(rows, columns, dtype=dtype, seed=4)
    want = x.double() @ w.double().t()
    within_one_rounding(rt.linear(x, w), want, "forward")
    within_one_rounding(rt.linear(x, w, b, "relu", residual=residual), want + b.double() + residual.double(), "with what follows")
    # the same contraction in the gradient of an input
    leaf = torch.zeros(rows, columns, dtype=dtype, device="cuda", requires_grad=True)
    dx, = torch.autograd.grad(rt.linear(leaf, w.t().contiguous()), leaf, x)
    within_one_rounding(dx, want, "dx")
    assert rt.device_status() == 0


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows, inner, outer", [(20011, 1200, 2056), (20011, 1203, 2055), (140, 20011, 136), (140, 20008, 131), (131, 136, 20011)])
@pytest.mark.parametrize("relu, p", [(False, 0.0), (True, 0.5)])
def test_whole_numbers_over_several_segments(dtype, rows, inner, outer, relu, p):
    """Sums of few terms, among them those at the ends of segments and of the contraction: exact."""
    x, w = torch.zeros(rows, inner, dtype=dtype, device="cuda"), torch.zeros(outer, inner, dtype=dtype, device="cuda")
    grad = torch.zeros(rows, outer, dtype=dtype, device="cuda")
    for t, d in ((x, 0), (x, 1), (w, 0), (w, 1), (grad, 0), (grad, 1)):
        for i, at in enumerate((0, 63, 64, 4095, 8191, 8192, 8193, 16383, 16384, t.size(d) - 1)):
            if at < t.size(d):
                part = whole(t.size(1 - d), dtype=dtype, seed=7 * i + d, largest=3)
                t[at].copy_(part) if d == 0 else t[:, at].copy_(part)
    b = whole(outer, dtype=dtype, seed=5)
    for t in (x, w, b):
        t.requires_grad_()
    y = rt.linear(x, w, b, "relu" if relu else None, p, seed=11)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), grad)
    with torch.no_grad():
        z = x.double() @ w.double().t() + b.double()
        factor = torch.where(z > 0, 1.0, 0.0) if relu else torch.ones_like(z)
        if p:
            factor = factor * (rt.dropout(torch.ones_like(y), p, seed=11) != 0) * 2
        g = grad.double() * factor
        for got, want in ((y, z * factor), (dx, g @ w.double()), (dw, g.t() @ x.double()), (db, g.sum(0))):
            assert torch.equal(got, want.to(dtype))


# ---------------------------------------------------------------------------------------------
# every term, once
# ---------------------------------------------------------------------------------------------
LONG = [(325557, 256, 128), (70001, 301, 173), (300000, 72, 136), (150000, 8, 520), (40017, 1030, 47), (2708, 128, 64), (9001, 257, 129)]


def products_of(x, w, b, grad, activation=None, p=0.0):
    """An output, its gradients, and what all of them are in 64 bits."""
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)]
    y = rt.linear(*leaves, activation, p, seed=6)
    got = [y.detach(), *torch.autograd.grad(y, leaves, grad)]
    assert rt.device_status() == 0
    x, w, b, g = (t.double() for t in (x, w, b, grad))
    z = x @ w.t() + b
    passed = torch.where(z > 0, 1.0, 0.0) if activation else torch.ones_like(z)
    if p:
        passed = passed * (rt.dropout(torch.ones_like(grad), p, seed=6) != 0) / (1 - p)
    g = g * passed
    return got, [z * passed, g @ w, g.t() @ x, g.sum(0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, inner, outer", LONG)
@pytest.mark.parametrize("activation, p", [(None, 0.0), ("relu", 0.5)])
def test_whole_numbers_come_out_to_the_bit(dtype, rows, inner, outer, activation, p):
    """Sums of whole numbers up to 4, at most 2 * 4 * 325,557 of them: exact in fp32 whatever their order, and rounded once.  A term
    that is lost, or counted twice, at the end of a split or anywhere else, shows."""
    x, w, b = whole(rows, inner, dtype=dtype, seed=1), whole(outer, inner, dtype=dtype, seed=2), whole(outer, dtype=dtype, seed=3)
    got, want = products_of(x, w, b, whole(rows, outer, dtype=dtype, seed=4), activation, p)
    for a, e, name in zip(got, want, ("y", "dx", "dweight", "dbias")):
        assert e.abs().max() < 2**24
        assert torch.equal(a, e.to(dtype)), name


@pytest.mark.parametrize("rows, inner, outer", LONG)
def test_a_single_term_has_all_of_fp32s_digits(rows, inner, outer):
    """One product an element, of numbers with digits in all three bf16 parts.  Left out are three products of parts, together
    below 2^-23 of it (parts of 2^-9 and 2^-17 at most: 2 * 2^-26 + 2^-34); the accumulators and their sum truncate or round five times
    by 2^-23 at most; the result as written."""
    few = 2.0**-23 * 6 + 2.0**-24
    gen = torch.Generator(device="cuda").manual_seed(1)

    def odd(*shape):
        """1 to 2 in size, the last digit set."""
        digits = torch.randint(0, 1 << 22, shape, device="cuda", generator=gen) * 2 + 1
        sign = torch.randint(0, 2, shape, device="cuda", generator=gen) * 2 - 1
        return (sign * (1 + digits.double() * 2.0**-23)).float()
    w, grad = odd(outer, inner), odd(rows, outer)
    at = torch.randint(0, inner, (rows,), device="cuda", generator=gen)
    of = torch.randint(0, outer, (rows,), device="cuda", generator=gen)
    values = odd(rows)
    x = torch.zeros(rows, inner, device="cuda").scatter_(1, at[:, None], values[:, None])
    want = values.double()[:, None] * w.double().t()[at]
    y = rt.linear(x, w)
    assert ((y.double() - want).abs() <= few * want.abs()).all()
    thin = torch.zeros(rows, outer, device="cuda").scatter_(1, of[:, None], values[:, None])
    leaf = torch.zeros(rows, inner, device="cuda", requires_grad=True)
    dx, = torch.autograd.grad(rt.linear(leaf, w), leaf, thin)
    want = values.double()[:, None] * w.double()[of]
    assert ((dx.double() - want).abs() <= few * want.abs()).all()
    for row in (0, rows // 2, rows - 1):
        x = torch.zeros(rows, inner, device="cuda")
        x[row] = odd(inner)
        v = torch.zeros(outer, inner, device="cuda", requires_grad=True)
        dw, = torch.autograd.grad(rt.linear(x, v), v, grad)
        want = grad[row].double()[:, None] * x[row].double()
        assert ((dw.double() - want).abs() <= few * want.abs()).all()
    assert rt.device_status() == 0


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows, inner, outer", LONG + [(100000, 1024, 256)])
@pytest.mark.parametrize("activation, p", [(None, 0.0), ("relu", 0.3)])
def test_errors_do_not_grow_with_the_number_of_rows(dtype, rows, inner, outer, activation, p):
    """Over all elements (root mean squares): an accumulator takes 16 terms an addition and truncates it, half a step of 2^-23 of the sum
    so far on average; of fp32 it takes 256 terms, whose 16 additions lose at most 8 steps of 2^-23 of a sum that is 0.7 of the last on
    average: 6.7e-7, by one sign within the 256 and by any from one 256 to the next.  Of 16 bits it takes 8192, 512 additions, 2.1e-5; the
    rounding of the result is half a step at most."""
    x, w, b = rand(rows, inner, dtype=dtype, seed=1), rand(outer, inner, dtype=dtype, seed=2), rand(outer, dtype=dtype, seed=3)
    got, want = products_of(x, w, b, rand(rows, outer, dtype=dtype, seed=4), activation, p)
    if activation:  # (a sum next to zero may lie on its other side in fp32: its gradient's terms are those that the kernel took)
        passed = (got[0] != 0).double() / (1 - p)
        g = rand(rows, outer, dtype=dtype, seed=4).double() * passed
        want[1:] = [g @ w.double(), g.t() @ x.double(), g.sum(0)]
    bound = 6.7e-7 if dtype == F32 else torch.finfo(dtype).eps / 2 + 2.1e-5
    for a, e, name in zip(got, want, ("y", "dx", "dweight", "dbias")):
        off = float(((a.double() - e).square().mean() / e.square().mean()).sqrt())
        assert off <= bound, f"{name}: {off:.3e} of {bound:.3e}"


# ---------------------------------------------------------------------------------------------
# the bias' gradient
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, inner, outer", [(325557, 256, 128), (2708, 128, 64), (40000, 64, 72), (200000, 16, 7), (9001, 257, 129),
                                                (700, 2048, 1), (20000, 1024, 2048)])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_bias_gradient_is_summed_in_64_bits(dtype, rows, inner, outer, p):
    """fp32: one rounding, of the result.  16 bits: eight rows may be added in fp32 before, seven roundings of them."""
    x, w = rand(rows, inner, dtype=dtype, seed=1), rand(outer, inner, dtype=dtype, seed=2).requires_grad_()
    b = rand(outer, dtype=dtype, seed=3).requires_grad_()
    grad = rand(rows, outer, dtype=dtype, seed=4)
    dw, beside = torch.autograd.grad(rt.linear(x, w, b, None, p, seed=5), (w, b), grad)
    alone, = torch.autograd.grad(rt.linear(x, w.detach(), b, None, p, seed=5), b, grad)
    kept = rt.dropout(torch.ones_like(grad), p, seed=5) != 0 if p else torch.ones_like(grad, dtype=torch.bool)
    terms_of = torch.where(kept, grad, 0).double() / (1 - p)
    want, size = terms_of.sum(0), terms_of.abs().sum(0)
    # (64-bit sums of 10^5 terms and a factor, here and there: 2^-36 of the sizes at most; a product with the factor in 64 bits)
    bound = torch.finfo(dtype).eps / 2 * want.abs() + 2.0**-36 * size + (7 * 2.0**-24 * size if dtype in (BF16, F16) else 0.0)
    for got, what in ((beside, "beside the weight's"), (alone, "alone")):
        assert ((got.double() - want).abs() <= bound).all(), (what, float(((got.double() - want).abs() - bound).max()))


# ---------------------------------------------------------------------------------------------
# fp32 operands near the end of their range
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows, inner, outer", [(40000, 64, 72), (3000, 1030, 301), (200, 16, 7)])
@pytest.mark.parametrize("exponent", [-100, -109, -112, -118, -124, -130])
def test_small_fp32_operands(rows, inner, outer, exponent):
    """Operands are off by 2^-134 at most, half of bf16's least number, beyond what they are off elsewhere; sums by half a step of 2^-149
    an addition.  By single elements nothing is lost beyond that half step."""
    tiles = rows * inner * outer >= 4e7
    x, w, grad = rand(rows, inner, seed=1, scale=2.0**exponent), rand(outer, inner, seed=2), rand(rows, outer, seed=3)

    def check(got, a, b, n, what):
        a, b = a.double(), b.double()
        bound = terms(n) * (a.abs() @ b.abs()) + (3 * n + 32) * 2.0**-149
        if tiles:
            bound += 2.0**-134 * b.abs().sum(0)
        excess = ((got.double() - a @ b).abs() - bound).max()
        assert excess <= 0, f"{what}: {excess:.3e}"
    check(rt.linear(x, w), x, w.t(), inner, "y")
    v = torch.zeros(outer, inner, device="cuda", requires_grad=True)
    dw, = torch.autograd.grad(rt.linear(x, v), v, grad)
    check(dw.t(), x.t(), grad, rows, "dweight")
    small, leaf = grad * 2.0**exponent, torch.zeros(rows, inner, device="cuda", requires_grad=True)
    dx, = torch.autograd.grad(rt.linear(leaf, w), leaf, small)
    check(dx, small, w, outer, "dx")
    assert rt.device_status() == 0


# ---------------------------------------------------------------------------------------------
# an optimiser step
# ---------------------------------------------------------------------------------------------
def test_a_step_reads_nothing_that_it_writes():
    """Warps take what they read and write in any order: a gradient that lies over a moment, or the rate in a parameter, is refused."""
    n = 5000
    held = rand(3 * n, seed=1)
    p, m, v, g = rand(n, seed=2), torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), rand(n, seed=3)

    def step(p=p, g=g, m=m, v=v, **more):
        t = torch.zeros((), dtype=torch.int64, device="cuda")
        return rt.adamw_step([p, rand(5)], [g, rand(5)], [m, torch.zeros(5, device="cuda")], [v, torch.zeros(5, device="cuda")],
                             [t, torch.zeros((), dtype=torch.int64, device="cuda")], **more)
    parts = held[:n], held[n - 1:2 * n - 1], held[2 * n:]
    before = held.clone()
    for wrong in (dict(g=parts[0], m=parts[1]), dict(g=parts[1], v=parts[0]), dict(g=parts[0], p=parts[1]), dict(g=held[:n], p=held[:n]),
                  dict(p=parts[0], lr=held[:1]), dict(v=parts[0], lr=held[n - 1])):
        with pytest.raises(RuntimeError, match="share memory"):
            step(**wrong)
    assert torch.equal(held, before)
    # beside each other, and read twice
    step(p=held[:n], g=held[n:2 * n], m=held[2 * n:])
    rate = torch.tensor(1e-3, device="cuda")
    two = [rand(n, seed=5), rand(n, seed=5)]
    rt.adamw_step(two, [g, g], [torch.zeros(n, device="cuda") for _ in two], [torch.zeros(n, device="cuda") for _ in two],
                  list(torch.zeros(2, dtype=torch.int64, device="cuda")), lr=[rate, rate])
    assert torch.equal(*two)
