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
