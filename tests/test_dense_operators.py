"""What the dense layer and the optimiser step refuse, without a GPU."""
import ctypes
import pickle

import pytest
import torch

from compressgnn_b200 import _lib, optim, runtime as rt
from compressgnn_b200.layer import Linear
from compressgnn_b200.model import GCN, GNNLayer


def test_host_tensors_and_names_are_refused():
    x, w = torch.randn(4, 8), torch.randn(3, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        rt.linear(x, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        Linear(8, 3)(x)
    with pytest.raises(RuntimeError, match="activations"):
        rt.linear(x, w, activation="gelu")
    with pytest.raises(ValueError, match="activations"):
        Linear(8, 3, activation="gelu")
    with pytest.raises(ValueError, match="linear"):
        GNNLayer(8, 3, linear="fast")
    p = torch.nn.Parameter(x)
    p.grad = torch.ones_like(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        optim.AdamW([p]).step()
    with pytest.raises(RuntimeError, match="CUDA"):
        rt.adamw_step([x], [x], [x], [x], [torch.tensor(0)])
    optim.AdamW([torch.nn.Parameter(w)]).step()  # no gradient, nothing to do


def test_a_model_says_how_its_layers_are_computed():
    model = GCN(8, 3, hidden_features=8, num_layers=3)
    assert not any(isinstance(layer.lin, Linear) for layer in model.layers)
    fused = GCN(8, 3, hidden_features=8, num_layers=3, linear="fused")
    assert [layer.lin.activation for layer in fused.layers] == ["relu", "relu", None]
    assert sorted(fused.state_dict()) == sorted(model.state_dict())
    model.load_state_dict(fused.state_dict())
    assert [layer.lin.activation for layer in pickle.loads(pickle.dumps(fused)).layers] == ["relu", "relu", None]
    assert all(layer.lin.activation is None for layer in GCN(8, 3, num_layers=3, norm="layer", linear="fused").layers)


def _linear(dtype=0, rows=4, inner=8, outer=3, stride=8, x=64, weight=64, p=0.0, y=64, mask=None, scratch=64, room=1 << 30):
    return _lib.lib().cgnn_linear(dtype, rows, inner, outer, stride, x, weight, None, None, 1, p, 0, None, y, mask, scratch, room, None)


def _backward(dtype=0, rows=4, inner=8, outer=3, stride=8, x=64, weight=64, mask=None, grad=64, p=0.0, dx=64, dweight=64, dbias=64,
              scratch=64, room=1 << 30):
    return _lib.lib().cgnn_linear_backward(dtype, rows, inner, outer, stride, x, weight, mask, grad, p, dx, dweight, dbias, scratch, room,
                                           None)


class Tensor(ctypes.Structure):
    _fields_ = [(name, ctypes.c_void_p) for name in ("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "step")] + \
        [("n", ctypes.c_int64), ("lr", ctypes.c_double), ("weight_decay", ctypes.c_double), ("device_lr", ctypes.c_void_p),
         ("dtype", ctypes.c_int32)]


def _adamw(count=1, beta1=0.9, beta2=0.999, eps=1e-8, max_norm=-1.0, scratch=64, room=1 << 20, none=False, **fields):
    values = dict(param=64, grad=64, exp_avg=64, exp_avg_sq=64, step=64, n=8, lr=0.1, weight_decay=0.0, dtype=0)
    t = Tensor(**dict(values, **fields))
    return _lib.lib().cgnn_adamw(None if none else ctypes.byref(t), count, beta1, beta2, eps, max_norm, 0, None, scratch, room, None)


HUGE = 2**28
REFUSED = [
    (_linear, dict(dtype=4), b"unknown dtype"), (_linear, dict(dtype=-1), b"unknown dtype"), (_linear, dict(rows=-1), b"negative"),
    (_linear, dict(inner=-1), b"negative"), (_linear, dict(outer=-1), b"negative"), (_linear, dict(stride=-1), b"negative"),
    (_linear, dict(inner=HUGE), b"not supported"), (_linear, dict(outer=HUGE), b"not supported"), (_linear, dict(p=1.0), b"probability"),
    (_linear, dict(p=float("nan")), b"probability"), (_linear, dict(x=None), b"null pointer"), (_linear, dict(weight=None), b"null pointer"),
    (_linear, dict(y=None), b"null pointer"), (_linear, dict(mask=68), b"8-byte"),
    (_backward, dict(dtype=9), b"unknown dtype"), (_backward, dict(rows=-1), b"negative"), (_backward, dict(outer=HUGE), b"not supported"),
    (_backward, dict(grad=None), b"null pointer"), (_backward, dict(weight=None), b"needs the weight"), (_backward, dict(x=None), b"needs the input"),
    (_backward, dict(mask=4), b"8-byte"), (_backward, dict(rows=10**6, room=4), b"scratch"), (_backward, dict(rows=10**6, scratch=None), b"scratch"),
    (_backward, dict(rows=10**6, scratch=72), b"16-byte"), (_backward, dict(p=-0.1), b"probability"),
    (_adamw, dict(count=-1), b"number of tensors"), (_adamw, dict(beta1=1.0), b"betas"), (_adamw, dict(beta2=-0.1), b"betas"),
    (_adamw, dict(eps=-1.0), b"eps"), (_adamw, dict(max_norm=float("nan")), b"max_norm"), (_adamw, dict(none=True), b"null pointer"),
    (_adamw, dict(dtype=4), b"unknown dtype"), (_adamw, dict(n=-1), b"number of elements"), (_adamw, dict(step=None), b"step count"),
    (_adamw, dict(step=68), b"step count"), (_adamw, dict(param=None), b"null pointer"), (_adamw, dict(grad=None), b"null pointer"),
    (_adamw, dict(exp_avg_sq=None), b"null pointer"), (_adamw, dict(exp_avg_scale=64), b"both moments"), (_adamw, dict(lr=-1.0), b"lr"),
    (_adamw, dict(weight_decay=-1.0), b"lr"), (_adamw, dict(dtype=1, exp_avg_scale=64, exp_avg_sq_scale=64), b"fp64"),
    (_adamw, dict(max_norm=1.0, scratch=None), b"scratch"), (_adamw, dict(max_norm=1.0, room=4), b"scratch"),
    (_adamw, dict(max_norm=1.0, scratch=68), b"8-byte"),
]


@pytest.mark.parametrize("which", range(len(REFUSED)))
def test_argument_errors_of_the_c_entries(which):
    """All found on the host: nothing is launched, so no GPU is needed and no address is looked at."""
    call, wrong, message = REFUSED[which]
    assert call(**wrong) == 1
    assert message in _lib.lib().cgnn_last_error(), _lib.lib().cgnn_last_error()


def test_empty_calls_do_nothing():
    assert _linear(rows=0, x=None, y=None) == 0 and _linear(outer=0, y=None) == 0
    assert _backward(rows=0, dx=None, dweight=None, dbias=None, grad=None) == 0
    assert _adamw(count=0, none=True) == 0


@pytest.mark.parametrize("dtype", range(4))
def test_scratch_sizes(dtype):
    lib = _lib.lib()
    assert lib.cgnn_linear_mask_bytes(0, 5) == 0 and lib.cgnn_linear_mask_bytes(3, 65) == 48
    for rows in (0, 1, 1000, 10**6):
        for inner in (0, 1, 64, 301, 4096):
            for outer in (0, 1, 47, 256, 4096):
                assert 0 <= lib.cgnn_linear_scratch_bytes(dtype, rows, inner, outer) < 1 << 31
                assert 0 <= lib.cgnn_linear_backward_scratch_bytes(dtype, rows, inner, outer) < 1 << 31
    t = Tensor(n=10**9)
    assert 8 <= lib.cgnn_adamw_scratch_bytes(ctypes.byref(t), 1) <= 1 << 16
    assert lib.cgnn_adamw_scratch_bytes(None, 3) == 0
