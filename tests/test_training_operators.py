"""What the row operators of a training step (normalisation, dropout, loss) refuse, without a GPU."""
import pickle

import pytest
import torch

from compressgnn_b200 import _lib, runtime as rt
from compressgnn_b200.layer import CrossEntropy, Dropout, LayerNorm
from compressgnn_b200.model import GCN, GNNLayer


def test_host_tensors_are_refused():
    x = torch.randn(4, 8)
    for call in (lambda: rt.layer_norm(x), lambda: rt.dropout(x, 0.5), lambda: rt.cross_entropy(x, torch.zeros(4, dtype=torch.int64)),
                 lambda: LayerNorm(8)(x), lambda: CrossEntropy()(x, torch.zeros(4, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(RuntimeError, match="CUDA"):
        Dropout(0.5)(x)
    assert Dropout(0.5).eval()(x) is x  # the identity outside of training touches nothing


def test_names_are_checked():
    x = torch.randn(4, 8)
    with pytest.raises(RuntimeError, match="activations"):
        rt.layer_norm(x, activation="gelu")
    with pytest.raises(RuntimeError, match="reductions"):
        rt.cross_entropy(x, torch.zeros(4, dtype=torch.int64), reduction="max")
    with pytest.raises(ValueError, match="activations"):
        LayerNorm(8, activation="gelu")
    with pytest.raises(ValueError, match="reductions"):
        CrossEntropy(reduction="max")
    for p in (1.0, -0.1):
        with pytest.raises(ValueError, match="probability"):
            Dropout(p)
    with pytest.raises(ValueError, match="norm"):
        GNNLayer(4, 4, norm="batch")


def test_a_model_without_the_new_parts_is_what_it_was():
    torch.manual_seed(0)
    model = GCN(8, 3, hidden_features=8, num_layers=3)
    assert model.residual is False and all(layer.norm is None for layer in model.layers)
    assert not any("norm" in name for name in model.state_dict())
    older = pickle.dumps(model)
    for layer in model.layers:
        del layer.norm
    del model.residual
    old = pickle.loads(pickle.dumps(model))  # as saved whole before there was a choice
    assert old.residual is False and all(layer.norm is None for layer in old.layers)
    assert all(layer.norm is None for layer in pickle.loads(older).layers)
    normalised = GCN(8, 3, hidden_features=8, num_layers=3, norm="layer")
    assert [layer.norm is None for layer in normalised.layers] == [False, False, True]
    assert normalised.layers[0].norm.activation == "relu"


def test_column_sharding_refuses_whole_row_models():
    from compressgnn_b200 import dist
    layer = GNNLayer(8, 8, use_transformation=True, norm="layer")
    with pytest.raises(ValueError, match="whole rows"):
        dist.ShardedGNNLayer(layer)
    with pytest.raises(ValueError, match="residual"):
        dist.ShardedGCN(GCN(8, 3, use_transformation=True, residual=True))


def test_placement_looks_into_a_model_only_where_it_would_shard_it():
    from compressgnn_b200 import dist
    anything = torch.nn.Linear(4, 4)
    assert dist.place_model(anything, 4096) == (anything, False)
    assert dist.needs_whole_rows(GCN(8, 3, norm="layer")) and dist.needs_whole_rows(GCN(8, 3, residual=True))
    assert not dist.needs_whole_rows(GCN(8, 3))


HUGE = 2**30


def _norm(dtype=0, params=0, rows=4, width=8, stride=8, x=64, weight=64, p=0.0, out=64, mean=64, rstd=64):
    return _lib.lib().cgnn_layer_norm(dtype, params, rows, width, stride, x, weight, None, 1e-5, 0, p, 0, None, out, mean, rstd,
                                      None)


def _norm_backward(dtype=0, params=0, rows=4, width=8, x=64, mean=64, grad=64, dweight=64, scratch=64, room=1 << 20):
    return _lib.lib().cgnn_layer_norm_backward(dtype, params, rows, width, width, x, 64, None, mean, 64, grad, 0, 0.0, 0, None, 64,
                                               dweight, None, scratch, room, None)


def _dropout(dtype=0, n=4, x=64, p=0.5, out=64):
    return _lib.lib().cgnn_dropout(dtype, n, x, None, p, 0, None, out, None)


def _loss(dtype=0, rows=4, classes=8, stride=8, logits=64, target=64, reduction=2, loss=64, grad=None, labelled=64, scratch=64,
          room=1 << 20, stats=None):
    return _lib.lib().cgnn_cross_entropy(dtype, rows, classes, stride, logits, target, -100, reduction, loss, stats, grad, labelled,
                                         scratch, room, None)


def _loss_backward(dtype=0, rows=4, classes=8, logits=64, reduction=2, stats=64, labelled=64, upstream=64, grad=64):
    return _lib.lib().cgnn_cross_entropy_backward(dtype, rows, classes, classes, logits, 64, -100, reduction, stats, labelled,
                                                  upstream, 0, grad, None)


REFUSED = [
    (_norm, dict(dtype=4), b"unknown dtype"), (_norm, dict(dtype=-1), b"unknown dtype"),
    (_norm, dict(params=2), b"matrix' type"), (_norm, dict(dtype=1, params=0), b"matrix' type"),
    (_norm, dict(dtype=2, params=3), b"matrix' type"), (_norm, dict(rows=-1), b"negative"), (_norm, dict(width=-1), b"negative"),
    (_norm, dict(stride=-8), b"negative"), (_norm, dict(width=HUGE), b"not supported"), (_norm, dict(p=1.0), b"probability"),
    (_norm, dict(p=-0.5), b"probability"), (_norm, dict(p=float("nan")), b"probability"), (_norm, dict(x=None), b"null pointer"),
    (_norm, dict(out=None), b"null pointer"), (_norm, dict(mean=None), b"statistics"),
    (_norm_backward, dict(dtype=4), b"unknown dtype"), (_norm_backward, dict(mean=None), b"null pointer"),
    (_norm_backward, dict(grad=None), b"null pointer"), (_norm_backward, dict(scratch=None), b"null scratch"),
    (_norm_backward, dict(room=16), b"too small"), (_norm_backward, dict(scratch=72), b"16-byte"),
    (_dropout, dict(dtype=4), b"unknown dtype"), (_dropout, dict(n=-1), b"negative"), (_dropout, dict(p=1.0), b"probability"),
    (_dropout, dict(p=float("nan")), b"probability"), (_dropout, dict(x=None), b"null pointer"),
    (_loss, dict(dtype=4), b"unknown dtype"), (_loss, dict(reduction=3), b"unknown reduction"), (_loss, dict(rows=-1), b"negative"),
    (_loss, dict(classes=0), b"not supported"), (_loss, dict(classes=HUGE), b"not supported"),
    (_loss, dict(logits=None), b"null pointer"), (_loss, dict(target=None), b"null pointer"), (_loss, dict(loss=None), b"null loss"),
    (_loss, dict(labelled=None), b"count"), (_loss, dict(scratch=None), b"scratch"), (_loss, dict(room=8), b"too small"),
    (_loss, dict(scratch=68), b"8-byte"), (_loss, dict(stats=68), b"boundaries"), (_loss, dict(dtype=1, stats=72), b"boundaries"),
    (_loss_backward, dict(stats=68), b"boundaries"), (_loss, dict(reduction=0, grad=64), b"unreduced"),
    (_loss_backward, dict(dtype=4), b"unknown dtype"), (_loss_backward, dict(stats=None), b"null pointer"),
    (_loss_backward, dict(labelled=None), b"null pointer"), (_loss_backward, dict(upstream=None), b"null pointer"),
]


@pytest.mark.parametrize("which", range(len(REFUSED)))
def test_argument_errors_of_the_c_entries(which):
    """All found on the host: nothing is launched, so no GPU is needed and no address is looked at."""
    call, wrong, message = REFUSED[which]
    assert call(**wrong) == 1
    assert message in _lib.lib().cgnn_last_error(), _lib.lib().cgnn_last_error()


def test_gradients_of_parameters_have_a_type_of_their_own_only_beside_16_bits():
    """Without a weight and a bias too: the sums would be written in the matrix' type behind arrays of a narrower one."""
    def call(dtype, params, rows=4, dweight=64, dbias=None):
        return _lib.lib().cgnn_layer_norm_backward(dtype, params, rows, 8, 8, 64, None, None, 64, 64, 64, 0, 0.0, 0, None, 64, dweight,
                                                   dbias, 64, 1 << 20, None)
    for dtype, params in ((1, 0), (0, 2), (1, 3), (2, 3), (2, 1), (0, 7)):
        for rows in (4, 0):
            for wanted in (dict(), dict(dweight=None, dbias=64)):
                assert call(dtype, params, rows, **wanted) == 1, (dtype, params, rows)
                assert b"matrix' type" in _lib.lib().cgnn_last_error()
    # (where nothing has the type it is not looked at)
    assert call(1, 0, rows=0, dweight=None) == 0


def test_empty_calls_do_nothing():
    assert _norm(rows=0, x=None, out=None) == 0 and _norm(width=0, x=None, out=None) == 0
    assert _dropout(n=0, x=None, out=None) == 0
    assert _loss(rows=0, reduction=0, logits=None, target=None, loss=None) == 0
    assert _loss_backward(rows=0, logits=None) == 0


@pytest.mark.parametrize("dtype", range(4))
def test_scratch_sizes(dtype):
    room = _lib.lib().cgnn_layer_norm_scratch_bytes
    assert room(dtype, 0, 8) == 0 and room(dtype, 8, 0) == 0 and room(4, 8, 8) == 0
    for rows in (1, 3, 1000, 10**7):
        for width in (1, 7, 64, 301, 2048, 4096, 16384, 50001, 10**6):
            one = 2 * width * (8 if dtype == 1 else 4)
            assert one <= room(dtype, rows, width) <= one * 148 * 8


def test_seeds_as_the_binding_takes_them():
    assert rt._seed_args(None) == (None, None)
    assert rt._seed_args(5) == (5, None) and rt._seed_args(2**64 - 1) == (-1, None) and rt._seed_args(-1) == (-1, None)
    key = torch.zeros(1, dtype=torch.int64)
    assert rt._seed_args(key)[1] is key
