"""Modules of a training step that stand between and behind the propagations: normalisation, dropout, loss.

The reference's model calls ``torch.nn.functional`` for its dropout and leaves the loss to the caller (ref:
``model/compressgnn/gcn.py:59``); these run on the package's own kernels (``runtime.layer_norm``, ``runtime.dropout``,
``runtime.cross_entropy``)."""
import torch

from .. import runtime as _native


def dropout_onto(residual, x, p, seed=None):
    """``residual + dropout(x)`` with whatever may be added to ``x``: in one pass where the two have the same shape, type and
    device, else broadcast and promoted by torch, as the sum is where nothing is dropped."""
    if residual.shape == x.shape and residual.dtype == x.dtype and residual.device == x.device:
        return _native.dropout(x, p, residual, seed)
    return residual + _native.dropout(x, p, None, seed)


class LayerNorm(torch.nn.Module):
    """Layer normalisation over the last dimension, with the ReLU and the dropout that follow it in the same pass."""

    def __init__(self, features, eps=1e-5, bias=True, activation=None, device=None, dtype=None):
        super().__init__()
        if activation not in (None, "relu"):
            raise ValueError("Supported activations: None, relu")
        self.eps, self.activation = eps, activation
        self.weight = torch.nn.Parameter(torch.ones(features, device=device, dtype=dtype))
        self.bias = torch.nn.Parameter(torch.zeros(features, device=device, dtype=dtype)) if bias else None

    def forward(self, x, dropout=0.0, seed=None):
        """``dropout``: its probability; the caller passes 0 outside of training."""
        return _native.layer_norm(x, self.weight, self.bias, self.eps, self.activation, dropout, seed)

    def extra_repr(self):
        return f"{self.weight.numel()}, eps={self.eps}, bias={self.bias is not None}, activation={self.activation}"


class Dropout(torch.nn.Module):
    """Dropout without a stored mask, added to a residual stream when one is given; the identity outside of training."""

    def __init__(self, p=0.5):
        super().__init__()
        if not 0.0 <= p < 1.0:
            raise ValueError("dropout probability must lie in [0, 1)")
        self.p = p

    def forward(self, x, residual=None, seed=None):
        if not (self.training and self.p):
            return x if residual is None else x + residual
        return _native.dropout(x, self.p, None, seed) if residual is None else dropout_onto(residual, x, self.p, seed)

    def extra_repr(self):
        return f"p={self.p}"


class CrossEntropy(torch.nn.Module):
    """Softmax cross entropy over the labelled nodes (``runtime.cross_entropy``)."""

    def __init__(self, ignore_index=-100, reduction="mean"):
        super().__init__()
        if reduction not in _native._REDUCTIONS:
            raise ValueError(f"Supported reductions: {', '.join(_native._REDUCTIONS)}")
        self.ignore_index, self.reduction = ignore_index, reduction

    def forward(self, logits, target):
        return _native.cross_entropy(logits, target, self.ignore_index, self.reduction)
