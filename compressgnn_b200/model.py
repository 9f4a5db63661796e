"""The caller of the hot path: ``GNNLayer`` (propagate, then either a Linear on all nodes or
cluster -> Linear on representatives -> fused reconstruct) and a GCN stack of them
(ref: ``model/compressgnn/gcn.py:12-71``; the reference hard-wires three layers, here the
depth is a parameter so the two-layer benchmark configurations can be built, and the ReLU
after a hidden layer is handed to the layer so that it runs inside the reconstruct kernel)."""
from typing import Optional

import torch
import torch.nn.functional as F
from torch import Tensor

from . import runtime as _native
from .layer import Compressgnn_Cluster, Compressgnn_Reconstruct, KPropagate, LayerNorm, Linear
from .layer.training import dropout_onto


class GNNLayer(torch.nn.Module):
    def __init__(self, in_features, out_features, param_H=1, use_transformation=False, refresh_interval=1,
                 process_group=None, activation=None, norm=None, linear=None):
        super().__init__()
        if linear not in (None, "fused"):
            raise ValueError("linear must be None or 'fused'")
        if norm not in (None, "layer"):
            raise ValueError("norm must be None or 'layer'")
        if activation not in (None, "relu"):
            raise ValueError("activation must be None or 'relu'")
        self.activation = activation  # applied to the layer's output (fused into the reconstruction)
        if linear:  # one product with what follows it, on the package's kernel
            self.lin = Linear(in_features, out_features, activation=None if norm else activation)
        else:
            self.lin = torch.nn.Linear(in_features=in_features, out_features=out_features, bias=True)
        self.P = KPropagate()
        self.use_transformation = use_transformation
        self.cluster = Compressgnn_Cluster(in_feature=in_features, param_H=param_H, training=True, cache=True,
                                           index_cache=False, refresh_interval=refresh_interval,
                                           process_group=process_group)
        self.reconstruct = Compressgnn_Reconstruct()
        # between the transformation and its activation; one pass with the activation and the dropout
        self.norm = LayerNorm(out_features, activation=activation) if norm else None

    def __setstate__(self, state):
        super().__setstate__(state)
        if not hasattr(self, "norm"):  # a layer that was saved whole before there was one
            self.norm = None

    def set_epoch(self, epoch, loss=None):
        self.cluster.set_epoch(epoch, loss=loss)

    def reset_cache(self):
        self.cluster.reset_cache()

    def forward(self, x: Tensor, edge_index, edge_weight=None, vertex_cnt: int = 0, rule_cnt: int = 0,
                dropout: float = 0.0, residual: Optional[Tensor] = None) -> Tensor:
        """``dropout``: probability of the dropout the model applies to this layer's (ReLU) output; with the
        transformation path it runs inside the reconstruct kernel, behind a normalisation inside its kernel.
        ``residual``: added to the layer's output, in the pass of the dropout when there is one."""
        fused = isinstance(self.lin, Linear) and not self.use_transformation and self.norm is None
        if fused:
            x = self.P(x=x, edge_index=edge_index, edge_weight=edge_weight, vertex_cnt=vertex_cnt, rule_cnt=rule_cnt)
            return self.lin(x, dropout, residual)
        if residual is not None:
            out = GNNLayer.forward(self, x, edge_index, edge_weight, vertex_cnt, rule_cnt)
            return dropout_onto(residual, out, dropout) if dropout else out + residual
        x = self.P(x=x, edge_index=edge_index, edge_weight=edge_weight, vertex_cnt=vertex_cnt, rule_cnt=rule_cnt)
        if self.norm is not None:
            return self.norm(self._transform(x, None, 0.0), dropout)
        return self._transform(x, self.activation, dropout)

    def _transform(self, x, activation, dropout):
        if self.use_transformation and x.is_cuda and x.dim() == 2 and self.cluster.is_training and \
                (activation == "relu" or not dropout):
            kept = self.cluster.assignment(x)
            # cluster mean, the Linear on the representatives and the fused reconstruction as ONE autograd node
            # (ref: the three modules chained in model/compressgnn/gcn.py:27-34)
            plan = _native.index_plan(kept.index, kept.counts.numel()).native if x.size(0) else None
            return _native.differentiable(_native.ops().transform, x, kept.index, kept.counts, plan, self.lin.weight,
                                          self.lin.bias, activation == "relu", float(dropout))
        if self.use_transformation:
            reps, index = self.cluster(x)
            fused = dropout if activation == "relu" else 0.0
            x = self.reconstruct(F.linear(reps, self.lin.weight, None), index, bias=self.lin.bias,
                                 activation=activation, dropout=fused)
            return F.dropout(x, p=dropout) if dropout and not fused else x
        x = self.lin(x)
        x = x.relu() if activation == "relu" else x
        return F.dropout(x, p=dropout) if dropout else x


class GCN(torch.nn.Module):
    residual = False  # (of a model that was saved whole before there was a choice)

    def __init__(self, in_features, out_features, hidden_features=128, param_H=1, dropout=0.3,
                 use_transformation=False, refresh_interval=1, num_layers=3, norm=None, residual=False, linear=None):
        """``norm="layer"`` normalises the hidden layers' outputs in front of their ReLU; ``residual`` adds a hidden layer's
        input to its output where the two are equally wide (neither is in the reference: deep stacks need them).
        ``linear="fused"`` computes the layers' products without the transformation with what follows them in one pass
        (``runtime.linear``): the same function, but its dropout draws from the package's generator."""
        super().__init__()
        dims = [in_features] + [hidden_features] * (num_layers - 1) + [out_features]
        self.layers = torch.nn.ModuleList(
            GNNLayer(dims[i], dims[i + 1], param_H=param_H, use_transformation=use_transformation,
                     refresh_interval=refresh_interval, activation="relu" if i + 1 < num_layers else None,
                     norm=norm if i + 1 < num_layers else None, linear=linear)
            for i in range(num_layers))
        self.dropout = dropout
        self.residual = residual

    def set_epoch(self, epoch, loss=None):
        for layer in self.layers:
            layer.set_epoch(epoch, loss=loss)

    def reset_cache(self):
        for layer in self.layers:
            layer.reset_cache()

    def _scores(self, x, edge_index, edge_weight, vertex_cnt, rule_cnt, dropout):
        last = len(self.layers) - 1
        for i, layer in enumerate(self.layers):
            # the hidden layers' ReLU and dropout are part of the layer (fused into the reconstruct kernel)
            p = self.dropout if (i != last and dropout and self.training) else 0.0
            added = {}
            if self.residual and i != last and layer.lin.in_features == layer.lin.out_features:
                added["residual"] = x
            x = layer(x=x, edge_index=edge_index, edge_weight=edge_weight, vertex_cnt=vertex_cnt, rule_cnt=rule_cnt,
                      dropout=p, **added)
        return x

    def forward(self, x: Tensor, edge_index, edge_weight=None, vertex_cnt: int = 0, rule_cnt: int = 0) -> Tensor:
        return F.log_softmax(self._scores(x, edge_index, edge_weight, vertex_cnt, rule_cnt, True), dim=1)

    def loss(self, x: Tensor, edge_index, target: Tensor, edge_weight=None, vertex_cnt: int = 0, rule_cnt: int = 0,
             ignore_index: int = -100, reduction: str = "mean") -> Tensor:
        """Cross entropy of the class scores with ``target`` (one class per node, ``ignore_index`` outside the training
        set): what ``F.nll_loss(self(x, ...), target)`` computes, without the log-probabilities in between."""
        scores = self._scores(x, edge_index, edge_weight, vertex_cnt, rule_cnt, True)
        return _native.cross_entropy(scores, target, ignore_index, reduction)

    def inference(self, x: Tensor, edge_index, edge_weight=None, vertex_cnt: int = 0, rule_cnt: int = 0) -> Tensor:
        return F.log_softmax(self._scores(x, edge_index, edge_weight, vertex_cnt, rule_cnt, False), dim=1)
