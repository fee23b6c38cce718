"""Two-layer GCN on the block-sparse SpMM: the caller of the hot path
(train/tcgnn_conv_release.py:49-250), on MI355X.

CNICSPMMFunction mirrors the reference's autograd function
(tcgnn_conv_release.py:49-166):
  forward : AX = A·X with the spmm_cnic split (BCSR part + BCSC part,
            spmm_launcher.cu:30-271), out = AX·W                (:130-134)
  backward: dW = AXᵀ·dY, G = Aᵀ·dY, dX = G·Wᵀ                    (:147-154)
The weight gradients AXᵀ·dY and Xᵀ·G are tall-skinny products over all nodes
(tcc_dense_tn: K split over workgroups on MFMA, of fp32 accuracy), where library GEMMs
reach a fraction of the GPU on this shape.
The reference's G = torch.sparse.mm(Aᵀ, dY) over unit values (:139-142, :152)
is the block-sparse transposed gather over a BCSC of the whole A
(tcc_bcsc_transpose_spmm), and dX is computed only when the layer's input
needs a gradient (the reference computes and discards it for the first
layer, whose input is the feature table).

A later layer whose output is narrower than its input (the last layer:
256 -> 2 classes) is evaluated as A·(X·W) instead of (A·X)·W — the same
product in exact arithmetic, with the SpMM at the output width and the
backward G = Aᵀ·dY, dW = Xᵀ·G, dX = G·Wᵀ (the aggregate-then-transform order
of :133-134 would gather 256-wide rows for a 2-wide result).

The first layer reads X through the hot/cold feature source of
spmm_kernel.cu:129-153: edges whose source row is hot (in the HBM feature
cache) go to the BCSR gather, edges with cold sources to the BCSC scatter,
which reads each cold row once per column window from mapped pinned host
memory.  Later layers read device-resident X and put every edge in the
BCSR gather.

GCN = conv1 (first layer, F_in -> hidden), ReLU, dropout, conv_final
(hidden -> classes), weights xavier-uniform (tcgnn_conv_release.py:168-250);
trained with cross-entropy and Adam (:448-449).  Without dropout and with at
most 8 classes the two layers run as one autograd node whose backward forms
both weight gradients in one pass (TwoLayerFunction).

EmbeddingGCN is the model where the node rows are learned (graphs without
features): rows of an embedding table (NodeEmbedding), conv1, a group norm
over the node rows of each graph with its activation (NodeGroupNorm),
conv_final, trained by ClippedAdam, over tcc_amd.training.  With layer norms
(NodeLayerNorm) it may have residual blocks between the two convolutions.  A
smaller model learns from a larger one's largest logits (top_logits of
tcc_amd.training, DistillationLoss).  The reference, whose features are given
and whose labels are classes, has no counterpart.
"""
from __future__ import annotations

import functools

import numpy as np
import torch

from . import swtcf
from .hostmem import PinnedArray


class _FirstOrder(torch.autograd.Function):
    """A gradient that is no constant (it depends on `sources`) but cannot be
    differentiated again."""

    @staticmethod
    def forward(ctx, name, grad, *sources):
        ctx.name = name
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError(f"{ctx.name} has no second derivative: its gradient was asked for with create_graph=True "
                           "and then differentiated")


def _first_order(backward):
    """For the backward of a node whose gradients are computed outside
    autograd: under create_graph=True they would count as constants.  Here a
    second differentiation raises instead."""

    @functools.wraps(backward)
    def checked(ctx, *grads):
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not torch.is_grad_enabled():
            return out
        sources = [t for t in (*grads, *ctx.saved_tensors) if t is not None and t.requires_grad]
        if not sources:
            return out
        several = isinstance(out, tuple)
        name = type(ctx).__name__.removesuffix("Backward")
        out = [t if t is None else _FirstOrder.apply(name, t, *sources) for t in (out if several else (out,))]
        return tuple(out) if several else out[0]

    return checked


class LayerGraph:
    """The block matrices of one layer's A [num_rows x num_cols]:
    forward BCSR (edges whose source is on the device) and BCSC (edges whose
    source is cold, or None), and the backward BCSC of every edge (shared
    between layers over the same A)."""

    def __init__(self, rows: torch.Tensor, cols: torch.Tensor, num_rows: int, num_cols: int,
                 hot_src: torch.Tensor | None = None, backward_bcsc: swtcf.BlockMatrix | None = None):
        rows, cols = rows.cuda(), cols.cuda()
        r = rows.to(torch.int32).contiguous()
        c = cols.to(torch.int32).contiguous()
        self.num_rows, self.num_cols = num_rows, num_cols
        if hot_src is None:
            self.bcsr = swtcf.coo_to_bcsr(r, c, None, num_rows, num_cols)
            self.bcsc = None
        else:
            h = hot_src[cols.long()]
            self.bcsr = _bcsr_or_empty(r[h].contiguous(), c[h].contiguous(), num_rows, num_cols)
            self.bcsc = _bcsc_or_empty(r[~h].contiguous(), c[~h].contiguous(), num_rows, num_cols)
        self.bwd = backward_bcsc if backward_bcsc is not None else swtcf.coo_to_bcsc(r, c, None, num_rows, num_cols)

    def aggregate(self, F: int, x: torch.Tensor | None = None, source=None) -> torch.Tensor:
        """AX [num_rows x F] (a view of the (RW+1)*8-row denseC buffer)."""
        RW = self.bcsr.view.num_rowWindows
        denseC = swtcf._empty(((RW + 1) * 8, F), torch.float32, "cuda")
        if source is not None:
            bcsc = self.bcsc if self.bcsc is not None else _EMPTY_BCSC
            swtcf.spmm_cnic_forward_mixed(self.bcsr, bcsc, source, denseC, F)
        elif self.bcsc is not None:
            swtcf.spmm_cnic_forward(self.bcsr, self.bcsc, x, denseC)
        else:
            denseC[RW * 8:].zero_()
            swtcf.bcsr_spmm(self.bcsr, x, denseC[: RW * 8])
        return denseC[: self.num_rows]

    def transpose_aggregate(self, dY: torch.Tensor) -> torch.Tensor:
        """Aᵀ dY [num_cols x F]."""
        out = swtcf.bcsc_transpose_spmm(self.bwd, dY.contiguous())
        return out[: self.num_cols]


def _bcsr_or_empty(r, c, num_rows, num_cols):
    if r.numel() > 0:
        return swtcf.coo_to_bcsr(r, c, None, num_rows, num_cols)
    RW = (num_rows + 7) // 8
    keep = (torch.zeros(RW + 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"),
            torch.full((8,), -1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda"))
    return swtcf.wrap_bcsr(num_rows, num_cols, 0, 0, RW, *keep)


def _bcsc_or_empty(r, c, num_rows, num_cols):
    if r.numel() > 0:
        return swtcf.coo_to_bcsc(r, c, None, num_rows, num_cols)
    return _EMPTY_BCSC


class _EmptyBCSC:
    view = swtcf.BCSC()  # no windows: the scatter launches nothing


_EMPTY_BCSC = _EmptyBCSC()


class CNICSPMMFunction(torch.autograd.Function):
    """out = (A X) W with the reference's backward (tcgnn_conv_release.py:49-166)."""

    @staticmethod
    def forward(ctx, graph: LayerGraph, source, x, weights):
        F = weights.shape[0]
        AX = graph.aggregate(F, x=None if source is not None else x.contiguous(), source=source)
        ctx.graph = graph
        ctx.save_for_backward(AX, weights)
        return torch.mm(AX, weights)

    @staticmethod
    @_first_order
    def backward(ctx, d_output):
        AX, weights = ctx.saved_tensors
        grad_weights = swtcf.dense_tn(AX, d_output)  # AXᵀ·dY (:150)
        grad_x = None
        if ctx.needs_input_grad[2]:
            grad_sp = ctx.graph.transpose_aggregate(d_output)
            grad_x = torch.mm(grad_sp, weights.t())
        return None, None, grad_x, grad_weights


class TransformFirstFunction(torch.autograd.Function):
    """out = A (X W), the same product as (A X) W associated the other way,
    for layers whose output is narrower than their input: the SpMM then runs
    at the output width (2 instead of 256 for the GCN's last layer).
    Backward: G = Aᵀ dY (needed for dX in either order), dW = Xᵀ G,
    dX = G Wᵀ — AX is never formed."""

    @staticmethod
    def forward(ctx, graph: LayerGraph, x, weights):
        xw = torch.mm(x, weights).contiguous()
        out = graph.aggregate(weights.shape[1], x=xw)
        ctx.graph = graph
        ctx.save_for_backward(x, weights)
        return out

    @staticmethod
    @_first_order
    def backward(ctx, d_output):
        x, weights = ctx.saved_tensors
        grad_sp = ctx.graph.transpose_aggregate(d_output)
        grad_weights = swtcf.dense_tn(x, grad_sp)  # Xᵀ·G
        grad_x = torch.mm(grad_sp, weights.t()) if ctx.needs_input_grad[1] else None
        return None, grad_x, grad_weights


class GCNConv(torch.nn.Module):
    def __init__(self, input_dim: int, output_dim: int, first_layer: bool = False):
        super().__init__()
        self.first_layer = first_layer
        self.weights = torch.nn.Parameter(torch.empty(input_dim, output_dim))
        torch.nn.init.xavier_uniform_(self.weights)

    def forward(self, graph: LayerGraph, source=None, x: torch.Tensor | None = None) -> torch.Tensor:
        in_dim, out_dim = self.weights.shape
        if not self.first_layer and out_dim < in_dim:
            # A(XW) = (AX)W: aggregate at the narrower width
            return TransformFirstFunction.apply(graph, x, self.weights)
        return CNICSPMMFunction.apply(graph, source if self.first_layer else None, x, self.weights)


class TwoLayerFunction(torch.autograd.Function):
    """conv_final(relu(conv1(X))) as one autograd node, for a last layer
    narrower than the hidden one and no dropout (what the layer-by-layer
    functions compute, with the backward fused):
      forward : AX = A X (first-layer source), then H = relu(AX W1) and
                XW = H W2 in one pass (tcc_gcn_relu_forward, F <= 128,
                hidden <= 256, classes <= 4), out = A XW
      backward: G = Aᵀ dOut, then one pass over AX, H and G for
                dW1 = AXᵀ((G W2ᵀ) ⊙ [H > 0]) and dW2 = Hᵀ G
                (tcc_gcn_relu_grad): G W2ᵀ, the relu mask and the hidden
                gradient are never written to memory."""

    @staticmethod
    def forward(ctx, g1: LayerGraph, g2: LayerGraph, source, w1, w2):
        AX = g1.aggregate(w1.shape[0], source=source)
        if swtcf.gcn_relu_forward_supported(w1.shape[0], w1.shape[1], w2.shape[1]):
            H, XW = swtcf.gcn_relu_forward(AX, w1, w2)  # one pass, H written once
        else:
            H = torch.relu(torch.mm(AX, w1))
            XW = torch.mm(H, w2).contiguous()
        out = g2.aggregate(w2.shape[1], x=XW)
        ctx.g2 = g2
        ctx.save_for_backward(AX, H, w2)
        return out

    @staticmethod
    @_first_order
    def backward(ctx, d_output):
        AX, H, w2 = ctx.saved_tensors
        G = ctx.g2.transpose_aggregate(d_output)
        dw1, dw2 = swtcf.gcn_relu_grad(AX, H, G, w2)
        return None, None, None, dw1, dw2


# Class counts the fused two-layer backward takes (tcc_gcn_relu_grad).
FUSED_MAX_CLASSES = 8


class GCN(torch.nn.Module):
    def __init__(self, num_features: int, hidden_dim: int, num_classes: int, dropout: float = 0.0,
                 fused: bool = True):
        super().__init__()
        self.conv1 = GCNConv(num_features, hidden_dim, first_layer=True)
        self.conv_final = GCNConv(hidden_dim, num_classes)
        self.dropout = torch.nn.Dropout(p=dropout)
        self.fused = fused

    def forward(self, g1: LayerGraph, g2: LayerGraph, source) -> torch.Tensor:
        w1, w2 = self.conv1.weights, self.conv_final.weights
        no_dropout = self.dropout.p == 0.0 or not self.training
        if self.fused and no_dropout and w2.shape[1] < w2.shape[0] and w2.shape[1] <= FUSED_MAX_CLASSES:
            return TwoLayerFunction.apply(g1, g2, source, w1, w2)
        x = torch.relu(self.conv1(g1, source=source))
        x = self.dropout(x)
        return self.conv_final(g2, x=x)


class EmbeddingFunction(torch.autograd.Function):
    """scale * table[ids] with the gradient of the table by sorted ids
    (tcc_amd.training.embedding_lookup / embedding_grad)."""

    @staticmethod
    def forward(ctx, table, ids, scale, padding_idx, device_error):
        from . import training

        ctx.save_for_backward(ids)
        ctx.args = table.shape[0], scale, padding_idx
        return training.embedding_lookup(table, ids, scale=scale, padding_idx=padding_idx, device_error=device_error)

    @staticmethod
    @_first_order
    def backward(ctx, d_out):
        from . import training

        (ids,) = ctx.saved_tensors
        num_rows, scale, padding_idx = ctx.args
        return training.embedding_grad(d_out, ids, num_rows, scale=scale, padding_idx=padding_idx), None, None, None, None


class GroupNormFunction(torch.autograd.Function):
    """act(group_norm(x)) over the rows of each segment, channels last
    (tcc_amd.training.group_norm / group_norm_grad)."""

    @staticmethod
    def forward(ctx, x, weight, bias, num_groups, offsets, eps, activation, max_rows):
        from . import training

        y, mean, rstd = training.group_norm(x, num_groups, weight, bias, offsets=offsets, eps=eps, activation=activation,
                                            max_rows=max_rows)
        ctx.save_for_backward(x, weight, bias, offsets, mean, rstd)
        ctx.args = num_groups, activation, max_rows
        return y

    @staticmethod
    @_first_order
    def backward(ctx, d_y):
        from . import training

        x, weight, bias, offsets, mean, rstd = ctx.saved_tensors
        num_groups, activation, max_rows = ctx.args
        dx, dw, db = training.group_norm_grad(d_y, x, mean, rstd, num_groups, weight, bias, offsets=offsets,
                                              activation=activation, max_rows=max_rows)
        dw = None if dw is None else dw.to(weight.dtype)
        db = None if db is None else db.to(bias.dtype)
        return dx, dw, db, None, None, None, None, None


def _capturable(*inputs) -> None:
    """Refuses what would end the process: a backward pass, captured into a graph,
    through nodes or to leaves that an eager graph made on the default stream still
    holds, behind these inputs."""
    if torch.is_grad_enabled() and torch.cuda.is_current_stream_capturing():
        from . import training

        if training.held_by_default_stream(inputs):
            raise RuntimeError("an output of an earlier eager pass over these parameters is alive, whose gradients belong "
                               "to the default stream: drop it before the capture, detach it, or make it on a side stream")


class LayerNormFunction(torch.autograd.Function):
    """act(layer_norm(x)), or (act(layer_norm(h)), h) of h = x + residual
    (tcc_amd.training.layer_norm / layer_norm_grad)."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, activation):
        from . import training

        y, h, mean, rstd = training.layer_norm(x, weight, bias, residual=residual, eps=eps, activation=activation)
        ctx.save_for_backward(h, weight, bias, mean, rstd)
        ctx.activation, ctx.summed = activation, residual is not None
        ctx.set_materialize_grads(False)
        return (y, h) if ctx.summed else y

    @staticmethod
    @_first_order
    def backward(ctx, d_y, d_sum=None):
        from . import training

        if d_y is None:  # only the sum was used
            return d_sum, d_sum, None, None, None, None
        h, weight, bias, mean, rstd = ctx.saved_tensors
        dx, dw, db = training.layer_norm_grad(d_y, h, mean, rstd, weight, bias, d_sum=d_sum, activation=ctx.activation,
                                              parameters=any(ctx.needs_input_grad[2:4]))
        dw = None if dw is None else dw.to(weight.dtype)
        db = None if db is None else db.to(bias.dtype)
        return dx, dx if ctx.summed else None, dw, db, None, None


class DistillationFunction(torch.autograd.Function):
    """tcc_amd.training.distill_loss with its gradient in the logits; the
    teacher's entries and the weights are constants."""

    @staticmethod
    def forward(ctx, logits, values, ids, rest, weight, temperature, reduction, device_error):
        from . import training

        loss, stats, total = training.distill_loss(logits, values, ids, rest=rest, temperature=temperature, weight=weight,
                                                   reduction=reduction, device_error=device_error)
        ctx.save_for_backward(logits, values, ids, rest, weight, stats, total)
        ctx.args = temperature, reduction
        return loss

    @staticmethod
    @_first_order
    def backward(ctx, d_loss):
        from . import training

        logits, values, ids, rest, weight, stats, total = ctx.saved_tensors
        temperature, reduction = ctx.args
        d = training.distill_grad(d_loss, logits, values, ids, stats, rest=rest, temperature=temperature, weight=weight,
                                  total=total, reduction=reduction)
        return d, None, None, None, None, None, None, None


class NodeEmbedding(torch.nn.Module):
    """A learned row of `dim` values for each of `num_nodes` nodes; forward
    gives scale * rows of `ids` (sqrt(dim) times rows that begin at
    1 / sqrt(dim) have unit variance).  The row of `padding_idx` stays zero.
    error() reports ids outside the table, as FeatureTable's does."""

    def __init__(self, num_nodes: int, dim: int, scale: float | None = None, padding_idx: int | None = None,
                 device="cuda", dtype=torch.float32):
        super().__init__()
        self.scale = dim**0.5 if scale is None else scale
        self.padding_idx = padding_idx
        self.weight = torch.nn.Parameter(torch.randn((num_nodes, dim), device=device).div_(dim**0.5).to(dtype))
        if padding_idx is not None:
            with torch.no_grad():
                self.weight[padding_idx].zero_()
        # a buffer, so that it moves with the module; no part of checkpoints
        self.register_buffer("device_error", torch.zeros(1, dtype=torch.int32, device=device), persistent=False)

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return EmbeddingFunction.apply(self.weight, ids, self.scale, self.padding_idx, self.device_error)

    def error(self) -> int:
        """TCC_DEVERR_FEATURE_INDEX if an id fell outside the table since the
        last call, else 0; synchronises the device and clears the word."""
        v = int(self.device_error.item())
        self.device_error.zero_()
        return v


class NodeGroupNorm(torch.nn.Module):
    """Group norm over the node rows of each graph (the rows offsets[b] ..
    offsets[b+1] of x; all rows without offsets) with its activation."""

    def __init__(self, num_groups: int, channels: int, activation: str = "none", eps: float = 1e-5, device="cuda"):
        super().__init__()
        self.num_groups, self.activation, self.eps = num_groups, activation, eps
        self.weight = torch.nn.Parameter(torch.ones(channels, device=device))
        self.bias = torch.nn.Parameter(torch.zeros(channels, device=device))

    def forward(self, x: torch.Tensor, offsets: torch.Tensor | None = None, max_rows: int | None = None) -> torch.Tensor:
        return GroupNormFunction.apply(x, self.weight, self.bias, self.num_groups, offsets, self.eps, self.activation,
                                       max_rows)


class NodeLayerNorm(torch.nn.Module):
    """Layer norm of every row with its activation.  With `residual`, the norm of
    x + residual and that sum: (y, h)."""

    def __init__(self, channels: int, activation: str = "none", eps: float = 1e-5, device="cuda"):
        super().__init__()
        self.activation, self.eps = activation, eps
        self.weight = torch.nn.Parameter(torch.ones(channels, device=device))
        self.bias = torch.nn.Parameter(torch.zeros(channels, device=device))

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        _capturable(x, residual, self.weight, self.bias)
        return LayerNormFunction.apply(x, residual, self.weight, self.bias, self.eps, self.activation)


class EmbeddingGCN(torch.nn.Module):
    """conv_final(act(norm(conv1(embedding[ids])))) over a batch of graphs
    (their block-diagonal A as one LayerGraph, `offsets` their first rows) or
    one graph (no offsets).  The norm is a group norm over each graph's rows, or
    norm="layer" one of each row; between that and conv_final lie then `blocks`
    residual ones, h = h + conv(act(norm(h)))."""

    def __init__(self, num_nodes: int, dim: int, hidden_dim: int, num_classes: int, num_groups: int = 8,
                 activation: str = "relu", padding_idx: int | None = None, norm: str = "group", blocks: int = 0):
        super().__init__()
        if norm not in ("group", "layer"):
            raise ValueError(f"norm must be 'group' or 'layer' (got {norm!r})")
        if blocks < 0 or (blocks > 0 and norm != "layer"):
            raise ValueError("residual blocks go with layer norms")
        self.embedding = NodeEmbedding(num_nodes, dim, padding_idx=padding_idx)
        self.conv1 = GCNConv(dim, hidden_dim).cuda()
        self.layer_norm = norm == "layer"
        self.norm = (NodeLayerNorm(hidden_dim, activation) if self.layer_norm
                     else NodeGroupNorm(num_groups, hidden_dim, activation))
        self.convs = torch.nn.ModuleList(GCNConv(hidden_dim, hidden_dim).cuda() for _ in range(blocks))
        self.norms = torch.nn.ModuleList(NodeLayerNorm(hidden_dim, activation) for _ in range(blocks))
        self.conv_final = GCNConv(hidden_dim, num_classes).cuda()

    def forward(self, graph: LayerGraph, ids: torch.Tensor, offsets: torch.Tensor | None = None,
                max_rows: int | None = None) -> torch.Tensor:
        h = self.conv1(graph, x=self.embedding(ids))
        y = self.norm(h) if self.layer_norm else self.norm(h, offsets, max_rows)
        for conv, norm in zip(self.convs, self.norms):
            y, h = norm(conv(graph, x=y), h)
        return self.conv_final(graph, x=y)


class DistillationLoss(torch.nn.Module):
    """The loss of logits against a teacher's entries, (values, ids, rest) as
    tcc_amd.training.top_logits gives them at this temperature (rest may be None:
    then the teacher's probabilities are those of the entries alone).  It takes
    the place of the class labels' loss in train_epoch and
    train_embedding_epoch, and the entries that of the labels.  Rows of weight 0
    do not count.  error() reports ids that are no class."""

    def __init__(self, temperature: float = 1.0, weight: torch.Tensor | None = None, reduction: str = "mean", device="cuda"):
        super().__init__()
        self.temperature, self.reduction = temperature, reduction
        self.register_buffer("weight", weight, persistent=False)
        self.register_buffer("device_error", torch.zeros(1, dtype=torch.int32, device=device), persistent=False)

    def forward(self, pred: torch.Tensor, entries) -> torch.Tensor:
        values, ids, rest = entries
        if any(t is not None and t.requires_grad for t in (values, rest, self.weight)):
            raise ValueError("the teacher's entries and the weights are constants: detach them")
        _capturable(pred)
        return DistillationFunction.apply(pred, values, ids, rest, self.weight, self.temperature, self.reduction,
                                          self.device_error)

    def error(self) -> int:
        """TCC_DEVERR_FEATURE_INDEX if an id was no class (and not -1) since the
        last call, else 0; synchronises the device and clears the word."""
        v = int(self.device_error.item())
        self.device_error.zero_()
        return v


class ClippedAdam(torch.optim.Optimizer):
    """Adam over one group of parameters whose gradients are clipped to
    `max_norm` as the update reads them (tcc_amd.training.adam_step): step()
    leaves the gradients as they are and returns their norm, a device scalar
    (None without max_norm).  step(closure) returns the closure's loss, as
    torch's optimizers do; the norm is in `norm` after either.  Steps are
    counted for each parameter, from its first gradient on; where the counts
    differ, the clipped gradients are written once, in their type, for an
    update a count.  Nothing synchronises but load_state_dict."""

    norm = None

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0,
                 decoupled: bool = True, max_norm: float | None = None):
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, decoupled=decoupled,
                                      max_norm=max_norm))

    def add_param_group(self, param_group):
        if self.param_groups:
            raise ValueError("ClippedAdam takes one group of parameters: the norm is over all of them")
        super().add_param_group(param_group)

    def load_state_dict(self, state_dict):
        """The moments come back in fp32 whatever the parameters' type, and the
        counts on their device: torch would round the first to the parameters'
        type and leave the second where the checkpoint was loaded to."""
        seen = []
        last = self.register_load_state_dict_pre_hook(lambda _, d: seen.append(d))
        try:
            super().load_state_dict(state_dict)
        finally:
            last.remove()
        (group,), state = seen[0]["param_groups"], seen[0]["state"]
        # checkpoints made while one count served all parameters have it in the group
        common = self.param_groups[0].pop("step", None)
        counts = {}
        for k, p in zip(group["params"], self.param_groups[0]["params"]):
            if not state.get(k):
                continue
            t = int(state[k].get("step", common))
            if t not in counts:
                counts[t] = torch.tensor(t, dtype=torch.int64, device=p.device)
            self.state[p]["step"] = counts[t]
            for name in ("exp_avg", "exp_avg_sq"):
                self.state[p][name] = state[k][name].to(p.device, torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self.norm = self._update()
        return self.norm if closure is None else loss

    def _update(self):
        from . import training

        group = self.param_groups[0]
        params = [p for p in group["params"] if p.grad is not None]
        if not params:
            return None
        ages = self._ages(params)
        grads, max_norm, norm = {p: p.grad for p in params}, group["max_norm"], None
        if max_norm is not None and len(ages) > 1:  # one norm for several updates
            out = [torch.empty_like(g) for g in grads.values()]
            norm = training.clip_grad_norm(list(grads.values()), max_norm, out=out)
            grads, max_norm = dict(zip(params, out)), None
        for some in ages:
            states = [self.state[p] for p in some]
            total = training.adam_step(some, [grads[p] for p in some], [s["exp_avg"] for s in states],
                                       [s["exp_avg_sq"] for s in states], states[0]["step"], lr=group["lr"],
                                       betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                                       decoupled=group["decoupled"], max_norm=max_norm)
            norm = total if norm is None else norm
        return norm

    def _ages(self, params):
        """`params` by the steps they have taken.  A count on the device serves
        all parameters that were always updated together; those that go on
        without the others get a copy of it."""
        fresh, ages = None, {}
        for p in params:
            state = self.state[p]
            if not state:
                if fresh is None:
                    fresh = torch.zeros((), dtype=torch.int64, device=p.device)
                state["step"] = fresh
                state["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
                state["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)
            ages.setdefault(id(state["step"]), []).append(p)
        here = set(params)
        left = {id(s["step"]) for p, s in self.state.items() if s and p not in here}
        for count, some in ages.items():
            if count in left:
                own = self.state[some[0]]["step"].clone()
                for p in some:
                    self.state[p]["step"] = own
        return list(ages.values())


class FeatureTable:
    """Features of every node: the hot rows (top `hot_fraction` of nodes by
    in-degree as a source, ties by id) in an HBM cache, all rows in mapped
    pinned host memory, and the tcc_feature_source that resolves them
    (cache_search_map = hot rank or -1, id_map = identity).

    packed=True stores both tables as TF32 rows packed by tcc_tf32_pack: the
    first layer's products round X to TF32 anyway, so they are the same bit
    for bit, and a cold row crosses the host link in 2.5 instead of 4 bytes
    per feature.  The default keeps the reference's fp32 rows."""

    def __init__(self, X: torch.Tensor, cols: torch.Tensor, hot_fraction: float = 0.2, packed: bool = False):
        n, F = X.shape
        deg = torch.bincount(cols.long().cuda(), minlength=n)
        n_hot = max(1, int(round(n * hot_fraction)))
        # degree descending, id ascending: sort by (-deg, id) through a stable sort
        order = torch.sort(-deg, stable=True).indices
        hot_ids = torch.sort(order[:n_hot]).values
        self.hot = torch.zeros(n, dtype=torch.bool, device="cuda")
        self.hot[hot_ids] = True
        csm = torch.full((n,), -1, dtype=torch.int32, device="cuda")
        csm[hot_ids] = torch.arange(n_hot, dtype=torch.int32, device="cuda")
        Xd = X.cuda()
        if packed:
            self.cache = swtcf.tf32_pack(Xd[hot_ids].contiguous())
            rows = swtcf.tf32_pack(Xd)
            self.host = PinnedArray((rows.numel(),), dtype=np.uint8)
            self.host.array[:] = rows.cpu().numpy()
            del rows
        else:
            self.cache = Xd[hot_ids].contiguous()
            self.host = PinnedArray((n, F))
            self.host.array[:] = X.cpu().numpy()
        del Xd
        self.ptrs = torch.tensor([self.cache.data_ptr()], dtype=torch.int64, device="cuda")
        self.ids = torch.arange(n, dtype=torch.int32, device="cuda")
        self.csm = csm
        fmt = swtcf.ROWS_TF32_PACKED if packed else swtcf.ROWS_FP32
        self.device_error = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.source = swtcf.feature_source(self.ids, csm, self.ptrs, n_hot, self.host.device_ptr, n * F, fmt,
                                           device_error=self.device_error)
        self.n_hot = n_hot
        self.packed = packed

    def error(self) -> int:
        """TCC_DEVERR_FEATURE_INDEX if a lookup fell outside the tables since
        the last call (or since the table was made), else 0; synchronises
        the device and clears the word, as spmm_cnic.feature_error does."""
        v = int(self.device_error.item())
        self.device_error.zero_()
        return v

    def free(self) -> None:
        self.host.free()


def build_gcn_graphs(rows: torch.Tensor, cols: torch.Tensor, n: int, hot: torch.Tensor):
    """(first-layer graph with the hot/cold split, later-layer graph), both
    over the same A, sharing the backward BCSC."""
    g2 = LayerGraph(rows, cols, n, n)
    g1 = LayerGraph(rows, cols, n, n, hot_src=hot, backward_bcsc=g2.bwd)
    return g1, g2


def cross_entropy(pred: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
    """Mean cross-entropy of logits [n x C] against class ids: the value and
    gradient of torch.nn.CrossEntropyLoss() (tcgnn_conv_release.py:437),
    evaluated as log_softmax, gather and mean.  torch's 2-D nll_loss with mean
    reduction runs its forward and backward in one workgroup (2.2 ms and
    1.1 ms for 2.45M rows on MI355X); these run across the GPU."""
    return -torch.log_softmax(pred, dim=1).gather(1, labels.view(-1, 1)).mean()


def train_epoch(model: GCN, g1: LayerGraph, g2: LayerGraph, source, labels: torch.Tensor,
                optimizer: torch.optim.Optimizer, loss_fcn=cross_entropy) -> torch.Tensor:
    """One full-graph step: forward, loss, backward, optimizer step
    (train_one_step, tcgnn_conv_release.py:284-329)."""
    pred = model(g1, g2, source)
    loss = loss_fcn(pred, labels)
    optimizer.zero_grad()
    loss.backward()
    optimizer.step()
    return loss


def train_embedding_epoch(model: EmbeddingGCN, graph: LayerGraph, ids: torch.Tensor, labels: torch.Tensor,
                          optimizer: torch.optim.Optimizer, offsets: torch.Tensor | None = None,
                          max_rows: int | None = None, loss_fcn=cross_entropy):
    """One step of EmbeddingGCN: forward, loss, backward, clipped update.
    Returns (loss, gradient norm), both on the device."""
    loss = loss_fcn(model(graph, ids, offsets, max_rows), labels)
    optimizer.zero_grad()
    loss.backward()
    return loss.detach(), optimizer.step()


def synthetic_labels(n: int, num_classes: int, seed: int) -> torch.Tensor:
    g = torch.Generator(device="cpu").manual_seed(seed + 2000)
    return torch.randint(0, num_classes, (n,), generator=g).cuda()

