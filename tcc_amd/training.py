"""Python host API of include/tcc_training.h: the operators that a GCN with
learned node rows, a deep one or one with a teacher trains with.

  embedding_lookup / embedding_grad   rows of a table, and their gradient
  group_norm / group_norm_grad        group norm over the node rows of each
                                      graph, channels last, with its activation
  layer_norm / layer_norm_grad        layer norm of every row, with the residual
                                      sum before it and its activation
  top_logits                          a teacher's largest logits of every row
  distill_loss / distill_grad         the loss against them, and its gradient
  grad_norm / clip_grad_norm          the global gradient norm, and clipping
  adam_step                           the Adam update, clipping as it reads

Tensors are fp32, bf16 or fp16 on the current device; sums, statistics and
moments are fp32 or wider inside, and outputs are rounded once.  All work runs
on torch's current stream or on `stream`, whose pool the outputs and
workspaces then come from; nothing synchronises, and a caller who passes
`stream` has it wait for the inputs and keeps them until it is done.  What a
call writes in place has a new version for autograd.  Tensors of another type
or place raise TypeError, sizes and strides that no call takes ValueError.  The
autograd nodes, modules and the model over these are in tcc_amd.gcn; the
checks and calls are in csrc/training_ext.cpp.
"""
from __future__ import annotations

import torch

from . import _lib

try:
    from . import _training as _ext
except ImportError as e:
    raise ImportError(f"the extension behind tcc_amd.training does not load ({e}): build it with "
                      "`python -m tcc_amd.build`") from e

_lib.lib()  # its errors are raised as _lib.TccError

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}  # TCC_ACT_*
REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}  # TCC_REDUCE_*


def _call(stream, f, *args):
    if stream is None:
        return f(*args)
    with torch.cuda.stream(stream):
        return f(*args)


def _code(codes: dict, kind: str, name: str) -> int:
    code = codes.get(name)
    if code is None:
        raise ValueError(f"{kind} must be one of {sorted(codes)} (got {name!r})")
    return code


def _activation(name: str) -> int:
    return _code(ACTIVATIONS, "activation", name)


def embedding_lookup(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0, padding_idx: int | None = None,
                     out: torch.Tensor | None = None, device_error: torch.Tensor | None = None,
                     stream=None) -> torch.Tensor:
    """scale * table[ids] (tcc_embedding_lookup), shape ids.shape + (D,), of
    the table's type.  Rows whose id is `padding_idx` are zeros; so are those
    whose id is no row of the table, which set TCC_DEVERR_FEATURE_INDEX in
    `device_error` (one int32 on the device)."""
    return _call(stream, _ext.embedding_lookup, table, ids, scale, padding_idx, out, device_error)


def embedding_grad(d_out: torch.Tensor, ids: torch.Tensor, num_rows: int, scale: float = 1.0,
                   padding_idx: int | None = None, grad: torch.Tensor | None = None, accumulate: bool = False,
                   device_error: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """The gradient [num_rows x D] of a table whose rows `ids` were looked up
    (tcc_embedding_grad), of d_out's type: scale times the sum of the rows of
    d_out of each id, in fp32 and in an order that the ids fix.  With
    accumulate=True the sums are added to `grad`, and only rows that occur
    are touched."""
    return _call(stream, _ext.embedding_grad, d_out, ids, num_rows, scale, padding_idx, grad, accumulate, device_error)


def group_norm(x: torch.Tensor, num_groups: int, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               offsets: torch.Tensor | None = None, eps: float = 1e-5, activation: str = "none",
               max_rows: int | None = None, stream=None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd) of act(group_norm(x)), channels last (tcc_group_norm).

    x [N x C] holds the node rows of a batch of graphs: segment b is the rows
    offsets[b] .. offsets[b+1] (int32 or int64, from 0 to N, never falling,
    which is not checked: rows outside all segments are not written; empty
    segments allowed); without offsets all rows are one segment.  x
    [B x ... x C] holds B segments of the same size.  Statistics run over a
    segment's rows and the channels of each of `num_groups` groups; mean and
    rstd are [B x G] fp32.  `weight` and `bias` [C] are of any one of the
    types.  `max_rows`, the longest segment's rows where the caller knows it,
    spares a batch of small graphs the launches for larger ones."""
    return _call(stream, _ext.group_norm, x, num_groups, weight, bias, offsets, eps, _activation(activation), max_rows)


def group_norm_grad(d_y: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, num_groups: int,
                    weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                    offsets: torch.Tensor | None = None, activation: str = "none", max_rows: int | None = None,
                    stream=None) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor | None]:
    """(dx, dweight, dbias) of group_norm (tcc_group_norm_grad), from d_y of
    x's shape and type and the forward's mean and rstd: dx of x's type,
    dweight and dbias [C] fp32 (None where there is no weight or bias)."""
    return _call(stream, _ext.group_norm_grad, d_y, x, mean, rstd, num_groups, weight, bias, offsets,
                 _activation(activation), max_rows)


def held_by_default_stream(tensors) -> bool:
    """Whether a gradient of one of these (None is none) would run through a node
    that an eager pass made on the default stream, or to a leaf whose gradient a
    living graph accumulates there, however far behind the tensor."""
    return _ext.held_by_default_stream(list(tensors))


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               residual: torch.Tensor | None = None, eps: float = 1e-5, activation: str = "none",
               stream=None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, h, mean, rstd) of act(layer_norm(h)) over the last dimension
    (tcc_layer_norm), with h = x + residual rounded to x's type, or x itself
    where there is no residual (of x's shape and type).  mean and rstd are fp32
    of shape x.shape[:-1].  `weight` and `bias` [C] are of any one of the types."""
    return _call(stream, _ext.layer_norm, x, weight, bias, residual, eps, _activation(activation))


def layer_norm_grad(d_y: torch.Tensor, h: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                    weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                    d_sum: torch.Tensor | None = None, activation: str = "none", stream=None,
                    parameters: bool = True) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor | None]:
    """(dx, dweight, dbias) of layer_norm (tcc_layer_norm_grad), from d_y of
    h's shape and type, the forward's h, mean and rstd, and `d_sum`, the
    gradient that h has from its other uses: dx of h's type is the gradient of
    x and of residual alike, dweight and dbias [C] are fp32 (None where there
    is no weight or bias, and without `parameters`, which spares their sums)."""
    return _call(stream, _ext.layer_norm_grad, d_y, h, mean, rstd, weight, bias, d_sum, _activation(activation), parameters)


def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0,
               stream=None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(values, ids, rest) of logits [n x C] (tcc_top_logits): the `k` largest of
    each row and their classes (int32), largest first, the lowest class first
    among equals, NaN above all, and one fp32 logit that stands for the other
    classes at this temperature (-inf where there are none).  k is at most 64."""
    return _call(stream, _ext.top_logits, logits, k, temperature)


def distill_loss(logits: torch.Tensor, values: torch.Tensor, ids: torch.Tensor, rest: torch.Tensor | None = None,
                 temperature: float = 1.0, weight: torch.Tensor | None = None, reduction: str = "mean",
                 device_error: torch.Tensor | None = None,
                 stream=None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """(loss, stats, total) of a student's logits [n x C] against a teacher's
    entries (tcc_distill_loss): T^2 times the divergence KL(p || q) of each row,
    p the softmax of values / T over the row's entries, q that of logits / T over
    all classes.  With `rest` (of the same temperature) both have one more class,
    which holds what the entries leave; without it p is that of the entries alone
    (a single entry at temperature 1: cross-entropy).  `weight` [n] fp32 weighs
    the rows; those of weight 0 are not read.  The loss is the mean over the
    weights, the sum, or the rows' own (reduction="none").  An id of -1 is no
    entry; others that are no class are none either and set
    TCC_DEVERR_FEATURE_INDEX in `device_error` (one int32 on the device).
    stats [n x 4] and total (None unless the loss is a mean with weights) are
    for the gradient."""
    return _call(stream, _ext.distill_loss, logits, values, ids, rest, temperature, weight,
                 _code(REDUCTIONS, "reduction", reduction), device_error)


def distill_grad(d_loss: torch.Tensor, logits: torch.Tensor, values: torch.Tensor, ids: torch.Tensor,
                 stats: torch.Tensor, rest: torch.Tensor | None = None, temperature: float = 1.0,
                 weight: torch.Tensor | None = None, total: torch.Tensor | None = None, reduction: str = "mean",
                 stream=None) -> torch.Tensor:
    """The gradient of distill_loss in the logits, of their type
    (tcc_distill_grad), from d_loss (fp32, of the loss's shape), the loss's
    arguments, and the stats and total that it gave."""
    return _call(stream, _ext.distill_grad, d_loss, logits, values, ids, stats, rest, temperature, weight, total,
                 _code(REDUCTIONS, "reduction", reduction))


def grad_norm(grads, stream=None) -> torch.Tensor:
    """sqrt of the sum of squares over every tensor of `grads`, as a 0-d fp32
    device tensor (tcc_grad_norm): what clip_grad_norm clips to."""
    return _call(stream, _ext.grad_norm, list(grads))


def clip_grad_norm(grads, max_norm: float, out=None, stream=None) -> torch.Tensor:
    """Scales every tensor of `grads` by min(1, max_norm / (norm + 1e-6)), in
    place or into the tensors of `out`, and returns the norm before, a 0-d
    fp32 device tensor (tcc_clip_grad_norm): torch.nn.utils.clip_grad_norm_
    without its host checks.  A tensor may have strides as long as its
    elements are rows at one distance."""
    return _call(stream, _ext.clip_grad_norm, list(grads), max_norm, None if out is None else list(out))


def adam_step(params, grads, exp_avg, exp_avg_sq, step: torch.Tensor, lr: float = 1e-3,
              betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0,
              decoupled: bool = True, max_norm: float | None = None, stream=None) -> torch.Tensor | None:
    """One Adam step in place over lists of parameters, gradients and fp32
    moments, and step += 1 (an int64 device scalar), as torch.optim.AdamW
    (decoupled=False: Adam) computes it (tcc_adam_step).  With `max_norm` the
    gradients are clipped to it as clip_grad_norm does, as they are read:
    `grads` stay as they are, and the norm before clipping is returned."""
    return _call(stream, _ext.adam_step, list(params), list(grads), list(exp_avg), list(exp_avg_sq), step, lr, betas[0],
                 betas[1], eps, weight_decay, decoupled, max_norm)
