"""Python host API of include/tcc_training.h: the operators that a GCN with
learned node rows trains with.

  embedding_lookup / embedding_grad   rows of a table, and their gradient
  group_norm / group_norm_grad        group norm over the node rows of each
                                      graph, channels last, with its activation
  grad_norm / clip_grad_norm          the global gradient norm, and clipping
  adam_step                           the Adam update, clipping as it reads

Tensors are fp32, bf16 or fp16 on the device; sums, statistics and moments
are fp32 or wider inside, and outputs are rounded once.  All work runs on
torch's current stream or on `stream`, whose pool the outputs and workspaces
then come from; nothing synchronises.  The autograd nodes, modules and the
model over these are in tcc_amd.gcn.
"""
from __future__ import annotations

import contextlib
import ctypes
from array import array

import torch

from . import _lib
from ._lib import check
from .swtcf import _empty, _ptr, _stream

F32, BF16, F16 = 0, 1, 2  # TCC_F32, TCC_BF16, TCC_F16
DTYPES = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}  # TCC_ACT_*
MAX_CHANNELS = 4096

_lib_handle = None
_norm_bytes = 0


def _library():
    global _lib_handle, _norm_bytes
    if _lib_handle is None:
        lib = _lib.lib()
        _norm_bytes = int(lib.tcc_grad_norm_workspace_bytes())
        _lib_handle = lib
    return _lib_handle


def _on(stream):
    """Allocations inside belong to `stream`'s work (None: the current stream)."""
    return contextlib.nullcontext() if stream is None else torch.cuda.stream(stream)


def _dtype(t: torch.Tensor, name: str) -> int:
    code = DTYPES.get(t.dtype)
    if code is None or not t.is_cuda:
        raise TypeError(f"{name} must be an fp32, bf16 or fp16 device tensor (got {t.dtype} on {t.device})")
    return code


def _same_device(t: torch.Tensor, *others) -> None:
    d = t.get_device()
    for o in others:
        if o is not None and o.get_device() != d:
            raise ValueError(f"tensors are on different devices ({t.device} and {o.device})")
    if d != torch.cuda.current_device():
        raise ValueError(f"tensors are on {t.device}, the current device is cuda:{torch.cuda.current_device()}")


def _rows(t: torch.Tensor, name: str) -> tuple[torch.Tensor, int]:
    """A matrix whose rows are contiguous, and its row stride (a copy where
    the rows are not contiguous or overlap)."""
    if t.dim() != 2 or t.shape[1] == 0:
        raise ValueError(f"{name} must be a matrix with columns (got {tuple(t.shape)})")
    n, d = t.shape
    if not t.is_contiguous():
        if t.stride(1) == 1 and t.stride(0) >= d:
            return t, t.stride(0)
        t = t.contiguous()
    return t, d


def _ids(ids: torch.Tensor) -> tuple[torch.Tensor, int]:
    if ids.dtype not in (torch.int32, torch.int64) or not ids.is_cuda:
        raise TypeError(f"ids must be an int32 or int64 device tensor (got {ids.dtype} on {ids.device})")
    return ids.contiguous(), 8 if ids.dtype == torch.int64 else 4


def _padding(padding_idx, num_rows: int) -> int:
    if padding_idx is None:
        return -1
    if not 0 <= padding_idx < num_rows:
        raise ValueError(f"padding_idx {padding_idx} is no row of a table of {num_rows}")
    return padding_idx


def _error_word(t):
    if t is not None and (t.dtype != torch.int32 or not t.is_cuda or t.numel() < 1):
        raise TypeError("device_error must be an int32 device tensor")
    return t


# ---------------------------------------------------------------- embedding


def embedding_lookup(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0, padding_idx: int | None = None,
                     out: torch.Tensor | None = None, device_error: torch.Tensor | None = None,
                     stream=None) -> torch.Tensor:
    """scale * table[ids] (tcc_embedding_lookup), shape ids.shape + (D,), of
    the table's type.  Rows whose id is `padding_idx` are zeros; so are those
    whose id is no row of the table, which set TCC_DEVERR_FEATURE_INDEX in
    `device_error` (one int32 on the device)."""
    lib = _library()
    code = _dtype(table, "table")
    table, ldt = _rows(table, "table")
    ids, width = _ids(ids)
    V, D = table.shape
    n = ids.numel()
    pad = _padding(padding_idx, V)
    _same_device(table, ids, out, _error_word(device_error))
    if out is None:
        with _on(stream):
            out = _empty((*ids.shape, D), table.dtype, table.device)
        ldo = D
    else:
        if out.dtype != table.dtype or tuple(out.shape) != (*ids.shape, D):
            raise ValueError(f"out must be {table.dtype} of shape {(*ids.shape, D)}")
        if out.dim() == 2 and out.stride(1) == 1 and out.stride(0) >= D:
            ldo = out.stride(0)
        elif out.is_contiguous():
            ldo = D
        else:
            raise ValueError("out must have contiguous rows")
    check(lib.tcc_embedding_lookup(table.data_ptr(), ldt, code, ids.data_ptr(), width, n, V, D, scale, pad,
                                   out.data_ptr(), ldo, _ptr(device_error), _stream(stream)))
    return out


def embedding_grad(d_out: torch.Tensor, ids: torch.Tensor, num_rows: int, scale: float = 1.0,
                   padding_idx: int | None = None, grad: torch.Tensor | None = None, accumulate: bool = False,
                   device_error: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """The gradient [num_rows x D] of a table whose rows `ids` were looked up
    (tcc_embedding_grad), of d_out's type: scale times the sum of the rows of
    d_out of each id, in fp32 and in an order that the ids fix.  With
    accumulate=True the sums are added to `grad`, and only rows that occur
    are touched."""
    lib = _library()
    code = _dtype(d_out, "d_out")
    if d_out.shape[:-1] != ids.shape:
        raise ValueError(f"d_out {tuple(d_out.shape)} does not have a row for each of the ids {tuple(ids.shape)}")
    ids, width = _ids(ids)
    n = ids.numel()
    D = d_out.shape[-1]
    d_out, ldd = _rows(d_out if d_out.dim() == 2 else d_out.reshape(n, D), "d_out")
    pad = _padding(padding_idx, num_rows)
    _same_device(d_out, ids, grad, _error_word(device_error))
    if grad is None:
        if accumulate:
            raise ValueError("accumulate=True needs a gradient to add to")
        with _on(stream):
            grad = _empty((num_rows, D), d_out.dtype, d_out.device)
        ldg = D
    else:
        if grad.dtype != d_out.dtype or tuple(grad.shape) != (num_rows, D):
            raise ValueError(f"grad must be {d_out.dtype} of shape {(num_rows, D)}")
        if grad.is_contiguous():
            ldg = D
        elif grad.stride(1) == 1 and grad.stride(0) >= D:
            ldg = grad.stride(0)
        else:
            raise ValueError("grad must have contiguous rows")
    need = int(lib.tcc_embedding_grad_workspace_bytes(n, num_rows, D))
    with _on(stream):
        ws = _empty(need, torch.uint8, d_out.device)
    check(lib.tcc_embedding_grad(d_out.data_ptr(), ldd, code, ids.data_ptr(), width, n, num_rows, D, scale, pad,
                                 grad.data_ptr(), ldg, int(accumulate), _ptr(device_error), ws.data_ptr(), need,
                                 _stream(stream)))
    return grad


# ---------------------------------------------------------------- group norm


def _norm_shape(x, num_groups, weight, bias, offsets, eps, activation, max_rows):
    """(tcc_group_norm_shape, x as rows, row stride, weight, bias, offsets)."""
    code = _dtype(x, "x")
    if x.dim() < 2:
        raise ValueError("x must be [rows x channels] or [segments x ... x channels]")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)} (got {activation!r})")
    C = x.shape[-1]
    if num_groups < 1 or C == 0 or C % num_groups:
        raise ValueError(f"{num_groups} groups do not divide {C} channels")
    if C > MAX_CHANNELS:
        raise ValueError(f"at most {MAX_CHANNELS} channels (got {C})")
    if offsets is not None:
        if x.dim() != 2:
            raise ValueError("offsets go with x of [rows x channels]")
        if offsets.dtype not in (torch.int32, torch.int64) or not offsets.is_cuda:
            raise TypeError(f"offsets must be an int32 or int64 device tensor (got {offsets.dtype} on {offsets.device})")
        if offsets.dim() != 1 or offsets.numel() < 2:
            raise ValueError("offsets are one more than the segments")
        offsets = offsets.contiguous()
        B = offsets.numel() - 1
    else:
        B = 1 if x.dim() == 2 else x.shape[0]
    rows, ld = _rows(x if x.dim() == 2 else x.reshape(-1, C), "x")
    N = rows.shape[0]
    if offsets is None:
        max_rows = N // B if B else 0
    if max_rows is not None and max_rows < 0:
        raise ValueError("max_rows is not negative")
    pcode = F32
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        pcode = _dtype(p, name)
        if p.dim() != 1 or p.shape[0] != C:
            raise ValueError(f"{name} must hold a value for each of the {C} channels (got {tuple(p.shape)})")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"weight and bias must be of one type (got {weight.dtype} and {bias.dtype})")
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    _same_device(rows, weight, bias, offsets)
    shape = _lib.GroupNormShape(N, B, max_rows or 0, C, num_groups, _ptr(offsets),
                                0 if offsets is None else offsets.element_size(), code, pcode,
                                ACTIVATIONS[activation], eps)
    return shape, rows, ld, weight, bias, offsets


def group_norm(x: torch.Tensor, num_groups: int, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               offsets: torch.Tensor | None = None, eps: float = 1e-5, activation: str = "none",
               max_rows: int | None = None, stream=None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd) of act(group_norm(x)), channels last (tcc_group_norm).

    x [N x C] holds the node rows of a batch of graphs: segment b is the rows
    offsets[b] .. offsets[b+1] (int32 or int64, from 0 to N, never falling;
    empty segments allowed); without offsets all rows are one segment.  x
    [B x ... x C] holds B segments of the same size.  Statistics run over a
    segment's rows and the channels of each of `num_groups` groups; mean and
    rstd are [B x G] fp32.  `weight` and `bias` [C] are of any one of the
    types.  `max_rows`, the longest segment's rows where the caller knows
    it, lets batches of small graphs run in one pass."""
    lib = _library()
    shape, rows, ld, weight, bias, offsets = _norm_shape(x, num_groups, weight, bias, offsets, eps, activation, max_rows)
    need = int(lib.tcc_group_norm_workspace_bytes(ctypes.byref(shape), 0))
    with _on(stream):
        y = _empty(x.shape, x.dtype, x.device)
        mean = _empty((shape.B, num_groups), torch.float32, x.device)
        rstd = _empty((shape.B, num_groups), torch.float32, x.device)
        ws = _empty(need, torch.uint8, x.device)
    check(lib.tcc_group_norm(ctypes.byref(shape), rows.data_ptr(), ld, _ptr(weight), _ptr(bias), y.data_ptr(), shape.C,
                             mean.data_ptr(), rstd.data_ptr(), ws.data_ptr(), need, _stream(stream)))
    return y, mean, rstd


def group_norm_grad(d_y: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, num_groups: int,
                    weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                    offsets: torch.Tensor | None = None, activation: str = "none", max_rows: int | None = None,
                    stream=None) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor | None]:
    """(dx, dweight, dbias) of group_norm (tcc_group_norm_grad), from d_y of
    x's shape and type and the forward's mean and rstd: dx of x's type,
    dweight and dbias [C] fp32 (None where there is no weight or bias)."""
    lib = _library()
    if d_y.dtype != x.dtype or d_y.shape != x.shape:
        raise ValueError(f"d_y must be {x.dtype} of shape {tuple(x.shape)} (got {d_y.dtype} {tuple(d_y.shape)})")
    shape, rows, ld, weight, bias, offsets = _norm_shape(x, num_groups, weight, bias, offsets, 0.0, activation, max_rows)
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.dtype != torch.float32 or tuple(t.shape) != (shape.B, num_groups) or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous float32 of shape {(shape.B, num_groups)}")
    C = shape.C
    d_rows, ldd = _rows(d_y if d_y.dim() == 2 else d_y.reshape(-1, C), "d_y")
    _same_device(rows, d_rows, mean, rstd)
    need = int(lib.tcc_group_norm_workspace_bytes(ctypes.byref(shape), 1))
    with _on(stream):
        dx = _empty(x.shape, x.dtype, x.device)
        dw = None if weight is None else _empty((C,), torch.float32, x.device)
        db = None if bias is None else _empty((C,), torch.float32, x.device)
        ws = _empty(need, torch.uint8, x.device)
    check(lib.tcc_group_norm_grad(ctypes.byref(shape), d_rows.data_ptr(), ldd, rows.data_ptr(), ld, mean.data_ptr(),
                                  rstd.data_ptr(), _ptr(weight), _ptr(bias), dx.data_ptr(), C, _ptr(dw), _ptr(db),
                                  ws.data_ptr(), need, _stream(stream)))
    return dx, dw, db


# ---------------------------------------------------------------- gradients


def _collapse(shape, stride) -> tuple[int, int, int] | None:
    """(rows, cols, row stride) of the elements in the order given, or None."""
    dims = [(n, s) for n, s in zip(shape, stride) if n != 1]
    cols, step = 1, 1
    while dims and dims[-1][1] == step:
        cols *= dims[-1][0]
        step = cols
        dims.pop()
    if not dims:
        return 1, cols, cols
    rows, ld = dims[-1]
    step = rows * ld
    for n, s in reversed(dims[:-1]):
        if s != step:
            return None
        rows *= n
        step = rows * ld
    return (rows, cols, ld) if ld >= cols else None


def _layouts(tensors, names) -> list[tuple[int, int, int]]:
    """The same elements of several tensors of one shape in the same order,
    each as rows `ld` apart: the first one's order in memory."""
    first = tensors[0]
    order = sorted(range(first.dim()), key=lambda d: -first.stride(d))
    found = []
    for t, name in zip(tensors, names):
        lay = _collapse([t.shape[d] for d in order], [t.stride(d) for d in order])
        if lay is None:
            raise ValueError(f"{name} of shape {tuple(t.shape)} and strides {t.stride()} is not rows at one distance "
                             f"in the order of {names[0]}")
        found.append(lay)
    split = next((f for f in found if f[0] > 1), found[0])
    for k, (f, name) in enumerate(zip(found, names)):
        if f[:2] != split[:2]:
            if f[0] > 1:
                raise ValueError(f"{name} is split into rows in another way than the other tensors")
            found[k] = (split[0], split[1], split[1])
    return found


def _lists(lists, names):
    """Each list as an array of tcc_tensor: for every tensor, the operands of
    one shape on one device.  Returns the arrays, in the lists' order."""
    count = len(lists[0])
    for x, name in zip(lists[1:], names[1:]):
        if len(x) != count:
            raise ValueError(f"{len(x)} {name} for {count} {names[0]}")
    arrays = [array("Q") for _ in lists]
    for ts in zip(*lists):
        shape = ts[0].shape
        plain = True
        for t, name in zip(ts, names):
            if t.dtype not in DTYPES or not t.is_cuda:
                _dtype(t, name)
            if t.shape != shape:
                raise ValueError(f"{name} of shape {tuple(t.shape)} for {names[0]} of shape {tuple(shape)}")
            plain = plain and t.is_contiguous()
        if plain:
            n = ts[0].numel()
            for a, t in zip(arrays, ts):
                a.extend((t.data_ptr(), 1, n, n, DTYPES[t.dtype]))
        else:
            for a, t, (rows, cols, ld) in zip(arrays, ts, _layouts(ts, names)):
                a.extend((t.data_ptr(), rows, cols, ld, DTYPES[t.dtype]))
    return arrays


def _list_device(lists):
    """The device of every tensor (the current one)."""
    d = torch.cuda.current_device()
    for x in lists:
        for t in x:
            if t.get_device() != d:
                raise ValueError(f"a tensor is on {t.device}, the current device is cuda:{d}")
    return torch.device("cuda", d)


def grad_norm(grads, stream=None) -> torch.Tensor:
    """sqrt of the sum of squares over every tensor of `grads`, as a 0-d fp32
    device tensor (tcc_grad_norm): what clip_grad_norm clips to."""
    lib = _library()
    grads = list(grads)
    (g,) = _lists([grads], ["grads"])
    dev = _list_device([grads])
    with _on(stream):
        norm = _empty((), torch.float32, dev)
        ws = _empty(_norm_bytes, torch.uint8, dev)
    check(lib.tcc_grad_norm(g.buffer_info()[0], len(grads), norm.data_ptr(), ws.data_ptr(), _norm_bytes,
                            _stream(stream)))
    return norm


def clip_grad_norm(grads, max_norm: float, out=None, stream=None) -> torch.Tensor:
    """Scales every tensor of `grads` by min(1, max_norm / (norm + 1e-6)), in
    place or into the tensors of `out`, and returns the norm before, a 0-d
    fp32 device tensor (tcc_clip_grad_norm): torch.nn.utils.clip_grad_norm_
    without its host checks.  A tensor may have strides as long as its
    elements are rows at one distance."""
    lib = _library()
    grads = list(grads)
    if not max_norm >= 0:
        raise ValueError(f"max_norm is not negative (got {max_norm})")
    to = grads if out is None else list(out)
    for a, b in zip(grads, to):
        if a.dtype != b.dtype:
            raise ValueError(f"out must be of the gradients' types (got {b.dtype} for {a.dtype})")
    g, o = _lists([grads, to], ["grads", "out"])
    dev = _list_device([grads] if out is None else [grads, to])
    with _on(stream):
        norm = _empty((), torch.float32, dev)
        ws = _empty(_norm_bytes, torch.uint8, dev)
    check(lib.tcc_clip_grad_norm(g.buffer_info()[0], o.buffer_info()[0], len(grads), max_norm, norm.data_ptr(),
                                 ws.data_ptr(), _norm_bytes, _stream(stream)))
    return norm


def adam_step(params, grads, exp_avg, exp_avg_sq, step: torch.Tensor, lr: float = 1e-3,
              betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0,
              decoupled: bool = True, max_norm: float | None = None, stream=None) -> torch.Tensor | None:
    """One Adam step in place over lists of parameters, gradients and fp32
    moments, and step += 1 (an int64 device scalar), as torch.optim.AdamW
    (decoupled=False: Adam) computes it (tcc_adam_step).  With `max_norm` the
    gradients are clipped to it as clip_grad_norm does, as they are read:
    `grads` stay as they are, and the norm before clipping is returned."""
    lib = _library()
    lists = [list(params), list(grads), list(exp_avg), list(exp_avg_sq)]
    if step.dtype != torch.int64 or not step.is_cuda or step.numel() != 1:
        raise TypeError("step must be an int64 device scalar")
    if max_norm is not None and not max_norm >= 0:
        raise ValueError(f"max_norm is not negative (got {max_norm})")
    if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1 and eps >= 0):
        raise ValueError(f"betas must be in [0, 1) and eps not negative (got {betas} and {eps})")
    for t in (*lists[2], *lists[3]):
        if t.dtype != torch.float32:
            raise TypeError(f"moments must be float32 (got {t.dtype})")
    arrays = _lists(lists, ["params", "grads", "exp_avg", "exp_avg_sq"])
    dev = _list_device([*lists, [step]])
    a = _lib.Adam(lr, betas[0], betas[1], eps, weight_decay, -1.0 if max_norm is None else max_norm, int(decoupled))
    with _on(stream):
        norm = None if max_norm is None else _empty((), torch.float32, dev)
        ws = _empty(_norm_bytes, torch.uint8, dev)
    check(lib.tcc_adam_step(*(x.buffer_info()[0] for x in arrays), len(lists[0]), ctypes.byref(a), step.data_ptr(),
                            _ptr(norm), ws.data_ptr(), _norm_bytes, _stream(stream)))
    return norm
