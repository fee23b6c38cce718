"""The operators of deeper GCNs and of GCNs trained from a larger one, as they
are timed.

Between them the cases are what surrounds the sparse products there: a layer
norm of every node row with the residual sum before it and the activation after
it, its gradient with those of weight and bias, the top logits that a teacher
leaves for every node, the distillation loss of a student against them and its
gradient.  `run` computes an operator through tcc_amd.training where `own` is
true and in plain torch operations in 32 bits where it is false; `exact` gives
the definition in 64 bits.

Node and channel counts come from the graphs this library is used on (4,096 to
2.45M nodes, 32 to 602 features, 256 hidden channels); class counts are generic:
the tens to hundreds of a node classifier, and the tens of thousands of a model
that predicts a node.  Inputs are seeded and made on the GPU.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-5
WEIGHTED = 0.9  # share of the rows that a weighted loss takes


# ---------------------------------------------------------------- cases


def listed():
    return [
        # The rows of one small sampled batch between two layers.  Launches count.
        dict(name="norm_small", kind="norm", rows=1000, C=64, dtype="fp32", act="relu", residual=False, grad=False),
        # Every node's 256 channels before a residual block: the block before
        # it added to the stream, the norm of that, relu.
        dict(name="norm_large", kind="norm", rows=2_450_000, C=256, dtype="fp32", act="relu", residual=True, grad=False),
        # Wide rows in 16 bits, the last norm before a projection.
        dict(name="norm_wide", kind="norm", rows=16_384, C=4096, dtype="bf16", act="none", residual=True, grad=False),
        # The backward pass of a batch of graphs with an odd number of channels.
        dict(name="norm_grad_batch", kind="norm", rows=169_000, C=301, dtype="bf16", act="gelu", residual=False,
             grad=True),
        # The backward pass of the full graph's residual block.
        dict(name="norm_grad_large", kind="norm", rows=2_450_000, C=256, dtype="fp32", act="relu", residual=True,
             grad=True),
        # A teacher's answers for a small batch.
        dict(name="top_small", kind="top", rows=1000, C=47, K=4, dtype="fp32", T=1.0),
        # A teacher's answers for every node of a large graph.
        dict(name="top_nodes", kind="top", rows=2_450_000, C=100, K=8, dtype="fp32", T=2.0),
        # A teacher that predicts one of 50,000 nodes.
        dict(name="top_wide", kind="top", rows=4096, C=50_000, K=32, dtype="bf16", T=2.0),
        # The student's loss on a small batch.
        dict(name="distill_small", kind="distill", rows=1000, C=47, K=4, dtype="fp32", T=1.0, rest=False, weighted=True,
             grad=False),
        # The student's loss over 50,000 classes, with the mass that the top
        # ones leave.
        dict(name="distill_wide", kind="distill", rows=4096, C=50_000, K=32, dtype="bf16", T=2.0, rest=True,
             weighted=False, grad=False),
        # The gradient for every node of a large graph, a tenth of them without
        # weight.
        dict(name="distill_grad_nodes", kind="distill", rows=2_450_000, C=100, K=8, dtype="fp32", T=2.0, rest=False,
             weighted=True, grad=True),
        # The gradient over an odd number of classes, rows of every alignment.
        dict(name="distill_grad_wide", kind="distill", rows=4096, C=50_001, K=32, dtype="bf16", T=2.0, rest=True,
             weighted=False, grad=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "top", "distill", "distill_grad"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if kind in ("norm", "norm_grad"):
        C = _log_int(rng, 16, 4096)
        return dict(kind="norm", rows=_log_int(rng, 500, min(2_450_000, 400_000_000 // C)), C=C, dtype=dtype,
                    act=rng.choice(["none", "relu", "silu", "gelu"]), residual=rng.random() < 0.5,
                    grad=kind == "norm_grad")
    C = _log_int(rng, 2, 300) if rng.random() < 0.5 else _log_int(rng, 300, 60_000)
    case = dict(rows=_log_int(rng, min(500, 100_000_000 // C), min(2_450_000, 200_000_000 // C)), C=C,
                K=_log_int(rng, 1, min(64, C - 1)), dtype=dtype, T=rng.choice([1.0, 2.0, 4.0]))
    if kind == "top":
        return dict(kind="top", **case)
    return dict(kind="distill", **case, rest=rng.random() < 0.5, weighted=rng.random() < 0.5,
                grad=kind == "distill_grad")


# ---------------------------------------------------------------- inputs


def _randn(shape, g, dtype=torch.float32, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(scale).to(dtype)


def _logits(case, g, like=None):
    """Logits of a trained classifier: a spread of 3 around each class's own
    level; a student's follow its teacher's (`like`)."""
    z = _randn((case["rows"], case["C"]), g, scale=3.0 if like is None else 1.5)
    if like is not None:
        return z.add_(like, alpha=0.8).to(DTYPES[case["dtype"]])
    return z.add_(_randn((1, case["C"]), g)).to(DTYPES[case["dtype"]])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case=case, kind=case["kind"])
    if case["kind"] == "norm":
        N, C, dt = case["rows"], case["C"], DTYPES[case["dtype"]]
        level = _randn((1, C), g)  # aggregated rows are not centred
        spread = torch.rand((1, C), generator=g, device="cuda") * 2 + 0.2
        s["x"] = torch.randn((N, C), generator=g, device="cuda").mul_(spread).add_(level).to(dt)
        s["weight"] = torch.rand(C, generator=g, device="cuda") + 0.5
        s["bias"] = _randn((C,), g, scale=0.3)
        s["act"] = case["act"]
        if case["grad"]:
            s["dy"] = _randn((N, C), g, dt, 1e-2)
            s["d_sum"] = _randn((N, C), g, dt, 1e-2) if case["residual"] else None
            # the statistics that the forward pass left
            s["mean"], s["rstd"] = _statistics(s["x"].float())
        else:
            s["residual"] = _randn((N, C), g, dt) if case["residual"] else None
        return s
    s["T"], s["K"] = case["T"], case["K"]
    z = _logits(case, g)
    if case["kind"] == "top":
        s["logits"] = z
        return s
    # the teacher's answers, as they were stored, and the student's logits
    top = torch.topk(z.float(), case["K"], dim=1)
    s["values"], s["ids"] = top.values.to(z.dtype), top.indices.to(torch.int32)
    s["rest"] = None
    if case["rest"]:
        left = z.float().scatter_(1, top.indices, float("-inf"))
        m, e = _shares(left, case["T"])
        s["rest"] = (m + case["T"] * torch.log(e)).squeeze(1)
        del left
    s["logits"] = _logits(case, g, like=z)
    s["weight"] = None
    if case["weighted"]:
        w = torch.rand(case["rows"], generator=g, device="cuda") + 0.5
        s["weight"] = w.mul_(torch.rand(case["rows"], generator=g, device="cuda") < WEIGHTED)
    if case["grad"]:
        s["d_loss"] = torch.ones((), device="cuda")
        # what the forward pass left
        s["stats"] = _stats(s)
        s["total"] = None if s["weight"] is None else s["weight"].sum()
    return s


# ---------------------------------------------------------------- plain forms


def _statistics(h):
    mean = h.sum(1) / h.shape[1]
    var = (h - mean.unsqueeze(1)).square().sum(1) / h.shape[1]
    return mean, torch.rsqrt(var + EPS)


def _cdf(z):
    return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))


_ACT = {
    "none": lambda z: z,
    "relu": lambda z: torch.where(z > 0, z, z * 0),
    "silu": lambda z: z / (1.0 + torch.exp(-z)),
    "gelu": lambda z: z * _cdf(z),
}


def _silu_slope(z):
    p = 1.0 / (1.0 + torch.exp(-z))
    return p * (1.0 + z * (1.0 - p))


_SLOPE = {
    "none": lambda z: torch.ones_like(z),
    "relu": lambda z: (z > 0).float(),
    "silu": _silu_slope,
    "gelu": lambda z: _cdf(z) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi)),
}


def _plain_norm(s):
    h = s["x"]
    if s["residual"] is not None:
        h = (h.float() + s["residual"].float()).to(h.dtype)
    mean, rstd = _statistics(h.float())
    z = (h.float() - mean.unsqueeze(1)) * rstd.unsqueeze(1) * s["weight"] + s["bias"]
    y = _ACT[s["act"]](z).to(h.dtype)
    return [y, mean, rstd] if s["residual"] is None else [y, h, mean, rstd]


def _plain_norm_grad(s):
    C = s["x"].shape[1]
    rstd = s["rstd"].unsqueeze(1)
    xh = (s["x"].float() - s["mean"].unsqueeze(1)) * rstd
    dz = s["dy"].float() * _SLOPE[s["act"]](xh * s["weight"] + s["bias"])
    # long sums of either sign
    d_bias = dz.sum(0, dtype=torch.float64).float()
    d_weight = (dz * xh).sum(0, dtype=torch.float64).float()
    a = dz * s["weight"]
    s1, s2 = a.sum(1, keepdim=True) / C, (a * xh).sum(1, keepdim=True) / C
    dx = (a - s1 - xh * s2) * rstd
    if s["d_sum"] is not None:
        dx = dx + s["d_sum"].float()
    return [dx.to(s["x"].dtype), d_weight, d_bias]


def _shares(z, T):
    """The maximum of each row and the sum of exp((z - maximum) / T)."""
    m = z.max(1, keepdim=True).values
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    return m, torch.exp((z - m) / T).sum(1, keepdim=True)


def _plain_top(s):
    z = s["logits"].float()
    order = torch.sort(z, dim=1, descending=True, stable=True)  # ties: lowest index first
    ids = order.indices[:, :s["K"]].contiguous()
    values = order.values[:, :s["K"]].to(s["logits"].dtype)
    del order
    m, e = _shares(z.scatter(1, ids, float("-inf")), s["T"])
    return [values, ids.to(torch.int32), (m + s["T"] * torch.log(e)).squeeze(1)]


def _others(s):
    """The logits of the classes that are none of a row's ids; -inf at those that are."""
    return s["logits"].float().scatter(1, s["ids"].long(), float("-inf"))


def _stats(s):
    """[n x 4]: maximum and sum of the shares of all classes, and of the
    classes that are none of the ids (0 and 0 where no rest is given); zeros
    for rows without weight."""
    m, e = _shares(s["logits"].float(), s["T"])
    if s["rest"] is None:
        mr, er = torch.zeros_like(m), torch.zeros_like(e)
    else:
        mr, er = _shares(_others(s), s["T"])
    stats = torch.cat([m, e, mr, er], 1)
    return stats if s["weight"] is None else stats * (s["weight"] != 0).unsqueeze(1)


def _targets(s):
    """The teacher's probabilities of the ids and of the rest, and their logarithms."""
    t = s["values"].float()
    if s["rest"] is not None:
        t = torch.cat([t, s["rest"].unsqueeze(1)], 1)
    m, e = _shares(t, s["T"])
    log_p = (t - m) / s["T"] - torch.log(e)
    return torch.exp(log_p), log_p


def _plain_loss(s):
    stats = _stats(s)
    m, e, mr, er = stats.split(1, 1)
    p, log_p = _targets(s)
    log_q = (s["logits"].float().gather(1, s["ids"].long()) - m) / s["T"] - torch.log(e)
    if s["rest"] is not None:
        log_q = torch.cat([log_q, (mr - m) / s["T"] + torch.log(er) - torch.log(e)], 1)
    rows = (p * (log_p - log_q)).sum(1) * (s["T"] * s["T"])
    if s["weight"] is None:
        loss = rows.sum(dtype=torch.float64) / rows.numel()
    else:
        rows = torch.where(s["weight"] == 0, torch.zeros_like(rows), rows * s["weight"])
        loss = rows.sum(dtype=torch.float64) / s["weight"].sum(dtype=torch.float64)
    return [loss.float(), stats]


def _plain_loss_grad(s):
    T = s["T"]
    m, e, mr, er = s["stats"].split(1, 1)
    p, _ = _targets(s)
    z, ids = s["logits"].float(), s["ids"].long()
    at_ids = torch.exp((z.gather(1, ids) - m) / T) / e - p[:, :s["K"]]
    if s["rest"] is None:
        d = torch.exp((z - m) / T) / e
    else:  # the rest's mass, off by what the teacher gave it, spread as the student spreads it
        left = torch.exp((mr - m) / T) * er / e - p[:, s["K"]:]
        d = torch.exp(torch.clamp((z - mr) / T, max=0.0)) / er * left
    d = d.scatter(1, ids, at_ids)
    if s["weight"] is not None:
        d = torch.where((s["weight"] == 0).unsqueeze(1), torch.zeros_like(d), d)
    if s["weight"] is None:
        scale = T / z.shape[0]
    else:
        scale = (s["weight"] * (T / s["total"])).unsqueeze(1)
    return (d * (s["d_loss"] * scale)).to(s["logits"].dtype)


# ---------------------------------------------------------------- the operators


def _own(s):
    from tcc_amd import training

    case = s["case"]
    if s["kind"] == "norm" and case["grad"]:
        return list(training.layer_norm_grad(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"], s["bias"],
                                             d_sum=s["d_sum"], activation=s["act"]))
    if s["kind"] == "norm":
        y, h, mean, rstd = training.layer_norm(s["x"], s["weight"], s["bias"], residual=s["residual"], eps=EPS,
                                               activation=s["act"])
        return [y, mean, rstd] if s["residual"] is None else [y, h, mean, rstd]
    if s["kind"] == "top":
        return list(training.top_logits(s["logits"], s["K"], temperature=s["T"]))
    if case["grad"]:
        return training.distill_grad(s["d_loss"], s["logits"], s["values"], s["ids"], s["stats"], rest=s["rest"],
                                     temperature=s["T"], weight=s["weight"], total=s["total"])
    loss, stats, _ = training.distill_loss(s["logits"], s["values"], s["ids"], rest=s["rest"], temperature=s["T"],
                                           weight=s["weight"])
    return [loss, stats]


def run(s):
    if own:
        return _own(s)
    if s["kind"] == "norm":
        return (_plain_norm_grad if s["case"]["grad"] else _plain_norm)(s)
    if s["kind"] == "top":
        return _plain_top(s)
    return (_plain_loss_grad if s["case"]["grad"] else _plain_loss)(s)


# ---------------------------------------------------------------- work


def work(case):
    elems, e = case["rows"] * case["C"], BYTES[case["dtype"]]
    if case["kind"] == "norm":
        small = 8 * case["rows"] + 8 * case["C"]
        tensors = (3 if case["grad"] else 2) + (1 if case["residual"] and case["grad"] else 0)
        tensors += 2 if case["residual"] and not case["grad"] else 0
        return dict(bytes=tensors * elems * e + small + (8 * case["C"] if case["grad"] else 0),
                    flops=(20 if case["grad"] else 10) * elems)
    top = case["rows"] * case["K"] * (e + 4)
    if case["kind"] == "top":
        return dict(bytes=elems * e + top + 4 * case["rows"], flops=4 * elems)
    part = WEIGHTED if case["weighted"] else 1.0
    rows = case["rows"] * ((4 if case["rest"] else 0) + (4 if case["weighted"] else 0))
    if not case["grad"]:
        return dict(bytes=part * (elems * e + top) + rows + 16 * case["rows"] + 4, flops=part * 5 * elems)
    # the rows without weight are written, not read
    return dict(bytes=(part + 1) * elems * e + part * (top + 16 * case["rows"]) + rows, flops=part * 6 * elems)


# ---------------------------------------------------------------- 64 bits


def _exact_act(name, z):
    """The activation and its derivative at z."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    p = torch.special.ndtr(z)
    return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def _pieces(case):
    """Row ranges of about 2^26 elements."""
    step = max(1, (1 << 26) // case["C"])
    return [(lo, min(lo + step, case["rows"])) for lo in range(0, case["rows"], step)]


def _exact_norm(s):
    case = s["case"]
    w, b = s["weight"].double(), s["bias"].double()
    out, sums, means, rstds = [], [], [], []
    for lo, hi in _pieces(case):
        h = s["x"][lo:hi]
        if s["residual"] is not None:
            h = (h.double() + s["residual"][lo:hi].double()).to(h.dtype)
            sums.append(h.double())
        h = h.double()
        var, mean = torch.var_mean(h, dim=1, correction=0)
        rstd = 1.0 / torch.sqrt(var + EPS)
        out.append(_exact_act(case["act"], torch.addcmul(b, (h - mean[:, None]) * rstd[:, None], w))[0])
        means.append(mean)
        rstds.append(rstd)
    y, mean, rstd = torch.cat(out), torch.cat(means), torch.cat(rstds)
    return [y, mean, rstd] if not sums else [y, torch.cat(sums), mean, rstd]


def _exact_norm_grad(s):
    case = s["case"]
    w, b = s["weight"].double(), s["bias"].double()
    dw, db, out = torch.zeros_like(w), torch.zeros_like(b), []
    for lo, hi in _pieces(case):
        rstd = s["rstd"][lo:hi, None].double()
        xh = (s["x"][lo:hi].double() - s["mean"][lo:hi, None].double()) * rstd
        slope = _exact_act(case["act"], torch.addcmul(b, xh, w))[1]
        if case["act"] == "relu":
            # relu masks what the forward pass masked, and that had z in 32
            # bits, rounded after each operation
            z = (s["x"][lo:hi].float() - s["mean"][lo:hi, None]).mul_(s["rstd"][lo:hi, None])
            slope = (z.mul_(s["weight"]).add_(s["bias"]) > 0).double()
        dz = s["dy"][lo:hi].double() * slope
        db += dz.sum(0)
        dw += (dz * xh).sum(0)
        dxh = dz * w
        dx = rstd * (dxh - dxh.mean(1, keepdim=True) - xh * (dxh * xh).mean(1, keepdim=True))
        out.append(dx if s["d_sum"] is None else dx + s["d_sum"][lo:hi].double())
    return [torch.cat(out), dw, db]


def _exact_top(s):
    """One maximum after the other, each taken out at its lowest index."""
    case, parts = s["case"], []
    for lo, hi in _pieces(case):
        z = s["logits"][lo:hi].double()
        columns = torch.arange(case["C"], device="cuda")
        values, ids = [], []
        for _ in range(case["K"]):
            top = torch.amax(z, dim=1)
            at = torch.where(z == top[:, None], columns, case["C"]).amin(dim=1)
            z[torch.arange(hi - lo, device="cuda"), at] = -math.inf
            values.append(top)
            ids.append(at)
        rest = torch.logsumexp(z / case["T"], dim=1) * case["T"]
        parts.append((torch.stack(values, 1), torch.stack(ids, 1).to(torch.int32), rest))
    return [torch.cat(p) for p in zip(*parts)]


def _exact_distill(s):
    case, T = s["case"], s["case"]["T"]
    n, C = s["logits"].shape
    weight = torch.ones(n, dtype=torch.float64, device="cuda") if s["weight"] is None else s["weight"].double()
    share = weight / weight.sum()
    total, out, stats = 0.0, [], []
    for lo, hi in _pieces(case):
        log_q = torch.log_softmax(s["logits"][lo:hi].double() / T, dim=1)
        counts = (weight[lo:hi, None] != 0).double()
        ids, t = s["ids"][lo:hi].long(), s["values"][lo:hi].double()
        picked = torch.zeros((hi - lo, C), dtype=torch.bool, device="cuda").scatter_(1, ids, True)
        at = log_q.gather(1, ids)
        if s["rest"] is not None:
            t = torch.cat([t, s["rest"][lo:hi, None].double()], 1)
            left = torch.logsumexp(log_q.masked_fill(picked, -math.inf), dim=1, keepdim=True)
            at = torch.cat([at, left], 1)
        log_p = torch.log_softmax(t / T, dim=1)
        p = log_p.exp()
        if not case["grad"]:
            total = total + (T * T * share[lo:hi] * (p * (log_p - at)).sum(1)).sum()
            z = s["logits"][lo:hi].double()
            both = [z] if s["rest"] is None else [z, z.masked_fill(picked, -math.inf)]
            tops = [torch.amax(v, dim=1, keepdim=True) for v in both]
            sums = [torch.exp(torch.logsumexp(v / T, dim=1, keepdim=True) - top / T) for v, top in zip(both, tops)]
            some = torch.cat([v for pair in zip(tops, sums) for v in pair], 1) * counts
            stats.append(torch.nn.functional.pad(some, (0, 4 - some.shape[1])))
            continue
        aim = torch.zeros_like(log_q)
        if s["rest"] is not None:
            aim = ((log_q - left).exp() * p[:, -1:]).masked_fill(picked, 0.0)
        aim.scatter_(1, ids, p[:, :case["K"]])
        out.append((log_q.exp() - aim) * (T * share[lo:hi, None]))
    return torch.cat(out) if case["grad"] else [total, torch.cat(stats)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        return (_exact_norm_grad if case["grad"] else _exact_norm)(s)
    return _exact_top(s) if case["kind"] == "top" else _exact_distill(s)
