"""The operators a GCN with learned node rows trains with, as they are timed.

Between them the cases are one training step around the sparse products:
rows of an embedding table looked up for the nodes of a batch, a group norm
with its activation over the node rows of each graph (channels last), their
gradients, the global gradient norm with clipping, and the Adam update that
takes the clipped gradient.  `run` computes an operator through
tcc_amd.training where `own` is true and in plain torch operations in 32 bits
where it is false; `exact` gives the definition in 64 bits.

Sizes come from the graphs this library is used on (4,096 to 2.45M nodes, 32
to 602 features, 256 hidden channels).  Inputs are seeded and made on the GPU.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


# ---------------------------------------------------------------- cases


def listed():
    return [
        # The node rows of one small sampled batch: 1,000 ids, many of them
        # hubs, into the table of a 4,096-node graph.  Launches count.
        dict(name="lookup_small", kind="lookup", V=4096, n=1000, D=32, dtype="fp32", ids="int64", skew=True, pad=False),
        # One row for every sampled neighbour of a 2.45M-node graph, the table
        # kept in 16 bits, ids as the graph stores them, absent neighbours
        # marked by a padding row.
        dict(name="lookup_large", kind="lookup", V=2_450_000, n=2_450_000, D=100, dtype="bf16", ids="int32", skew=True,
             pad=True),
        # The gradient of the small batch's rows.
        dict(name="lookup_grad_small", kind="lookup_grad", V=4096, n=1000, D=32, dtype="fp32", ids="int64", skew=True,
             pad=False),
        # The gradient of the 2.45M-node graph's table: 2.45M rows of 100, a
        # few hubs in thousands of them, a third of the table in none.
        dict(name="lookup_grad_large", kind="lookup_grad", V=2_450_000, n=2_450_000, D=100, dtype="fp32", ids="int32",
             skew=True, pad=True),
        # A small batch of small graphs, ragged, between two layers.
        dict(name="norm_small", kind="norm", segments=64, rows=2200, C=64, G=8, dtype="fp32", act="relu", grad=False),
        # The hidden layer of one full graph: every node's 256 channels.
        dict(name="norm_large", kind="norm", segments=1, rows=2_450_000, C=256, G=32, dtype="fp32", act="relu",
             grad=False),
        # The backward pass of a batch of 2,000 graphs, ragged, in 16 bits.
        dict(name="norm_grad_batch", kind="norm", segments=2000, rows=169_000, C=128, G=16, dtype="bf16", act="gelu",
             grad=True),
        # The backward pass of the full graph's hidden layer.
        dict(name="norm_grad_large", kind="norm", segments=1, rows=2_450_000, C=256, G=32, dtype="fp32", act="relu",
             grad=True),
        # The gradients of the two-layer GCN's own weights (100 -> 256 -> 2).
        dict(name="clip_small", kind="clip", V=0, F=100, hidden=256, layers=1, table="fp32", rest="fp32"),
        # A 16-bit embedding table's gradient with those of twelve layers.
        dict(name="clip_large", kind="clip", V=2_450_000, F=100, hidden=256, layers=12, table="bf16", rest="fp32"),
        # The update of the two-layer GCN's own weights.
        dict(name="adam_small", kind="adam", V=0, F=100, hidden=256, layers=1, table="fp32", rest="fp32"),
        # The update of a 2.45M x 100 table with the weights of five layers.
        dict(name="adam_large", kind="adam", V=2_450_000, F=100, hidden=256, layers=5, table="fp32", rest="fp32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["lookup", "lookup_grad", "norm", "norm_grad", "clip", "adam"])
    if kind in ("lookup", "lookup_grad"):
        D = _log_int(rng, 8, 602)
        top = min(2_450_000, 245_000_000 // D)
        return dict(kind=kind, V=_log_int(rng, 1000, top), n=_log_int(rng, 100, top), D=D,
                    dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]), ids=rng.choice(["int32", "int64"]),
                    skew=rng.random() < 0.7, pad=rng.random() < 0.4)
    if kind in ("norm", "norm_grad"):
        G = rng.choice([1, 2, 4, 7, 8, 16, 32])
        C = G * max(1, _log_int(rng, 16, 602) // G)
        rows = _log_int(rng, 500, min(2_450_000, 400_000_000 // C))
        segments = 1 if rng.random() < 0.4 else min(20_000, max(1, rows // _log_int(rng, 8, 600)))
        return dict(kind="norm", segments=segments, rows=rows, C=C, G=G, dtype=rng.choice(["fp32", "bf16", "fp16"]),
                    act=rng.choice(["none", "relu", "silu", "gelu"]), grad=kind == "norm_grad")
    F = _log_int(rng, 16, 602)
    return dict(kind=kind, V=_log_int(rng, 1000, min(2_450_000, 245_000_000 // F)), F=F,
                hidden=_log_int(rng, 16, 300), layers=rng.randint(1, 5), table=rng.choice(["fp32", "bf16", "fp16"]),
                rest=rng.choice(["fp32", "fp32", "bf16"]))


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(shape, g, dtype, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(scale).to(dtype)


def _ids(case, g):
    """Node ids: uniform, or with hubs (the k-th most frequent node in about
    k^(-2/3) of the rows), nodes numbered at random."""
    V, n = case["V"], case["n"]
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    ids = (u.pow_(3) if case["skew"] else u).mul_(V).to(torch.int64).clamp_(max=V - 1)
    if case["skew"]:
        ids = torch.randperm(V, generator=g, device="cuda")[ids]
    if case["pad"]:  # one row in ten is absent
        ids[torch.rand(n, generator=g, device="cuda") < 0.1] = 0
    return ids.to(torch.int32 if case["ids"] == "int32" else torch.int64)


def _offsets(case, g):
    """First rows of ragged segments; some are empty, some hold one row."""
    B, N = case["segments"], case["rows"]
    cuts = torch.randint(0, N + 1, (B - 1,), generator=g, device="cuda")
    ends = torch.tensor([0, N], device="cuda")
    return torch.sort(torch.cat([ends, cuts])).values.to(torch.int32)


def _shapes(case):
    F, H = case["F"], case["hidden"]
    first = [("table", (case["V"], F))] if case["V"] else []
    wide = [("rest", (F, H)), ("rest", (H,)), ("rest", (H,))]
    more = [("rest", (H, H)), ("rest", (H,)), ("rest", (H,))] * (case["layers"] - 1)
    return first + wide + more + [("rest", (H, 2))]


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    s = dict(case=case, kind=kind)
    if kind in ("lookup", "lookup_grad"):
        dt = DTYPES[case["dtype"]]
        s.update(ids=_ids(case, g), scale=math.sqrt(case["D"]), pad=0 if case["pad"] else None, V=case["V"])
        if kind == "lookup":
            s["table"] = _randn((case["V"], case["D"]), g, dt, 1.0 / math.sqrt(case["D"]))
        else:
            s["d_out"] = _randn((case["n"], case["D"]), g, dt, 1e-2)
    elif kind == "norm":
        N, C, dt = case["rows"], case["C"], DTYPES[case["dtype"]]
        level = _randn((1, C), g, torch.float32)  # aggregated rows are not centred
        spread = torch.rand((1, C), generator=g, device="cuda") * 2 + 0.2
        s["x"] = torch.randn((N, C), generator=g, device="cuda").mul_(spread).add_(level).to(dt)
        s["weight"] = torch.rand(C, generator=g, device="cuda") + 0.5
        s["bias"] = _randn((C,), g, torch.float32, 0.3)
        s["offsets"] = None if case["segments"] == 1 else _offsets(case, g)
        s.update(G=case["G"], eps=1e-5, act=case["act"])
        if case["grad"]:
            s["dy"] = _randn((N, C), g, dt, 1e-2)
            # the statistics that the forward pass left
            s["mean"], s["rstd"] = _statistics(s)
    else:
        # gradients of uneven size, as layers have them
        types = [DTYPES[case["table"] if w == "table" else case["rest"]] for w, _ in _shapes(case)]
        s["grads"] = [_randn(shape, g, t, 10.0 ** (-1 - i % 3))
                      for i, ((_, shape), t) in enumerate(zip(_shapes(case), types))]
        s["max_norm"] = 1.0
        if kind == "clip":
            s["out"] = [torch.empty_like(x) for x in s["grads"]]
        else:
            s["params"] = [_randn(x.shape, g, x.dtype, 0.1) for x in s["grads"]]
            s["exp_avg"] = [_randn(x.shape, g, torch.float32, 1e-3) for x in s["grads"]]
            s["exp_avg_sq"] = [_randn(x.shape, g, torch.float32, 1e-3).square_() for x in s["grads"]]
            s["step"] = torch.tensor(100, dtype=torch.int64, device="cuda")
            s["hyper"] = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2)
    return s


# ---------------------------------------------------------------- plain forms


def _present(s):
    """1 for the rows that count, 0 for padding."""
    return torch.ones(1, device="cuda") if s["pad"] is None else (s["ids"] != s["pad"]).unsqueeze(1).float()


def _plain_lookup(s):
    return (s["table"][s["ids"].long()].float() * (_present(s) * s["scale"])).to(s["table"].dtype)


def _plain_lookup_grad(s):
    d = s["d_out"].float() * (_present(s) * s["scale"])
    out = torch.zeros((s["V"], d.shape[1]), device="cuda")
    return out.index_add_(0, s["ids"].long(), d).to(s["d_out"].dtype)


def _segment(s):
    """The segment of every row, and each segment's number of rows."""
    count = (s["offsets"][1:] - s["offsets"][:-1]).long()
    return torch.repeat_interleave(torch.arange(count.numel(), device="cuda"), count), count


def _over_rows(v, seg, B):
    """Sums over the rows of each segment: [N x ...] -> [B x ...]."""
    if seg is None:
        return v.sum(0, keepdim=True)
    return torch.zeros((B,) + v.shape[1:], device="cuda").index_add_(0, seg, v)


def _for_rows(v, seg):
    """A value of each segment given to its rows."""
    return v if seg is None else v[seg]


def _split(s):
    """x as [N x G x C/G] in 32 bits, its rows' segments, B, and the values in each group."""
    N, C = s["x"].shape
    x = s["x"].float().view(N, s["G"], C // s["G"])
    if s["offsets"] is None:
        return x, None, 1, torch.full((1, 1), float(N * (C // s["G"])), device="cuda")
    seg, count = _segment(s)
    return x, seg, count.numel(), (count * (C // s["G"])).clamp(min=1).unsqueeze(1).float()


def _statistics(s):
    x, seg, B, size = _split(s)
    mean = _over_rows(x.sum(2), seg, B) / size
    var = _over_rows((x - _for_rows(mean, seg).unsqueeze(2)).square().sum(2), seg, B) / size
    return mean, torch.rsqrt(var + s["eps"])


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


def _normalised(s, mean, rstd):
    x, seg, B, size = _split(s)
    xh = (x - _for_rows(mean, seg).unsqueeze(2)) * _for_rows(rstd, seg).unsqueeze(2)
    w = s["weight"].view(1, x.shape[1], x.shape[2])
    z = xh * w + s["bias"].view(w.shape)
    return xh, z, w, seg, B, size


def _plain_norm(s):
    mean, rstd = _statistics(s)
    z = _normalised(s, mean, rstd)[1]
    return [_ACT[s["act"]](z).view(s["x"].shape).to(s["x"].dtype), mean, rstd]


def _plain_norm_grad(s):
    xh, z, w, seg, B, size = _normalised(s, s["mean"], s["rstd"])
    dz = s["dy"].float().view(z.shape) * _SLOPE[s["act"]](z)
    zx = dz * xh
    d_bias, d_weight = dz.sum(0).reshape(-1), zx.sum(0).reshape(-1)
    s1 = _over_rows((dz * w).sum(2), seg, B) / size
    s2 = _over_rows((zx * w).sum(2), seg, B) / size
    dx = (dz * w - _for_rows(s1, seg).unsqueeze(2) - xh * _for_rows(s2, seg).unsqueeze(2))
    dx = dx * _for_rows(s["rstd"], seg).unsqueeze(2)
    return [dx.view(s["x"].shape).to(s["x"].dtype), d_weight, d_bias]


def _plain_total(s):
    norm = torch.stack([x.float().square().sum() for x in s["grads"]]).sum().sqrt()
    return norm, torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)


def _plain_clip(s):
    norm, coef = _plain_total(s)
    return [norm] + [o.copy_(x.float() * coef) for x, o in zip(s["grads"], s["out"])]


def _plain_adam_one(p, x, m, v, coef, c1, c2, lr, betas, eps, weight_decay):
    g = x.float() * coef
    m.mul_(betas[0]).add_(g * (1 - betas[0]))
    v.mul_(betas[1]).add_(g * g * (1 - betas[1]))
    new = p.float() * (1 - lr * weight_decay) - (lr / c1) * m / (v.sqrt() / c2.sqrt() + eps)
    p.copy_(new)


def _plain_adam(s):
    norm, coef = _plain_total(s)
    h = s["hyper"]
    s["step"].add_(1)
    c1, c2 = (1 - torch.pow(torch.full((), b, dtype=torch.float64, device="cuda"), s["step"]) for b in h["betas"])
    c1, c2 = c1.float(), c2.float()
    for p, x, m, v in zip(s["params"], s["grads"], s["exp_avg"], s["exp_avg_sq"]):
        _plain_adam_one(p, x, m, v, coef, c1, c2, **h)
    return norm


# ---------------------------------------------------------------- the operators


def _own(s):
    from tcc_amd import training

    kind = s["kind"]
    if kind == "lookup":
        return training.embedding_lookup(s["table"], s["ids"], scale=s["scale"], padding_idx=s["pad"])
    if kind == "lookup_grad":
        return training.embedding_grad(s["d_out"], s["ids"], s["V"], scale=s["scale"], padding_idx=s["pad"])
    if kind == "norm" and s["case"]["grad"]:
        return training.group_norm_grad(s["dy"], s["x"], s["mean"], s["rstd"], s["G"], s["weight"], s["bias"],
                                        offsets=s["offsets"], activation=s["act"])
    if kind == "norm":
        return training.group_norm(s["x"], s["G"], s["weight"], s["bias"], offsets=s["offsets"], eps=s["eps"],
                                   activation=s["act"])
    if kind == "clip":
        return [training.clip_grad_norm(s["grads"], s["max_norm"], out=s["out"])] + s["out"]
    return training.adam_step(s["params"], s["grads"], s["exp_avg"], s["exp_avg_sq"], s["step"],
                              max_norm=s["max_norm"], **s["hyper"])


def run(s):
    kind = s["kind"]
    if own:
        out = _own(s)
    elif kind == "norm":
        out = (_plain_norm_grad if s["case"]["grad"] else _plain_norm)(s)
    else:
        out = dict(lookup=_plain_lookup, lookup_grad=_plain_lookup_grad, clip=_plain_clip, adam=_plain_adam)[kind](s)
    if kind == "adam":
        return [out, s["step"]] + s["params"] + s["exp_avg"] + s["exp_avg_sq"]
    return list(out) if isinstance(out, tuple) else out


# ---------------------------------------------------------------- work


def _distinct(case):
    """Expected distinct ids of a batch."""
    V, n = case["V"], case["n"]
    if not case["skew"]:
        return V * -math.expm1(n * math.log1p(-1.0 / V))
    edge = np.cbrt(np.arange(V + 1, dtype=np.float64) / V)
    return float(-np.expm1(n * np.log1p(-np.minimum(np.diff(edge), 1 - 1e-12))).sum())


def work(case):
    kind = case["kind"]
    if kind in ("lookup", "lookup_grad"):
        n, D, e = case["n"], case["D"], BYTES[case["dtype"]]
        ids = n * (4 if case["ids"] == "int32" else 8)
        if kind == "lookup":
            return dict(bytes=ids + (n + _distinct(case)) * D * e, flops=n * D)
        return dict(bytes=ids + (n + case["V"]) * D * e, flops=2 * n * D)
    if kind == "norm":
        elems = case["rows"] * case["C"]
        small = 8 * case["C"] + 12 * case["segments"] * case["G"]
        if case["grad"]:
            return dict(bytes=3 * elems * BYTES[case["dtype"]] + 2 * small, flops=20 * elems)
        return dict(bytes=2 * elems * BYTES[case["dtype"]] + small, flops=10 * elems)
    size = [(math.prod(shape), BYTES[case["table"] if w == "table" else case["rest"]]) for w, shape in _shapes(case)]
    count = sum(k for k, _ in size)
    if kind == "clip":
        return dict(bytes=sum(2 * k * e for k, e in size), flops=3 * count)
    return dict(bytes=sum(3 * k * e + 16 * k for k, e in size), flops=18 * count)


# ---------------------------------------------------------------- 64 bits


def _exact_lookup(s):
    out = s["table"].double().index_select(0, s["ids"].long()) * s["scale"]
    if s["pad"] is not None:
        out[s["ids"] == s["pad"]] = 0.0
    return out


def _exact_lookup_grad(s):
    # rows in the order of their ids, summed run by run on the host
    ids = s["ids"].cpu().numpy()
    order = np.argsort(ids, kind="stable")
    if s["pad"] is not None:
        order = order[ids[order] != s["pad"]]
    run = ids[order]
    out = np.zeros((s["V"], s["d_out"].shape[1]))
    if run.size:
        first = np.flatnonzero(np.concatenate([[True], run[1:] != run[:-1]]))
        d = s["d_out"].float().cpu().numpy()
        for c in range(0, d.shape[1], 32):
            out[run[first], c:c + 32] = np.add.reduceat(d[order, c:c + 32].astype(np.float64), first, axis=0)
    return torch.from_numpy(out * s["scale"])


def _exact_segments(s):
    N = s["x"].shape[0]
    at = [0, N] if s["offsets"] is None else s["offsets"].tolist()
    return list(zip(at[:-1], at[1:]))


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


def _exact_norm(s, grad):
    N, C = s["x"].shape
    G, K = s["G"], C // s["G"]
    B = len(_exact_segments(s))
    w, b = s["weight"].double().view(G, K), s["bias"].double().view(G, K)
    mean, rstd = torch.zeros((B, G), dtype=torch.float64), torch.zeros((B, G), dtype=torch.float64)
    mean, rstd = mean.cuda(), rstd.cuda()
    out = torch.empty((N, C), dtype=torch.float64, device="cuda")
    dw, db = torch.zeros_like(w), torch.zeros_like(b)
    for i, (lo, hi) in enumerate(_exact_segments(s)):
        if lo == hi:
            rstd[i] = 1.0 / math.sqrt(s["eps"])
            continue
        x = s["x"][lo:hi].double().view(hi - lo, G, K)
        if grad:
            mean[i], rstd[i] = s["mean"][i].double(), s["rstd"][i].double()
        else:
            mean[i] = x.mean(dim=(0, 2))
            rstd[i] = 1.0 / torch.sqrt((x - mean[i].view(1, G, 1)).pow(2).mean(dim=(0, 2)) + s["eps"])
        xh = (x - mean[i].view(1, G, 1)) * rstd[i].view(1, G, 1)
        y, slope = _exact_act(s["act"], torch.addcmul(b.unsqueeze(0), xh, w.unsqueeze(0)))
        if not grad:
            out[lo:hi] = y.view(hi - lo, C)
            continue
        dz = s["dy"][lo:hi].double().view(hi - lo, G, K) * slope
        db += dz.sum(0)
        dw += (dz * xh).sum(0)
        dxh = dz * w
        dx = dxh - dxh.mean(dim=(0, 2), keepdim=True) - xh * (dxh * xh).mean(dim=(0, 2), keepdim=True)
        out[lo:hi] = (dx * rstd[i].view(1, G, 1)).view(hi - lo, C)
    return [out, dw.view(-1), db.view(-1)] if grad else [out, mean, rstd]


def _exact_steps(s):
    total = math.sqrt(sum(float(torch.linalg.vector_norm(x.double())) ** 2 for x in s["grads"]))
    coef = min(1.0, s["max_norm"] / (total + 1e-6))
    if s["kind"] == "clip":
        return [torch.tensor(total, dtype=torch.float64)] + [x.double() * coef for x in s["grads"]]
    h, t = s["hyper"], int(s["step"]) + 1
    (b1, b2), new, ms, vs = h["betas"], [], [], []
    for p, x, m, v in zip(s["params"], s["grads"], s["exp_avg"], s["exp_avg_sq"]):
        g = x.double() * coef
        ms.append(b1 * m.double() + (1 - b1) * g)
        vs.append(b2 * v.double() + (1 - b2) * g.pow(2))
        mh, vh = ms[-1] / (1 - b1 ** t), vs[-1] / (1 - b2 ** t)
        new.append(p.double() - h["lr"] * (h["weight_decay"] * p.double() + mh / (torch.sqrt(vh) + h["eps"])))
    return [torch.tensor(total, dtype=torch.float64), None] + new + ms + vs


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "lookup":
        return _exact_lookup(s)
    if case["kind"] == "lookup_grad":
        return _exact_lookup_grad(s)
    if case["kind"] == "norm":
        return _exact_norm(s, case["grad"])
    return _exact_steps(s)
