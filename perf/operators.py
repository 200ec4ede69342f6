"""Workloads of the per-graph operators: group norm with an activation, activation checkpoints in 8 bits, and attention
among the nodes of one graph.

Every case is one pass of a user's program over a batch of graphs.  ``run`` computes it in plain torch operations, or -
where ``own`` is set - with the operators of ``hgvae_amd``; ``exact`` computes the same outputs in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

# The eight molecules of the bundled data set (nodes per graph).
BUNDLED = "454,2627,4697,11213,11455,11940,13239,15200"
BLOCK = 32                     # columns that share one scale of an 8-bit checkpoint


# --------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------
def listed():
    return [
        # a batch of 32 chignolin frames, the loops' own batch size: a level of the 138-wide model, bound by latency
        {"name": "norm_chignolin_train", "op": "norm", "graphs": 32, "low": 138, "high": 138, "shape": 0, "channels": 138,
         "groups": 6, "act": "silu", "train": True, "keep8": False},
        # evaluation of the 256-wide model on one graph of each bundled size: ragged, forward only
        {"name": "norm_bundled_forward", "op": "norm", "sizes": BUNDLED, "channels": 256, "groups": 32, "act": "gelu",
         "train": False, "keep8": False},
        # the benchmark's own batch (256 protein-like graphs) through one 138-wide level: the largest matrix
        {"name": "norm_protein256_train", "op": "norm", "graphs": 256, "low": 4500, "high": 5500, "shape": 1, "channels": 138,
         "groups": 6, "act": "silu", "train": True, "keep8": False},
        # a level of the 256-wide model that keeps its input in 8 bits for the backward pass
        {"name": "norm_protein32_keep8", "op": "norm", "graphs": 32, "low": 4500, "high": 5500, "shape": 2, "channels": 256,
         "groups": 8, "act": "silu", "train": True, "keep8": True},
        # an activation matrix put into 8 bits and taken out again
        {"name": "pack_protein32", "op": "pack", "rows": 160001, "columns": 256},
        # a projection of the 138-wide model at the loops' own batch size
        {"name": "linear8_chignolin_train", "op": "linear8", "rows": 4416, "columns": 138, "outputs": 138},
        # the attention model's first projection (105 features to 256 columns) over the bundled graphs
        {"name": "linear8_bundled_train", "op": "linear8", "rows": 70825, "columns": 105, "outputs": 256},
        # a hidden projection over the benchmark's batch: the largest matrix
        {"name": "linear8_protein256_train", "op": "linear8", "rows": 1283529, "columns": 138, "outputs": 138},
        # evaluation on 32 chignolin frames: 256 channels as four heads, bound by latency
        {"name": "attention_chignolin_forward", "op": "attention", "graphs": 32, "low": 138, "high": 138, "shape": 3, "heads": 4,
         "kv_heads": 4, "width": 64, "train": False, "masked": False},
        # one graph of each bundled size, 138 channels as six heads of 23 that share two key heads; a mask takes some nodes
        # out as keys and leaves the first graph without any
        {"name": "attention_bundled_train", "op": "attention", "sizes": BUNDLED, "heads": 6, "kv_heads": 2, "width": 23,
         "train": True, "masked": True},
        # the longest bundled molecule, four frames, evaluation
        {"name": "attention_long_forward", "op": "attention", "sizes": "15200,15200,15200,15200", "heads": 4, "kv_heads": 4,
         "width": 64, "train": False, "masked": False},
        # a step on 32 protein-like graphs, 256 channels as four heads
        {"name": "attention_protein32_train", "op": "attention", "graphs": 32, "low": 4500, "high": 5500, "shape": 4, "heads": 4,
         "kv_heads": 4, "width": 64, "train": True, "masked": False},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    limits = {}
    for c in listed():
        w = work(c)
        b, f = limits.get(c["op"], (0, 0))
        limits[c["op"]] = (max(b, w["bytes"]), max(f, w["flops"]))
    while True:
        op = rng.choice(["norm", "norm", "pack", "linear8", "linear8", "attention", "attention"])
        if op in ("norm", "attention"):
            low = _log_int(rng, 1, 15200)
            case = {"op": op, "graphs": _log_int(rng, 1, 300), "low": low, "high": _log_int(rng, low, min(4 * low, 15200)),
                    "shape": rng.randrange(10 ** 6)}
        if op == "norm":
            per = _log_int(rng, 1, 64)
            case.update(channels=per * rng.randint(1, max(1, 320 // per)), act=rng.choice(["silu", "gelu", "none"]),
                        train=rng.random() < 0.7)
            case.update(groups=case["channels"] // per, keep8=case["train"] and rng.random() < 0.4)
        elif op == "attention":
            kv = rng.randint(1, 4)
            case.update(kv_heads=kv, heads=kv * rng.randint(1, 3), width=_log_int(rng, 4, 128), train=rng.random() < 0.6,
                        masked=rng.random() < 0.5)
        elif op == "pack":
            case = {"op": op, "rows": _log_int(rng, 1, 400000), "columns": _log_int(rng, 1, 320)}
        else:
            case = {"op": op, "rows": _log_int(rng, 1, 1300000), "columns": _log_int(rng, 4, 288), "outputs": _log_int(rng, 4, 288)}
        w = work(case)
        if w["bytes"] <= limits[op][0] and w["flops"] <= limits[op][1]:
            return case


def _sizes(case):
    if "sizes" in case:
        return [int(s) for s in case["sizes"].split(",")]
    r = random.Random(case["shape"])
    return [r.randint(case["low"], case["high"]) for _ in range(case["graphs"])]


def _rows(case):
    return case["rows"] if "rows" in case else sum(_sizes(case))


def work(case):
    """Bytes and operations that one pass cannot do without: inputs read once, outputs written once."""
    n, op = _rows(case), case["op"]
    if op == "norm":
        c = case["channels"]
        return {"bytes": (16 if case["train"] else 8) * n * c + (16 if case["train"] else 8) * c,
                "flops": (30 if case["train"] else 10) * n * c}
    if op == "pack":
        return {"bytes": 8 * n * case["columns"], "flops": 4 * n * case["columns"]}
    if op == "linear8":
        k, m = case["columns"], case["outputs"]
        return {"bytes": 4 * (2 * n * k + 2 * n * m + 2 * k * m + 2 * m), "flops": 6 * n * k * m}
    h, hk, d = case["heads"], case["kv_heads"], case["width"]
    pairs = sum(s * s for s in _sizes(case))
    q, kv = 4 * n * h * d, 4 * n * hk * d
    return {"bytes": (4 * q + 4 * kv if case["train"] else 2 * q + 2 * kv) + (n if case["masked"] else 0),
            "flops": (14 if case["train"] else 4) * pairs * h * d}


# --------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------
def _chunks(sizes, per_pair):
    """Runs of graphs that the plain form pads to one length: no more than twice the pairs, no more than 2^28 of them."""
    runs, cur = [], []
    for g, s in enumerate(sizes):
        if s == 0:
            continue
        trial = [sizes[i] for i in cur] + [s]
        dense = len(trial) * max(trial) ** 2
        if cur and (dense > 2 * sum(t * t for t in trial) or dense * per_pair > 2 ** 28):
            runs.append(cur)
            cur = []
        cur.append(g)
    return runs + [cur] if cur else runs


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device=dev) * scale

    op, n = case["op"], _rows(case)
    st = {"case": case}
    if op in ("norm", "attention"):
        sizes = _sizes(case)
        st["batch"] = torch.repeat_interleave(torch.arange(len(sizes), device=dev), torch.tensor(sizes, device=dev))
        if own:
            from hgvae_amd import Segments
            st["segments"] = Segments.from_sizes(sizes, dev)
    if op == "norm":
        c = case["channels"]
        # pre-activations of a projection: every column with an offset and a spread of its own
        st["x"] = normal(n, c).mul_(torch.rand(c, generator=gen, device=dev) + 0.5).add_(normal(c, scale=0.5))
        st["weight"], st["bias"] = torch.rand(c, generator=gen, device=dev) + 0.5, normal(c, scale=0.3)
        if case["train"]:
            st["g"] = normal(n, c, scale=1e-2)
    elif op == "pack":
        st["x"] = normal(n, case["columns"]) * (torch.rand(case["columns"], generator=gen, device=dev) + 0.1)
    elif op == "linear8":
        k, m = case["columns"], case["outputs"]
        # activations behind a smooth rectifier: mostly small, some large
        st["x"] = torch.nn.functional.silu(normal(n, k))
        st["weight"], st["bias"] = normal(m, k, scale=1.0 / math.sqrt(k)), normal(m, scale=0.1)
        st["g"] = normal(n, m, scale=1e-2)
    else:
        h, hk, d = case["heads"], case["kv_heads"], case["width"]
        st["q"], st["k"], st["v"] = normal(n, h, d, scale=1.5), normal(n, hk, d), normal(n, hk, d)
        if case["train"]:
            st["g"] = normal(n, h, d, scale=1e-2)
        st["mask"] = None
        if case["masked"]:
            st["mask"] = torch.rand(n, generator=gen, device=dev) < 0.85
            st["mask"][:sizes[0]] = False
        if not own:
            starts = [0]
            for s in sizes:
                starts.append(starts[-1] + s)
            st["runs"] = []
            for run in _chunks(sizes, h):
                top = max(sizes[g] for g in run)
                first = torch.tensor([starts[g] for g in run], device=dev).unsqueeze(1)
                size = torch.tensor([sizes[g] for g in run], device=dev).unsqueeze(1)
                pos = torch.arange(top, device=dev).unsqueeze(0)
                there = pos < size
                st["runs"].append((torch.where(there, first + pos, 0), there))
    return st


# --------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "pack": _own_pack, "linear8": _own_linear8, "attention": _own_attention}[op](state)
    return {"norm": _plain_norm, "pack": _plain_pack, "linear8": _plain_linear8, "attention": _plain_attention}[op](state)


def _own_norm(st):
    from hgvae_amd import functional as Fn
    case = st["case"]
    if not case["train"]:
        with torch.no_grad():
            return Fn.group_norm_act(st["x"], st["segments"], case["groups"], st["weight"], st["bias"], act=case["act"])
    x, w, b = (st[n].detach().requires_grad_() for n in ("x", "weight", "bias"))
    out = Fn.group_norm_act(x, st["segments"], case["groups"], w, b, act=case["act"], keep8=case["keep8"])
    return (out.detach(), *torch.autograd.grad(out, (x, w, b), st["g"]))


def _own_pack(st):
    from hgvae_amd import functional as Fn
    return Fn.pack8(st["x"]).unpack()


def _own_linear8(st):
    from hgvae_amd import functional as Fn
    x, w, b = (st[n].detach().requires_grad_() for n in ("x", "weight", "bias"))
    y = Fn.linear8(x, w, b)
    return (y.detach(), *torch.autograd.grad(y, (x, w, b), st["g"]))


def _own_attention(st):
    from hgvae_amd import functional as Fn
    if not st["case"]["train"]:
        with torch.no_grad():
            return Fn.graph_attention(st["q"], st["k"], st["v"], st["segments"], mask=st["mask"])
    q, k, v = (st[n].detach().requires_grad_() for n in "qkv")
    out = Fn.graph_attention(q, k, v, st["segments"], mask=st["mask"])
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), st["g"]))


# ---- plain forms ----
def _plain_values8(x):
    """x as 8-bit integers times a power of two per row and block of columns, and back."""
    n, c = x.shape
    nb = (c + BLOCK - 1) // BLOCK
    p = torch.zeros(n, nb * BLOCK, dtype=x.dtype, device=x.device)
    p[:, :c] = x
    p = p.view(n, nb, BLOCK)
    amax = p.abs().amax(-1, keepdim=True)
    e = torch.frexp(amax)[1] - 7
    e = torch.where(amax >= torch.ldexp(torch.full_like(amax, 127.5), e), e + 1, e).clamp(min=-126)
    q = torch.round(torch.ldexp(p, -e))
    return torch.ldexp(q, e).view(n, nb * BLOCK)[:, :c].contiguous()


def _plain_pack(st):
    return _plain_values8(st["x"])


def _act(z, kind):
    """(activation, its derivative)"""
    if kind == "none":
        return z, torch.ones_like(z)
    if kind == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_norm(st):
    case, x, batch = st["case"], st["x"], st["batch"]
    n, c = x.shape
    grp, b = case["groups"], len(_sizes(case))
    per = c // grp
    rows = torch.bincount(batch, minlength=b)
    ends = torch.cumsum(rows, 0)

    def group_mean(t):                                  # t [n, groups, per]: long sums, as differences of prefix sums in 64 bits
        s = torch.zeros(grp, n + 1, dtype=torch.float64, device=x.device)
        torch.cumsum(t.sum(-1, dtype=torch.float64).t().contiguous(), 1, out=s[:, 1:])
        return (s[:, ends] - s[:, ends - rows]).t() / (rows.clamp(min=1) * per).double().unsqueeze(1)

    def rows_of(t):                                     # [graphs, groups] -> [n, groups, 1]
        return t.float()[batch].unsqueeze(-1)

    xg = x.view(n, grp, per)
    mean = rows_of(group_mean(xg))
    d = xg - mean
    rstd = rows_of(torch.rsqrt(group_mean(d * d) + 1e-5))
    w, bias = st["weight"].view(1, grp, per), st["bias"].view(1, grp, per)
    out = _act(d * rstd * w + bias, case["act"])[0].reshape(n, c)
    if not case["train"]:
        return out
    if case["keep8"]:
        d = _plain_values8(x).view(n, grp, per) - mean
    xh = d * rstd
    dz = st["g"].view(n, grp, per) * _act(xh * w + bias, case["act"])[1]
    gw, gb = (dz * xh).sum(0, dtype=torch.float64).reshape(c).float(), dz.sum(0, dtype=torch.float64).reshape(c).float()
    dxh = dz * w
    gx = rstd * (dxh - rows_of(group_mean(dxh)) - xh * rows_of(group_mean(dxh * xh)))
    return out, gx.reshape(n, c), gw, gb


def _plain_linear8(st):
    x, w, g = st["x"], st["weight"], st["g"]
    y = torch.matmul(x, w.t()) + st["bias"]
    v = _plain_values8(x)
    gx = torch.matmul(g, w)
    gw = torch.zeros(w.shape, dtype=torch.float64, device=w.device)       # long sums: blocks of rows, joined in 64 bits
    for i in range(0, x.size(0), 65536):
        gw += torch.matmul(g[i:i + 65536].t(), v[i:i + 65536])
    return y, gx, gw.float(), g.sum(0, dtype=torch.float64).float()


def _plain_attention(st):
    case = st["case"]
    h, hk, d = case["heads"], case["kv_heads"], case["width"]
    r, scale = h // hk, 1.0 / math.sqrt(d)
    outs = [torch.zeros_like(st["q"])]
    if case["train"]:
        outs += [torch.zeros_like(st["q"]), torch.zeros_like(st["k"]), torch.zeros_like(st["v"])]
    for index, there in st["runs"]:
        b, top = index.shape

        def heads(t, per):                              # [n, heads, d] -> [b, hk, per * top, d], zero where there is no row
            t = torch.where(there[:, :, None, None], t[index], 0.0)
            return t.view(b, top, hk, per, d).permute(0, 2, 3, 1, 4).reshape(b, hk, per * top, d).contiguous()

        def put(dst, t, per):
            t = t.view(b, hk, per, top, d).permute(0, 3, 1, 2, 4).reshape(b, top, hk * per, d)
            dst[index[there]] = t[there]

        keys = there if st["mask"] is None else there & st["mask"][index]
        keys = keys[:, None, None, :]
        q, k, v = heads(st["q"], r), heads(st["k"], 1), heads(st["v"], 1)
        kt, vt = k.transpose(2, 3).contiguous(), v.transpose(2, 3).contiguous()
        s = torch.matmul(q, kt).mul_(scale).masked_fill_(~keys, -float("inf"))
        top_s = s.amax(-1, keepdim=True)
        p = s.sub_(torch.where(top_s.isinf(), 0.0, top_s)).exp_()
        p /= p.sum(-1, keepdim=True).clamp(min=1e-30)
        o = torch.matmul(p, v)
        put(outs[0], o, r)
        if case["train"]:
            do = heads(st["g"], r)
            dp = torch.matmul(do, vt)
            put(outs[3], torch.matmul(p.transpose(2, 3).contiguous(), do), 1)
            ds = dp.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
            put(outs[1], torch.matmul(ds, k), r)
            put(outs[2], torch.matmul(ds.transpose(2, 3).contiguous(), q), 1)
    return tuple(outs) if case["train"] else outs[0]


# --------------------------------------------------------------------------------------
# the same outputs in 64 bits
# --------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"norm": _exact_norm, "pack": _exact_pack, "linear8": _exact_linear8, "attention": _exact_attention}[case["op"]](st)


def _exact_values8(x):
    parts = []
    for cols in torch.split(x.double(), BLOCK, dim=1):
        top = cols.abs().max(dim=1, keepdim=True).values
        exponent = torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - 6
        exponent = torch.where(top >= 127.5 * torch.exp2(exponent), exponent + 1, exponent)
        step = torch.exp2(torch.where(top > 0, exponent, -126.0).clamp(min=-126.0))
        parts.append(torch.round(cols / step) * step)
    return torch.cat(parts, dim=1)


def _exact_pack(st):
    return _exact_values8(st["x"])


def _exact_norm(st):
    case = st["case"]
    c, grp = st["x"].size(1), case["groups"]
    per = c // grp
    w, b = st["weight"].double(), st["bias"].double()
    values = _exact_values8(st["x"]) if case["keep8"] else None

    def act(z):
        if case["act"] == "silu":
            return z * torch.sigmoid(z)
        if case["act"] == "gelu":
            return 0.5 * z * torch.erfc(-z / math.sqrt(2.0))
        return z * 1.0

    out, gx = [], []
    gw, gb = torch.zeros_like(w), torch.zeros_like(b)
    at = 0
    for s in _sizes(case):
        if s == 0:
            continue
        x = st["x"][at:at + s].double()
        cols = x.view(s, grp, per).transpose(0, 1).reshape(grp, s * per)
        var, mean = torch.var_mean(cols, dim=1, correction=0)
        sd = torch.sqrt(var + 1e-5).repeat_interleave(per)
        mean = mean.repeat_interleave(per)
        out.append(act((x - mean) / sd * w + b))
        if case["train"]:
            # gradient with respect to z at the kept values, then through the normalisation, whose Jacobian is
            # (identity - mean - projection on the kept normalised values) / sd
            xh = ((values[at:at + s] if case["keep8"] else x) - mean) / sd
            z = (xh * w + b).requires_grad_()
            (dz,) = torch.autograd.grad(act(z), z, st["g"][at:at + s].double())
            gw += (dz * xh).sum(0)
            gb += dz.sum(0)
            a = (dz * w).view(s, grp, per)
            xg = xh.view(s, grp, per)
            a = a - a.mean((0, 2), keepdim=True) - xg * (a * xg).mean((0, 2), keepdim=True)
            gx.append(a.reshape(s, c) / sd)
        at += s
    if not case["train"]:
        return torch.cat(out)
    return torch.cat(out), torch.cat(gx), gw, gb


def _exact_linear8(st):
    x, w, g = st["x"].double(), st["weight"].double(), st["g"].double()
    return torch.addmm(st["bias"].double(), x, w.t()), g @ w, g.t() @ _exact_values8(st["x"]), g.sum(0)


def _exact_attention(st):
    case = st["case"]
    h, hk, d = case["heads"], case["kv_heads"], case["width"]
    r = h // hk
    q, k, v = (st[n].double() for n in "qkv")
    out = torch.zeros_like(q)
    grads = [torch.zeros_like(t) for t in (q, k, v)] if case["train"] else None
    at = 0
    for s in _sizes(case):
        rows = slice(at, at + s)
        at += s
        ok = torch.arange(s, device=q.device) if st["mask"] is None else st["mask"][rows].nonzero().squeeze(1)
        if ok.numel() == 0:
            continue
        for head in range(h):
            a = [q[rows, head].contiguous(), k[rows, head // r][ok], v[rows, head // r][ok]]
            if not case["train"]:
                out[rows, head] = torch.softmax(a[0] @ a[1].t().contiguous() / math.sqrt(d), dim=-1) @ a[2]
                continue
            a = [t.requires_grad_() for t in a]
            o = torch.softmax(a[0] @ a[1].t() / math.sqrt(d), dim=-1) @ a[2]
            gq, gk, gv = torch.autograd.grad(o, a, st["g"][rows, head].double())
            out[rows, head] = o.detach()
            grads[0][rows, head] = gq
            grads[1][rows, head // r] = grads[1][rows, head // r].index_add(0, ok, gk)
            grads[2][rows, head // r] = grads[2][rows, head // r].index_add(0, ok, gv)
    return (out, *grads) if case["train"] else out
