"""Operators of a query head on the sparse encoder and of its training step, as cases that can be timed: cross attention of a
head's queries to the rows of their scan, the norms around a block fused with its gate and residual scale, and the global norm of
many gradients with clipping.

A case is a dict of plain values:
  op        attention | residual | clip
  dtype     type of the rows (attention, residual) or of the parameters that the clipped gradients go to (clip)
  train     attention, residual: forward and backward
  attention: B scans with about `nq` queries and `nk` rows each; hq query heads over hkv key heads of d channels; `ragged`: 0, or a
            number that the scans' different lengths are drawn by (the last but one of three or more scans has no rows); `masked`:
            every eighth row or so is no key, and holds NaN
  residual: n rows of c channels; center: layer norm (else RMS); gate: none | row | element; scaled: a residual scale per channel
  clip:     tensors gradients of up to `largest` values; source: fp32 (a flat buffer's slices) or same (as the parameters)
"""
import math
import random

import torch

own = False                                              # True: run() calls this framework's operators

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ESIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
MOST_FLOPS = 9e10                                         # of a drawn attention case, a quarter of it in float32
MOST_SCORES = 6e8                                         # queries x rows x heads of one


def listed():
    return [
        # a head of one query over a small scan, fp32: latency of a call
        dict(name="query_small", op="attention", dtype="fp32", train=False, B=1, nq=1, nk=700, hq=4, hkv=4, d=16, ragged=0, masked=False),
        # one token a scan asks about the encoder's output of 8 scans (about 87 k rows each): reads keys and values once
        dict(name="token_8", op="attention", dtype="bf16", train=False, B=8, nq=1, nk=87000, hq=8, hkv=2, d=64, ragged=5, masked=False),
        # a detection head's 200 queries over the same rows, narrow heads
        dict(name="head_8", op="attention", dtype="fp16", train=False, B=8, nq=200, nk=87000, hq=4, hkv=4, d=32, ragged=0, masked=False),
        # a text decoder's prompt over an encoder's states, wide heads, four query heads to a key head
        dict(name="prompt_wide", op="attention", dtype="bf16", train=False, B=4, nq=2048, nk=4096, hq=16, hkv=4, d=128, ragged=3, masked=False),
        # a training step's attention: 300 queries, 8 heads, scans of different lengths
        dict(name="head_train", op="attention", dtype="bf16", train=True, B=8, nq=300, nk=12000, hq=8, hkv=8, d=64, ragged=1, masked=False),
        # odd sizes, masked rows, a scan without rows, float32, both directions
        dict(name="odd_train", op="attention", dtype="fp32", train=True, B=3, nq=131, nk=3001, hq=6, hkv=2, d=40, ragged=2, masked=True),
        # the queries of a head after a block: few rows
        dict(name="queries_norm", op="residual", dtype="fp16", train=False, n=200, c=128, center=True, gate="none", scaled=False),
        # the encoder's output rows of 8 scans, both directions
        dict(name="rows_train", op="residual", dtype="bf16", train=True, n=696000, c=64, center=False, gate="row", scaled=True),
        # a wide model's tokens, both directions, everything on
        dict(name="tokens_train", op="residual", dtype="bf16", train=True, n=16384, c=2048, center=False, gate="element", scaled=True),
        # channels that are no multiple of anything, float32, layer norm
        dict(name="odd_norm", op="residual", dtype="fp32", train=True, n=50001, c=100, center=True, gate="element", scaled=True),
        # the 8-layer encoder's gradients from the flat float32 buffer to bf16 parameters
        dict(name="clip_encoder", op="clip", dtype="bf16", tensors=16, largest=110592, source="fp32"),
        # many gradients of a large model, in their own type
        dict(name="clip_large", op="clip", dtype="bf16", tensors=60, largest=8388608, source="same"),
    ]


def draw(rng):
    def between(lo, hi):                                  # over the logarithm, both ends included
        return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    op = rng.choice(["attention", "attention", "attention", "residual", "residual", "clip"])
    dtype = rng.choice(["fp32", "fp16", "bf16", "bf16"])
    if op == "attention":
        train = rng.random() < 0.5
        hkv, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 3, 4, 8])
        c = dict(op=op, dtype=dtype, train=train, B=rng.randint(1, 8), nq=1 if rng.random() < 0.25 and not train else between(2, 2048),
                 nk=between(16, 100000), hq=hkv * group, hkv=hkv, d=rng.choice([16, 32, 64, 128, 8 * rng.randint(1, 16)]),
                 ragged=rng.choice([0, rng.randint(1, 999)]), masked=rng.random() < 0.3)
        most = min(MOST_SCORES, MOST_FLOPS / ((14 if train else 4) * c["d"] * (4 if dtype == "fp32" else 1)))
        while c["B"] * c["nq"] * c["nk"] * c["hq"] > most:
            c["nk" if c["nk"] > 4 * c["nq"] else "nq"] //= 2
        while c["B"] * c["nk"] * hkv * c["d"] > 1.6e8:
            c["nk"] //= 2
        return c
    if op == "residual":
        ch = rng.choice([16, 32, 64, 128, 256, 1024, 4096, rng.randint(3, 2000)])
        return dict(op=op, dtype=dtype, train=rng.random() < 0.6, n=between(1, max(1, 32_000_000 // ch)), c=ch, center=rng.random() < 0.4,
                    gate=rng.choice(["none", "row", "element"]), scaled=rng.random() < 0.6)
    return dict(op=op, dtype=dtype, tensors=between(1, 60), largest=between(64, 8_000_000), source=rng.choice(["fp32", "same"]))


# ---- sizes ----------------------------------------------------------------------------------------------------------

def _lengths(case):
    """(queries, rows) of every scan."""
    B, nq, nk = case["B"], case["nq"], case["nk"]
    if not case["ragged"]:
        return [nq] * B, [nk] * B
    r = random.Random(case["ragged"])
    q = [max(1, int(nq * r.uniform(0.4, 1.0))) for _ in range(B)]
    k = [max(1, int(nk * r.uniform(0.3, 1.0))) for _ in range(B)]
    if B >= 3:
        k[B - 2] = 0
    return q, k


def _sizes(case):
    """Numbers of values of the clipped tensors: weights and biases, as a model's parameters come."""
    r = random.Random(case["tensors"] * 1000003 + case["largest"])
    return [max(1, int(case["largest"] * r.random() ** 2)) if i % 2 == 0 else r.randint(1, max(1, min(4096, case["largest"])))
            for i in range(case["tensors"])]


def work(case):
    e = ESIZE[case["dtype"]]
    if case["op"] == "attention":
        lq, lk = _lengths(case)
        scores = case["hq"] * sum(a * b for a, b in zip(lq, lk))
        rows = case["hq"] * case["d"] * sum(lq) * e, case["hkv"] * case["d"] * sum(lk) * e
        if not case["train"]:
            return {"bytes": 2 * rows[0] + 2 * rows[1], "flops": 4 * case["d"] * scores}
        return {"bytes": 4 * rows[0] + 4 * rows[1], "flops": 14 * case["d"] * scores}
    if case["op"] == "residual":
        n, c = case["n"], case["c"]
        gate = {"none": 0, "row": n, "element": n * c}[case["gate"]]
        if not case["train"]:
            return {"bytes": e * (4 * n * c + gate), "flops": 12 * n * c}
        return {"bytes": e * (8 * n * c + 2 * gate), "flops": 40 * n * c}      # block, residual, 2 gradients in; 2 rows, 2 gradients out
    total = sum(_sizes(case))
    return {"bytes": total * ((4 if case["source"] == "fp32" else e) + e), "flops": 3 * total}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    t = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, type=t):
        return (torch.randn(*shape, generator=gen, device=dev) * scale).to(type)

    s = {"case": case}
    if case["op"] == "attention":
        lq, lk = _lengths(case)
        s["lq"], s["lk"] = lq, lk
        s["q_ptr"] = torch.tensor([sum(lq[:i]) for i in range(len(lq) + 1)], dtype=torch.int32, device=dev)
        s["k_ptr"] = torch.tensor([sum(lk[:i]) for i in range(len(lk) + 1)], dtype=torch.int32, device=dev)
        s["q"] = normal(sum(lq), case["hq"], case["d"], scale=1.5)
        kv = normal(sum(lk), 2, case["hkv"], case["d"])  # one projection makes keys and values, side by side
        s["mask"] = None
        if case["masked"]:
            s["mask"] = torch.rand(sum(lk), generator=gen, device=dev) < 0.875
            kv[~s["mask"]] = float("nan")
        s["k"], s["v"] = kv[:, 0], kv[:, 1]
        names = ["q", "k", "v"]
        s["d_out"] = normal(sum(lq), case["hq"], case["d"]) if case["train"] else None
    elif case["op"] == "residual":
        n, c = case["n"], case["c"]
        s["block"], s["residual"] = normal(n, c, scale=0.7), normal(n, c, scale=2.0)
        s["gate"] = {"none": None, "row": normal(n, 1), "element": normal(n, c)}[case["gate"]] if case["gate"] != "none" else None
        for name, mean, wanted in (("weight", 1.0, True), ("bias", 0.0, case["center"]), ("scale", 0.5, case["scaled"]),
                                   ("next_weight", 1.0, True), ("next_bias", 0.0, case["center"])):
            s[name] = (mean + 0.2 * torch.randn(c, generator=gen, device=dev)) if wanted else None
        names = ["block", "residual", "gate", "weight", "bias", "scale", "next_weight", "next_bias"]
        s["d_out"], s["d_normed"] = (normal(n, c), normal(n, c)) if case["train"] else (None, None)
    else:
        sizes = _sizes(case)
        if case["source"] == "fp32":
            s["grads"] = list(normal(sum(sizes), scale=0.01, type=torch.float32).split(sizes))
        else:
            s["grads"] = [normal(n, scale=0.01) for n in sizes]
        s["out"] = [torch.empty(n, dtype=t, device=dev) for n in sizes]
        s["max_norm"] = 0.37 * 0.01 * math.sqrt(sum(sizes))
        names = []
    s["leaves"] = [n for n in names if s[n] is not None]
    if case.get("train"):
        for n in s["leaves"]:
            s[n] = s[n].detach().requires_grad_()
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        return _own(state)
    with torch.no_grad():
        if case["op"] == "attention":
            return _attention(state)
        if case["op"] == "residual":
            return _residual(state)
        return _clip(state)


def _own(s):
    case = s["case"]
    if case["op"] == "clip":
        from sphconv_b200 import sharding
        return {"norm": sharding.clip_gradients(s["grads"], s["max_norm"], out=s["out"]), "grads": s["out"]}
    with torch.set_grad_enabled(case["train"]):
        if case["op"] == "attention":
            from sphconv_b200.attention import cross_attention
            out = {"out": cross_attention(s["q"], s["k"], s["v"], s["q_ptr"], s["k_ptr"], key_mask=s["mask"])}
            upstream = [s["d_out"]]
        else:
            from sphconv_b200.norm import residual_norm
            out = dict(zip(("out", "normed"), residual_norm(
                s["block"], s["residual"], s["weight"], s["bias"], gate=s["gate"], scale=s["scale"], next_weight=s["next_weight"],
                next_bias=s["next_bias"], eps=1e-5, center=case["center"])))
            upstream = [s["d_out"], s["d_normed"]]
        if case["train"]:
            grads = torch.autograd.grad(list(out.values()), [s[n] for n in s["leaves"]], upstream)
            out.update({"d_" + n: g for n, g in zip(s["leaves"], grads)})
    return out


def _scan(s, b):
    """Forward (and backward) of one scan in float32, heads first."""
    case = s["case"]
    lq, lk = s["lq"], s["lk"]
    q0, k0, nq, nk = sum(lq[:b]), sum(lk[:b]), lq[b], lk[b]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    heads = lambda x, at, n, h: x[at:at + n].float().transpose(0, 1).reshape(hkv, h // hkv * n, d)  # noqa: E731
    rows = lambda x, n, h: x.reshape(h, n, d).transpose(0, 1)  # noqa: E731
    q = heads(s["q"], q0, nq, hq)
    k, v = heads(s["k"], k0, nk, hkv), heads(s["v"], k0, nk, hkv)
    scale = 1.0 / math.sqrt(d)
    mask = s["mask"]
    if mask is not None:                                  # what is no key may hold anything
        m = mask[k0:k0 + nk].view(1, nk, 1)
        k, v = torch.where(m, k, 0.0), torch.where(m, v, 0.0)
    if nk == 0:
        out = torch.zeros_like(q)
    else:
        p = torch.matmul(q, k.transpose(1, 2)).mul_(scale)
        if mask is not None:
            p.masked_fill_(~mask[k0:k0 + nk], float("-inf"))
        top = p.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
        p = p.sub_(top).exp_()
        total = p.sum(-1, keepdim=True)
        p.div_(torch.where(total > 0, total, 1.0))
        out = torch.matmul(p, v)
    result = {"out": rows(out, nq, hq)}
    if case["train"]:
        do = heads(s["d_out"], q0, nq, hq)
        if nk == 0:
            result.update(d_q=rows(torch.zeros_like(q), nq, hq), d_k=rows(torch.zeros_like(k), nk, hkv), d_v=rows(torch.zeros_like(v), nk, hkv))
        else:
            dv = torch.matmul(p.transpose(1, 2), do)
            ds = torch.matmul(do, v.transpose(1, 2)).sub_((do * out).sum(-1, keepdim=True)).mul_(p)
            result.update(d_q=rows(torch.matmul(ds, k).mul_(scale), nq, hq), d_k=rows(torch.matmul(ds.transpose(1, 2), q).mul_(scale), nk, hkv),
                          d_v=rows(dv, nk, hkv))
    return result


def _attention(s):
    scans = [_scan(s, b) for b in range(s["case"]["B"])]
    t = DTYPES[s["case"]["dtype"]]
    return {name: torch.cat([x[name] for x in scans]).to(t) for name in scans[0]}


def _norm_forward(x, center):
    x = x - x.mean(-1, keepdim=True) if center else x
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5)
    return x * r, r


def _norm_backward(d, xn, r, center):
    dx = d - xn * (d * xn).mean(-1, keepdim=True)
    return r * (dx - d.mean(-1, keepdim=True) if center else dx)


def _residual(s):
    case = s["case"]
    t, center = DTYPES[case["dtype"]], case["center"]
    x = s["residual"].float()
    bn, br = _norm_forward(s["block"].float(), center)
    inner = bn * s["weight"] + s["bias"] if center else bn * s["weight"]
    gate = torch.sigmoid(s["gate"].float()) if s["gate"] is not None else torch.ones((), device=x.device)
    scale = s["scale"] if s["scale"] is not None else torch.ones((), device=x.device)
    out = x + scale * gate * inner
    on, orr = _norm_forward(out, center)
    normed = on * s["next_weight"] + s["next_bias"] if center else on * s["next_weight"]
    result = {"out": out.to(t), "normed": normed.to(t)}
    if case["train"]:
        do, dn = s["d_out"].float(), s["d_normed"].float()
        total = do + _norm_backward(dn * s["next_weight"], on, orr, center)
        d_inner = total * scale * gate
        grads = {"d_block": _norm_backward(d_inner * s["weight"], bn, br, center).to(t), "d_residual": total.to(t),
                 "d_weight": (d_inner * bn).sum(0, dtype=torch.float64).float(), "d_next_weight": (dn * on).sum(0, dtype=torch.float64).float()}
        if center:
            grads["d_bias"], grads["d_next_bias"] = (x.sum(0, dtype=torch.float64).float() for x in (d_inner, dn))
        if s["gate"] is not None:
            dg = total * scale * inner * gate * (1.0 - gate)
            grads["d_gate"] = (dg.sum(-1, keepdim=True) if case["gate"] == "row" else dg).to(t)
        if s["scale"] is not None:
            grads["d_scale"] = (total * gate * inner).sum(0, dtype=torch.float64).float()
        result.update(grads)
    return result


def _clip(s):
    norm = torch.stack([g.double().square().sum() for g in s["grads"]]).sum().sqrt().float()
    by = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    return {"norm": norm, "grads": [o.copy_(g.float() * by) for o, g in zip(s["out"], s["grads"])]}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "attention":
            return _exact_attention(case, s)
        return _exact_residual(case, s) if case["op"] == "residual" else _exact_clip(case, s)


def _exact_attention(case, s):
    lq, lk = _lengths(case)
    d, group = case["d"], case["hq"] // case["hkv"]
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    keep = s["mask"] if s["mask"] is not None else torch.ones(k.shape[0], dtype=torch.bool, device=k.device)
    res = {"out": torch.zeros_like(q)}
    if case["train"]:
        do = s["d_out"].double()
        res.update(d_q=torch.zeros_like(q), d_k=torch.zeros_like(k), d_v=torch.zeros_like(v))
    q0 = k0 = 0
    for nq, nk in zip(lq, lk):
        at = k0 + torch.nonzero(keep[k0:k0 + nk]).flatten()
        for h in range(case["hq"] if at.numel() else 0):
            kh, vh = k[at, h // group], v[at, h // group]
            for r in range(q0, q0 + nq, 512):
                rows = slice(r, min(r + 512, q0 + nq))
                logits = torch.einsum("id,jd->ij", q[rows, h], kh) / math.sqrt(d)
                prob = torch.exp(logits - torch.logsumexp(logits, 1, keepdim=True))
                o = prob @ vh
                res["out"][rows, h] = o
                if case["train"]:
                    dl = prob * (do[rows, h] @ vh.T - torch.einsum("id,id->i", do[rows, h], o)[:, None]) / math.sqrt(d)
                    res["d_q"][rows, h] = dl @ kh
                    res["d_k"].index_put_((at, torch.full_like(at, h // group)), dl.T @ q[rows, h], accumulate=True)
                    res["d_v"].index_put_((at, torch.full_like(at, h // group)), prob.T @ do[rows, h], accumulate=True)
        q0, k0 = q0 + nq, k0 + nk
    return res


def _exact_residual(case, s):
    v = {n: s[n].detach().double() for n in s["leaves"]}
    n, c = case["n"], case["c"]
    keys = ["out", "normed"] + (["d_" + m for m in s["leaves"]] if case["train"] else [])
    sums = ("d_weight", "d_bias", "d_scale", "d_next_weight", "d_next_bias")
    parts = {m: [] for m in keys}
    step = max(1, 8_000_000 // c)
    for r in range(0, n, step):                          # derivatives by 64-bit automatic differentiation, some rows at a time
        leaf = {m: (x[r:r + step] if m in ("block", "residual", "gate") else x).clone().requires_grad_(case["train"]) for m, x in v.items()}

        def norm(x, w, b):
            dev = x - x.mean(1, keepdim=True) if case["center"] else x
            y = dev / torch.sqrt(torch.mean(dev ** 2, 1, keepdim=True) + 1e-5) * leaf[w]
            return y + leaf[b] if b in leaf else y

        with torch.set_grad_enabled(case["train"]):
            step_ = norm(leaf["block"], "weight", "bias")
            if "gate" in leaf:
                step_ = step_ / (1.0 + torch.exp(-leaf["gate"]))
            if "scale" in leaf:
                step_ = step_ * leaf["scale"]
            out = leaf["residual"] + step_
            normed = norm(out, "next_weight", "next_bias")
            got = {"out": out.detach(), "normed": normed.detach()}
            if case["train"]:
                up = [s["d_out"][r:r + step].double(), s["d_normed"][r:r + step].double()]
                got.update({"d_" + m: g for m, g in zip(s["leaves"], torch.autograd.grad([out, normed], [leaf[m] for m in s["leaves"]], up))})
        for m in keys:
            parts[m].append(got[m])
    return {m: torch.stack(p).sum(0) if m in sums else torch.cat(p) for m, p in parts.items()}


def _exact_clip(case, s):
    norm = torch.linalg.vector_norm(torch.cat([x.double() for x in s["grads"]]))
    return {"norm": norm, "grads": [x.double() * min(1.0, s["max_norm"] / (float(norm) + 1e-6)) for x in s["grads"]]}
