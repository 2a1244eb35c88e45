"""Cross attention scan by scan in 64 bits, with bounds on what rounding may do to each result."""
import math

import torch


def attention64(q, k, v, q_ptr, k_ptr, mask=None, scale=None, d_out=None):
    """{name: (value, bound)} of out, and with d_out of d_q, d_k, d_v; rows of no scan are zero, with a bound of zero.

    The bounds, with u = 2^-24 (float32) and h half a step of the rows' type (the rounding of P, dS and of results; u in float32):
      a score is a sum of d products: |err| <= 2 (d + 4) u sum|q k| scale =: e, so P is off by 2 e + s relative, s = 16 u + n u / 4 for
      2^x, the running sum over n keys (16 threads' or one thread's) and its rescalings;
      out: (2 e + s + h) (P |V|) + h |out|
      dV : (2 e + s + h) (P^T |dO|) + h |dV|
      dS = P (dP - delta): dP is off by (d + 4) u |dO| |V|^T, delta by that of its own sum and h |dO| |out| for the rounded out, dS itself
      by its P and its rounding:  f = P ((d + 4) u (|dO| |V|^T + |dO| |out|) + 2 h |dO| |out|) + (2 e + s + 2 h) |dS| ;
      dQ: scale f |K| + (h + n u) scale |dS| |K| + h |dQ| ; dK likewise.
    fp16 results and operands lose more below the normal range: 2^-25 absolute (and operands are kept above it by scaling)."""
    t = q.dtype
    u = 2.0 ** -24
    h = torch.finfo(t).eps / 2
    tiny = 2.0 ** -24 if t == torch.float16 else 0.0
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else scale
    hq, hkv, d = q.shape[1], k.shape[1], q.shape[2]
    g = hq // hkv
    Q, K, V = q.detach().double(), k.detach().double(), v.detach().double()
    dO = None if d_out is None else d_out.double()
    zero = lambda x: torch.zeros(x.shape, dtype=torch.float64, device=x.device)  # noqa: E731
    names = {"out": Q} if dO is None else {"out": Q, "d_q": Q, "d_k": K, "d_v": V}
    val, tol = {n: zero(x) for n, x in names.items()}, {n: zero(x) for n, x in names.items()}
    qp, kp = q_ptr.tolist(), k_ptr.tolist()
    for b in range(len(qp) - 1):
        qs, ks = slice(qp[b], qp[b + 1]), torch.arange(kp[b], kp[b + 1], device=q.device)
        if mask is not None:
            ks = ks[mask[ks]]
        if ks.numel() == 0 or qp[b] == qp[b + 1]:
            continue
        n = max(ks.numel(), (qp[b + 1] - qp[b]) * g)
        s_ = 16 * u + n * u / 4
        for head in range(hq):
            A, Kh, Vh = Q[qs, head], K[ks, head // g], V[ks, head // g]
            S = A @ Kh.T * scale
            top = S.amax(1, keepdim=True)
            none = top == -math.inf
            P = torch.where(none, 0.0, torch.exp(S - torch.where(none, 0.0, top)))
            P = P / torch.where(none, 1.0, P.sum(1, keepdim=True))
            e = 2 * (d + 4) * u * (A.abs() @ Kh.abs().T) * abs(scale)
            e = e + (e * P).sum(1, keepdim=True)                  # its own score, and those of the sum
            rel = 2 * e + s_ + h
            O = P @ Vh
            val["out"][qs, head] = O
            tol["out"][qs, head] = (rel * P) @ Vh.abs() + h * O.abs() + tiny
            if dO is None:
                continue
            G = dO[qs, head]
            dP = G @ Vh.T
            go = (G.abs() * O.abs()).sum(1, keepdim=True)
            dS = P * (dP - (G * O).sum(1, keepdim=True))
            f = P * ((d + 4) * u * (G.abs() @ Vh.abs().T + go) + 2 * h * go) + (rel + h) * dS.abs()
            f = f + (h + n * u) * dS.abs()
            dQ, dK, dV = scale * dS @ Kh, scale * dS.T @ A, P.T @ G
            val["d_q"][qs, head] = dQ
            tol["d_q"][qs, head] = abs(scale) * f @ Kh.abs() + h * dQ.abs() + tiny
            val["d_k"][ks, head // g] += dK
            tol["d_k"][ks, head // g] += abs(scale) * f.T @ A.abs() + h * dK.abs() + tiny
            val["d_v"][ks, head // g] += dV
            tol["d_v"][ks, head // g] += ((rel + n * u) * P).T @ G.abs() + h * dV.abs() + tiny
    return {n: (val[n], tol[n]) for n in names}


def check(results, wants):
    """Every result within its bound (plus 2^-100, for results that are exactly zero in 64 bits only)."""
    for name, got in results.items():
        want, tol = wants[name]
        over = ((got.double() - want).abs() - tol).max().item() if want.numel() else 0.0
        assert over <= 2.0 ** -100, (name, over, (got.double() - want).abs().max().item(), tol.max().item())
