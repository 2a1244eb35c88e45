"""The query decoder: cross attention, gated residual norms and gradient clipping as a head of the encoder runs and trains them,
against the same head of plain operations in 64 bits."""
import copy
import math

import pytest
import torch
import torch.nn.functional as F

import sphconv_b200 as sphconv
from sphconv_b200 import sharding, synthetic
from sphconv_b200.attention import cross_attention, scan_rows
from sphconv_b200.encoder import build_encoder8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SHAPE = [12, 20, 32]


def scans(lengths, channels, dtype=torch.float32, seed=0):
    """A tensor whose scan b has lengths[b] rows."""
    g = torch.Generator().manual_seed(seed)
    cells = [torch.randperm(math.prod(SHAPE), generator=g)[:n] for n in lengths]
    idx = torch.cat([torch.stack([torch.full_like(c, b), c // (SHAPE[1] * SHAPE[2]), c // SHAPE[2] % SHAPE[1], c % SHAPE[2]], 1)
                     for b, c in enumerate(cells)])
    rows = torch.randn(sum(lengths), channels, generator=g).to(DEV, dtype)
    return sphconv.SparseConvTensor(rows, SHAPE, len(lengths), indices=idx.int().to(DEV))


def plain_norm(x, weight, bias, eps, center):
    x = x - x.mean(-1, keepdim=True) if center else x
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight
    return y if bias is None else y + bias


def plain_attention(m, queries, rows, q_ptr, k_ptr, mask, notes=None):
    q = m.to_q(queries).view(-1, m.heads, m.head_channels)
    k, v = (t.repeat_interleave(m.heads // m.key_heads, 1) for t in m.to_kv(rows).view(-1, 2, m.key_heads, m.head_channels).unbind(1))
    out, seen, scale = [], [], 1 / math.sqrt(m.head_channels)
    for b in range(len(q_ptr) - 1):
        ks = torch.arange(k_ptr[b], k_ptr[b + 1], device=DEV)
        ks = ks if mask is None else ks[mask[ks]]
        s = torch.einsum("qhd,khd->hqk", q[q_ptr[b]:q_ptr[b + 1]], k[ks]) * scale
        out.append(torch.einsum("hqk,khd->qhd", F.softmax(s, -1), v[ks]))
        seen.append((F.softmax(s, -1).detach(), k[ks].detach().abs(), v[ks].detach().abs()))
    out = torch.cat(out)

    def score_gradients(d_out):
        """What the product's gradient of to_q.weight may be off by for `compare`'s second reason."""
        off = []
        for b, (p, k, v) in enumerate(seen):
            d = d_out[q_ptr[b]:q_ptr[b + 1]].abs()
            each = torch.einsum("qhd,khd->hqk", d, v)
            both = each + torch.einsum("hqk,hqk->hq", p, each)[..., None]
            off.append(torch.einsum("hqk,khd->qhd", p * both, k) * scale * 2 * (m.head_channels + 4) * 2.0 ** -24)
        return torch.cat(off).flatten(1).T @ queries.detach().abs()

    if notes is not None:
        notes.append((m.to_q.weight, out, score_gradients))
    return m.to_out(out.flatten(1))


def plain_decoder(net, feature, rows, q_ptr, k_ptr, mask=None, notes=None):
    """What QueryDecoder computes, from its parameters (of any type) with torch's operations alone."""
    norm = lambda m, x: plain_norm(x, m.weight, m.bias, m.eps, m.center)  # noqa: E731

    def behind(m, block, x, gate=None):
        step = block if m.scale is None else block * m.scale
        x = x + (step if gate is None else step * torch.sigmoid(gate))
        return x, plain_norm(x, m.next_weight, m.next_bias, m.eps, m.center)

    memory, normed = norm(net.norm_rows, feature), norm(net.norm, rows)
    for layer in net.layers:
        rows, normed = behind(layer.after_attention, plain_attention(layer.attention, normed, memory, q_ptr, k_ptr, mask, notes), rows,
                              layer.gate(normed))
        rows, normed = behind(layer.after_mlp, layer.mlp(normed), rows)
    return normed


def compare(got, plain, exact, more):
    """Both sides round in the same places, in sums of their own order: a sum of n terms is off by at most n u, commonly by sqrt(n) u of
    their size, and what follows carries it on alike.  So `got` may be 8 times as far from 64 bits as torch's float32 is, and a few
    roundings of the largest value (16 u) where that happens to be exact.

    In one place they do not round alike.  A score's gradient is P (dP - delta) with dP = d_out . v and delta = sum over keys of P dP, which
    is d_out . out: the kernels take it from there, torch from the products.  Where a query has a single key the difference is zero, and
    torch's is so exactly.  d_out . v and d_out . out are sums of d products, of error (d + 4) u of the products' sizes each, so a
    score's gradient is off by 2 (d + 4) u P (|d_out| |v| + |d_out| P |v|), a query's by that times scale |k|, summed over keys, and
    to_q.weight's by that times the queries, summed over them: `more`."""
    for g, p, e, m in zip(got, plain, exact, more):
        bound = m + 8 * (p.double() - e).abs().max() + 16 * 2.0 ** -24 * e.abs().max()
        assert g.shape == e.shape and bool(((g.double() - e).abs().max() <= bound).item()), ((g.double() - e).abs().max(), bound)


def make(channels=64, row_channels=48, seed=5, **kw):
    torch.manual_seed(seed)
    net = sphconv.QueryDecoder(channels, row_channels, **dict(dict(heads=4, layers=2), **kw)).to(DEV)
    with torch.no_grad():                       # norms and scales that are not all the same
        for name, p in net.named_parameters():
            if p.dim() == 1:
                p.add_(0.2 * torch.randn_like(p))
    return net


@pytest.mark.parametrize("kw,ragged,masked", [
    (dict(queries=7), False, False),
    (dict(queries=33, key_heads=2, center=True, initial_scale=0.5), False, True),
    (dict(key_heads=1, channels=40, row_channels=64, hidden=24, layers=1), True, False),
    (dict(heads=2, channels=256, initial_scale=1.0), True, True),
])
def test_against_plain_operations(kw, ragged, masked):
    x = scans([300, 0, 41, 1, 129], kw.get("row_channels", 48))
    net = make(**kw)
    x.feature = x.feature.detach().requires_grad_()
    lengths = [5, 3, 0, 70, 1] if ragged else [kw.get("queries", 0)] * 5
    q_ptr = [sum(lengths[:i]) for i in range(6)]
    k_ptr = scan_rows(x).tolist()
    mask = torch.rand(x.feature.shape[0], generator=torch.Generator(device=DEV).manual_seed(1), device=DEV) < 0.6 if masked else None
    given = torch.randn(sum(lengths), kw.get("channels", 64), device=DEV) if ragged else None
    g = torch.randn(sum(lengths), kw.get("channels", 64), device=DEV)

    def run(net, feature, rows, call):
        wrt = [p for p in net.parameters() if p.requires_grad] + [feature] + ([rows] if ragged else [])
        out = call(net, feature, rows if ragged else net.queries.repeat(5, 1))
        grads = torch.autograd.grad(out, wrt + [o for _, o, _ in notes], g.to(out.dtype))
        more = {w: off(d).max() for (w, _, off), d in zip(notes, grads[len(wrt):])}
        notes.clear()
        return [out.detach()] + list(grads[:len(wrt)]), [0.0] + [more.get(w, 0.0) for w in wrt]

    def own(net, feature, rows):
        if ragged:
            return net(x, rows, torch.tensor(q_ptr, dtype=torch.int32, device=DEV), key_mask=mask)
        return net(x, key_mask=mask).flatten(0, 1)

    notes = []
    plain = lambda net, f, r: plain_decoder(net, f, r, q_ptr, k_ptr, mask, notes)  # noqa: E731
    leaf = lambda t, dtype: None if t is None else t.detach().to(dtype).requires_grad_()  # noqa: E731
    got, _ = run(net, x.feature, leaf(given, torch.float32), own)
    want32, _ = run(net, leaf(x.feature, torch.float32), leaf(given, torch.float32), plain)
    want64, more = run(copy.deepcopy(net).double(), leaf(x.feature, torch.float64), leaf(given, torch.float64), plain)
    compare(got, want32, want64, more)
    sphconv.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_after_token_reads_the_same_memory(dtype):
    """Queries of a scan do not see one another: taken one at a time they give what they give together."""
    x = scans([200, 90, 333], 48, dtype)
    net = make().to(dtype).eval()
    rows = torch.randn(3, 6, 64, device=DEV).to(dtype)
    step = torch.arange(4, dtype=torch.int32, device=DEV)
    with torch.no_grad():
        memory = net.memory(x)
        all_at_once = net.decode(rows.flatten(0, 1), step * 6, memory).view(3, 6, 64)
        one_by_one = torch.stack([net.decode(rows[:, i].contiguous(), step, memory) for i in range(6)], 1)
        # the same step captured once and replayed with other rows in place
        held = rows[:, 0].contiguous()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            net.decode(held, step, memory)
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            replayed = net.decode(held, step, memory)
        for i in (4, 2):
            held.copy_(rows[:, i])
            graph.replay()
            # each of about 20 operations rounds to the type once, and each is carried on by the norms at its relative size
            assert (replayed - one_by_one[:, i]).abs().max() <= 40 * torch.finfo(dtype).eps / 2 * one_by_one.abs().max()
    # two roundings of different sums instead of one at each place
    assert (all_at_once - one_by_one).abs().max() <= 40 * torch.finfo(dtype).eps / 2 * one_by_one.abs().max()
    sphconv.check_status()


def test_training_step_with_the_encoder():
    """Encoder, decoder, loss, gradients in one buffer, clipped on their way into bf16: with the norm and the values that the buffer's
    float32 gradients have in 64 bits."""
    torch.manual_seed(0)
    b = synthetic.make_batch(dict(id=3, B=2, shape=[16, 32, 64], occ=0.9, nbins="uniform", nmax=4, depth="lognormal", C=4), batch=2)
    x = sphconv.SparseConvTensor(torch.as_tensor(b["feature"], device=DEV).bfloat16(), b["shape"], b["B"],
                                 z_idx=torch.as_tensor(b["z_idx"], device=DEV), z_ptr=torch.as_tensor(b["z_ptr"], device=DEV))
    encoder = build_encoder8(torch.bfloat16, DEV)
    head = sphconv.QueryDecoder(64, 64, heads=4, layers=2, queries=20, key_heads=2, initial_scale=0.5).to(DEV, torch.bfloat16)
    params = list(encoder.parameters()) + list(head.parameters())
    buffer = sharding.GradBuffer(params)
    optimizer = torch.optim.SGD(params, lr=1e-3)
    target = torch.randn(2, 20, 64, device=DEV)
    for _ in range(2):
        buffer.zero()
        optimizer.zero_grad()
        before = [p.detach().clone() for p in params]
        F.mse_loss(head(encoder(x)).float(), target).backward()
        buffer.absorb_autograd()
        buffer.all_reduce()
        exact = buffer.flat.double().norm()
        assert exact > 0 and bool(torch.isfinite(exact))
        limit = float(exact) / 3
        norm = buffer.to_grads(max_norm=limit)
        # squares are summed in float32 over at most 64 values a thread before the sums are joined
        assert abs(norm.double() - exact) <= 128 * 2.0 ** -24 * exact
        for p, v in zip(params, buffer.views):
            want = v.double() * (limit / (exact + 1e-6))
            assert ((p.grad.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -16) * want.abs() + 1e-38).all()
        assert buffer.views[0].abs().max() > 0 and head.queries.grad.abs().max() > 0      # the first layer of either was reached
        optimizer.step()
        assert any(not torch.equal(p, q) for p, q in zip(params, before))
    sphconv.check_status()


def test_refusals():
    x = scans([10, 4], 48)
    net = make(queries=3)
    with pytest.raises(ValueError, match="q_ptr"):
        net(x, torch.randn(5, 64, device=DEV))
    with pytest.raises(RuntimeError, match="dtype"):
        net.layers[0].after_mlp(torch.randn(5, 64, device=DEV).half(), torch.randn(5, 64, device=DEV))
    with pytest.raises(RuntimeError, match="key_mask"):
        net(x, key_mask=torch.ones(13, dtype=torch.bool, device=DEV))
    k, v = net.layers[0].attention.project(x.feature)
    assert k.data_ptr() + 64 * 4 == v.data_ptr()             # read where the product left them
    q = torch.randn(6, 4, 16, device=DEV)
    assert cross_attention(q, k, v, torch.tensor([0, 3, 6], dtype=torch.int32, device=DEV), scan_rows(x)).shape == q.shape
