"""The global gradient norm and clipping: on the CPU (the plain path of a gloo job), and the kernels against 64-bit sums."""
import math

import pytest
import torch

from sphconv_b200 import sharding
from sphconv_b200.sharding import GradBuffer, clip_grad_norm_, clip_gradients, grad_norm

gpu = pytest.mark.gpu
DEV = "cuda:0"
EPS = {torch.float32: 2 ** -24, torch.float16: 2 ** -11, torch.bfloat16: 2 ** -8}     # half a step, relative


def want(grads, max_norm, largest=False):
    flat = torch.cat([g.double().flatten() for g in grads])
    norm = flat.abs().max().item() if largest else flat.square().sum().sqrt().item()
    return norm, min(1.0, max_norm / (norm + 1e-6))


def check(grads, out, norm, max_norm, largest=False):
    ref, by = want(grads, max_norm, largest)
    # the norm is rounded once to float32; the factor by a sum and a division, the product once, then the destination's type
    assert abs(norm.item() - ref) <= 2 ** -23 * ref
    for g, o in zip(grads, out):
        e = (o.double() - g.double() * by).abs()
        tiny = 2 ** -25 if o.dtype == torch.float16 else 0.0            # half a step below the normal range
        assert (e <= (EPS[o.dtype] + 2 ** -21) * (g.double() * by).abs() + tiny).all()


def tensors(sizes, types, device, scale=0.01, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale).to(t).to(device) for n, t in zip(sizes, types)]


def test_cpu_lists_and_buffer():
    grads = tensors([5, 1, 300], [torch.float32, torch.bfloat16, torch.float32], "cpu")
    out = [torch.empty(g.shape, dtype=torch.float32) for g in grads]
    norm = clip_gradients(grads, 0.05, out=out)
    check(grads, out, norm, 0.05)
    assert abs(grad_norm(grads, math.inf).item() - want(grads, 1.0, True)[0]) < 1e-7
    lin = torch.nn.Linear(7, 3).to(torch.bfloat16)
    gb = GradBuffer(lin.parameters())
    gb.flat.copy_(torch.randn(gb.flat.shape))
    kept = gb.flat.clone()
    norm = gb.to_grads(max_norm=0.5)
    check(gb.views, [p.grad for p in lin.parameters()], norm, 0.5)
    assert torch.equal(gb.flat, kept) and torch.equal(gb.norm(), norm)
    assert gb.to_grads() is None and torch.equal(lin.weight.grad, gb.views[0].to(torch.bfloat16))


def test_cpu_refusals():
    g = torch.ones(4)
    with pytest.raises(ValueError):
        grad_norm([g], 1.0)
    with pytest.raises(ValueError):
        clip_gradients([g], -1.0)
    with pytest.raises(ValueError):
        clip_gradients([g], 1.0, out=[])
    with pytest.raises(RuntimeError, match="twice"):
        clip_gradients([g, g], 1.0)
    assert clip_grad_norm_([torch.nn.Parameter(g)], 1.0).item() == 0.0 and grad_norm([]).item() == 0.0


def test_cpu_refuses_what_the_gpu_refuses():
    g = torch.ones(64)
    other = torch.empty(32)
    for grads, out in (([g, g], None), ([g[:40], g[30:]], None), ([g[:40], g[:8]], None),
                       ([g[:32], g[32:]], [g[1:33], other]), ([g[:32], g[32:]], [other, other]),
                       ([g[:32], g[32:]], [other, other[:32]]), ([g[32:], g[:32]], [g[:32], other]),
                       ([g], [torch.empty(63)]), ([g[:4]], [torch.empty(1, 4)]), ([g[:1]], [torch.empty(4)]),
                       ([g.view(8, 8)], [torch.empty(8, 8).t()]), ([g.double()], None), ([g], [torch.empty(64).double()]),
                       ([g[::2]], None), ([g[:1].expand(4)], None), ([g.bfloat16()], [g.bfloat16().view(torch.float16).double()]),
                       ([g[:32]], [g.view(torch.bfloat16)[:32]]), ([g, g.to("meta")], None)):
        kept = g.clone()
        with pytest.raises(RuntimeError):
            clip_gradients(grads, 1.0, out=out)
        assert torch.equal(g, kept)                           # nothing was written
    assert grad_norm([g[:40], g[30:]]).item() == pytest.approx(math.sqrt(74))         # reading twice is fine
    # and what is allowed: neighbours, reading a value for two destinations, an order of dimensions that both have, nothing at all
    a, b = torch.ones(64), torch.ones(64)
    clip_gradients([a[:32], a[32:]], 0.5)
    clip_gradients([b[:32], b[:32]], 0.5, out=[other, torch.empty(32)])
    clip_gradients([b.view(8, 8).t()], 0.5, out=[torch.empty(8, 8).t()])
    clip_gradients([b[:0], b[:0], b[:1]], 0.5)
    check([torch.ones(64)], [a], torch.tensor(8.0), 0.5)


SIZES = {
    "one": [1], "odd": [1, 7, 8, 9, 2047, 2048, 2049, 0, 100003], "many": [((i * 7919) % 5000) + 1 for i in range(400)],
    "large": [40_000_001, 3],
}


@gpu
@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("source,to", [("fp32", "bf16"), ("bf16", "bf16"), ("fp16", "fp32"), ("mixed", "mixed")])
def test_against_64_bits(sizes, source, to):
    pick = lambda name, i: {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}.get(name) or \
        [torch.float32, torch.float16, torch.bfloat16][i % 3]  # noqa: E731
    n = SIZES[sizes]
    grads = tensors(n, [pick(source, i) for i in range(len(n))], DEV)
    out = [torch.full(g.shape, 7.0, dtype=pick(to, i + 1 if to == "mixed" else i), device=DEV) for i, g in enumerate(grads)]
    max_norm = 0.3 * want(grads, 1.0)[0]
    norm = clip_gradients(grads, max_norm, out=out)
    assert norm.dtype == torch.float32 and norm.dim() == 0 and norm.is_cuda
    check(grads, out, norm, max_norm)
    top = clip_gradients(grads, 0.001, out=out, norm_type=math.inf)
    check(grads, out, top, 0.001, True)
    assert torch.equal(grad_norm(grads), norm) and torch.equal(grad_norm(grads, math.inf), top)
    kept = [g.clone() for g in grads]
    assert torch.equal(clip_gradients(grads, max_norm), norm)           # in place
    check(kept, grads, norm, max_norm)


@gpu
def test_slices_of_a_buffer_and_what_lies_between():
    flat = torch.randn(5000, device=DEV)
    kept = flat.clone()
    cut = [flat[1:4], flat[4:1001], flat[1003:1004], flat[2000:4999]]   # the first two follow one another
    clip_gradients(cut, 1.0)
    inside = torch.zeros(5000, dtype=torch.bool, device=DEV)
    for a, b in ((1, 1001), (1003, 1004), (2000, 4999)):
        inside[a:b] = True
    assert torch.equal(flat[~inside], kept[~inside])
    check([kept[inside]], [flat[inside]], kept[inside].double().norm().float(), 1.0)


@gpu
def test_no_clipping_leaves_the_bits():
    g = tensors([1000, 33], [torch.bfloat16, torch.float32], DEV)
    kept = [x.clone() for x in g]
    norm = clip_gradients(g, 1e9)
    assert all(torch.equal(a, b) for a, b in zip(g, kept)) and torch.equal(norm, grad_norm(g))
    out = [torch.empty_like(x) for x in g]
    clip_gradients(g, 1e9, out=out)
    assert all(torch.equal(a, b) for a, b in zip(out, kept))


@gpu
@pytest.mark.parametrize("scale", [1e-30, 1e-22, 1e20, 3e37])
def test_norms_whose_squares_leave_float32(scale):
    g = [torch.full((3001,), scale, device=DEV), torch.full((7,), 2 * scale, device=DEV)]
    ref = scale * math.sqrt(3001 + 28)
    norm = grad_norm(g).item()
    assert norm == math.inf if ref > 3.4e38 else abs(norm - ref) <= 2 ** -20 * ref      # scale itself is rounded to float32


@gpu
def test_values_that_are_not_finite():
    g = [torch.ones(100, device=DEV), torch.ones(5, device=DEV, dtype=torch.bfloat16)]
    g[1][2] = float("nan")
    assert clip_gradients([x.clone() for x in g], 1.0).isnan() and grad_norm(g, math.inf).isnan()
    mine = [x.clone() for x in g]
    clip_gradients(mine, 1.0)
    assert all(x.isnan().all() for x in mine)
    g[1][2] = float("inf")
    mine = [x.clone() for x in g]
    assert clip_gradients(mine, 1.0).isinf()
    assert not mine[0].any() and mine[1].isnan().tolist() == [False, False, True, False, False]


@gpu
def test_same_bits_on_another_stream_and_in_graphs():
    g = tensors([(i * 997) % 3000 + 1 for i in range(200)], [torch.bfloat16] * 200, DEV)
    out = [torch.empty_like(x) for x in g]
    norm = clip_gradients(g, 0.1, out=out).clone()
    kept = [x.clone() for x in out]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(clip_gradients(g, 0.1, out=out), norm)
    side.synchronize()
    graphs, norms = [torch.cuda.CUDAGraph() for _ in range(2)], []
    other = [torch.empty_like(x) for x in g]
    for graph, to in zip(graphs, (out, other)):
        with torch.cuda.graph(graph):
            norms.append(clip_gradients(g, 0.1, out=to))
    for x in out + other:
        x.zero_()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):                                   # side by side: each graph has a workspace of its own
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(norms[0], norm) and torch.equal(norms[1], norm)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(kept, out, other))


@gpu
def test_grad_buffer_and_parameters():
    net = torch.nn.Sequential(torch.nn.Linear(33, 65), torch.nn.Linear(65, 3)).to(DEV).to(torch.bfloat16)
    gb = GradBuffer(net.parameters())
    gb.flat.copy_(torch.randn_like(gb.flat))
    norm = gb.to_grads(max_norm=1.0)
    check(gb.views, [p.grad for p in gb.params], norm, 1.0)
    assert torch.equal(gb.norm(), norm)
    kept = [p.grad.clone() for p in gb.params]
    assert torch.equal(clip_grad_norm_(list(net.parameters()) * 2, 0.25), grad_norm(kept))      # each parameter once
    check(kept, [p.grad for p in gb.params], grad_norm(kept), 0.25)


@gpu
def test_writes_are_seen_by_autograd():
    g = torch.randn(10, device=DEV)
    leaf = torch.randn(10, device=DEV, requires_grad=True)
    y = (leaf * g).sum()
    clip_gradients([g], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@gpu
def test_refusals():
    g = torch.randn(64, device=DEV)
    for call in (lambda: clip_gradients([g, g], 1.0), lambda: clip_gradients([g[:40], g[30:]], 1.0),
                 lambda: clip_gradients([g[:32], g[32:]], 1.0, out=[g[1:33], torch.empty(32, device=DEV)]),
                 lambda: clip_gradients([g], 1.0, out=[torch.empty(63, device=DEV)]), lambda: clip_gradients([g.double()], 1.0),
                 lambda: clip_gradients([g[::2]], 1.0), lambda: clip_gradients([g, torch.ones(3)], 1.0),
                 lambda: clip_gradients([g.view(8, 8)], 1.0, out=[torch.empty(8, 8, device=DEV).t()])):
        with pytest.raises(RuntimeError):
            call()
    assert sharding.grad_norm([g[:40], g[30:]]).item() > 0              # reading twice is fine
