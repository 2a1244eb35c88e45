"""Cross attention of queries to the rows of their scan, against the formulas in 64 bits."""
import ctypes
import math
import os

import pytest
import torch

import sphconv_b200 as sphconv
from sphconv_b200 import _capi as C
from sphconv_b200 import build as sph_build
from sphconv_b200.attention import cross_attention, scan_rows
from attention_oracle import attention64, check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def ptr(lengths, first=0):
    p = [first]
    for n in lengths:
        p.append(p[-1] + n)
    return torch.tensor(p, dtype=torch.int32, device=DEV)


def inputs(lq, lk, hq, hkv, d, t, seed=0, masked=False, layout="apart", extra=(0, 0), size=1.5):
    """q, k, v, q_ptr, k_ptr, mask.  layout: apart | together (keys and values of one projection) | heads (heads outermost) |
    odd (rows off a 16-byte boundary).  extra: rows in front of the first and behind the last scan."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: (torch.randn(*s, generator=g, device=DEV)).to(t)  # noqa: E731
    nq, nk = sum(lq) + sum(extra), sum(lk) + sum(extra)
    if layout == "heads":
        q, k, v = r(hq, nq, d).transpose(0, 1), r(hkv, nk, d).transpose(0, 1), r(hkv, nk, d).transpose(0, 1)
    elif layout == "odd":
        q, k, v = r(nq, hq, d + 3)[..., 1:d + 1], r(nk, hkv, d + 1)[..., :d], r(nk, hkv, d + 5)[..., 3:d + 3]
    elif layout == "together":
        kv = r(nk, 2, hkv, d)
        q, k, v = r(nq, hq, d), kv[:, 0], kv[:, 1]
    else:
        q, k, v = r(nq, hq, d), r(nk, hkv, d), r(nk, hkv, d)
    q = q * size if layout != "odd" else q
    mask = None
    if masked:
        mask = torch.rand(nk, generator=g, device=DEV) < 0.7
        k, v = k.clone() if layout == "apart" else k, v.clone() if layout == "apart" else v
        k[~mask] = float("nan")
        v[~mask] = float("inf")
    return q, k, v, ptr(lq, extra[0]), ptr(lk, extra[0]), mask


def both(args, train, scale=None, seed=3):
    q, k, v, q_ptr, k_ptr, mask = args
    if not train:
        return {"out": cross_attention(q, k, v, q_ptr, k_ptr, mask, scale)}, attention64(q, k, v, q_ptr, k_ptr, mask, scale)
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    out = cross_attention(q, k, v, q_ptr, k_ptr, mask, scale)
    d_out = torch.randn(out.shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(out.dtype)
    got = dict(zip(("d_q", "d_k", "d_v"), torch.autograd.grad(out, (q, k, v), d_out)), out=out)
    return got, attention64(q, k, v, q_ptr, k_ptr, mask, scale, d_out)


SHAPES = [
    # queries, keys, query heads, key heads, channels
    ([1], [1], 1, 1, 8),
    ([1], [700], 4, 4, 16),
    ([1, 1, 1, 1], [129, 1, 0, 4000], 8, 2, 64),
    ([63, 64, 65], [64, 65, 63], 2, 2, 32),
    ([127, 128, 129], [129, 127, 128], 2, 1, 64),
    ([5, 0, 300, 1], [1000, 50, 0, 2], 6, 3, 128),
    ([200], [3001], 3, 1, 40),
    ([17, 31], [513, 255], 8, 1, 24),
    ([2, 3], [5, 7], 5, 5, 3),
    ([33], [65], 2, 2, 1),
    ([400], [100], 4, 2, 96),
    ([1000], [70], 2, 2, 128),
    ([3], [20011], 2, 1, 64),
    ([130], [9000], 7, 1, 56),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("lq,lk,hq,hkv,d", SHAPES)
def test_forward_and_gradients(lq, lk, hq, hkv, d, dtype):
    args = inputs(lq, lk, hq, hkv, d, TYPES[dtype])
    check(*both(args, True))
    check(*both(args, False))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("layout", ["apart", "together", "heads", "odd"])
@pytest.mark.parametrize("masked", [False, True])
def test_layouts_and_masks(dtype, layout, masked):
    args = inputs([70, 0, 133], [301, 5, 150], 4, 2, 48, TYPES[dtype], masked=masked, layout=layout, extra=(3, 2))
    check(*both(args, True))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_rows_without_keys_and_of_no_scan(dtype):
    t = TYPES[dtype]
    q, k, v, q_ptr, k_ptr, _ = inputs([40, 200, 7], [300, 129, 0], 2, 2, 64, t, extra=(5, 9))
    mask = torch.ones(k.shape[0], dtype=torch.bool, device=DEV)
    mask[305:434] = False                                 # every key of the second scan
    for x in (k, v):
        x[~mask] = float("nan")
        x[:5] = float("inf")                              # rows of no scan, next to the first one's
        x[-9:] = float("nan")
    q[:5], q[-9:] = float("nan"), float("nan")
    got, want = both((q, k, v, q_ptr, k_ptr, mask), True)
    check(got, want)
    for name in got:
        assert torch.isfinite(got[name]).all()
    for rows in (slice(0, 5), slice(45, 252), slice(252, None)):
        assert not got["out"][rows].any() and not got["d_q"][rows].any()
    assert not got["d_k"][~mask].any() and not got["d_v"][~mask].any()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_the_next_scan_does_not_leak(dtype):
    """Tiles end inside a scan; what follows belongs to another one and may be anything."""
    t = TYPES[dtype]
    q, k, v, q_ptr, k_ptr, _ = inputs([30, 30], [70, 70], 2, 1, 64, t)
    k[70:], v[70:] = float("nan"), float("inf")
    q[30:] = float("nan")
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = cross_attention(*leaves, q_ptr, k_ptr)
    d_out = torch.ones_like(out)
    d_out[30:] = float("inf")
    grads = torch.autograd.grad(out, leaves, d_out)
    cut = [q[:30], k[:70], v[:70]]
    want = attention64(*cut, q_ptr[:2], k_ptr[:2], d_out=torch.ones_like(out[:30]))
    check({"out": out[:30], "d_q": grads[0][:30], "d_k": grads[1][:70], "d_v": grads[2][:70]}, want)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_large_scores_and_tiny_gradients(dtype):
    """Rows whose maximum moves from tile to tile by more than a type's range; gradients far below 1."""
    t = TYPES[dtype]
    q, k, v, q_ptr, k_ptr, _ = inputs([100], [1500], 2, 2, 64, t, size=6.0)
    k = (k * torch.linspace(0.1, 6.0, 1500, device=DEV).view(-1, 1, 1)).to(t)
    got, want = both((q, k, v, q_ptr, k_ptr, None), True)
    check(got, want)
    leaves = [x.detach().requires_grad_() for x in inputs([60], [5000], 2, 2, 64, t, size=0.2)[:3]]
    small = 2.0 ** -8
    out = cross_attention(*leaves, ptr([60]), ptr([5000]))
    d_out = (torch.randn(out.shape, device=DEV) * small).to(t)
    got = dict(zip(("d_q", "d_k", "d_v"), torch.autograd.grad(out, leaves, d_out)))
    want = attention64(*leaves, ptr([60]), ptr([5000]), d_out=d_out)
    check(got, want)
    for name in got:                                      # and not lost below the type's range on the way
        value = want[name][0]
        assert (got[name].double() - value).norm() <= 0.02 * value.norm() + 2.0 ** -25 * math.sqrt(value.numel()), name


@pytest.mark.parametrize("dtype", list(TYPES))
def test_scores_that_overflow_and_values_that_are_not_finite(dtype):
    t = TYPES[dtype]
    q, k, v, q_ptr, k_ptr, _ = inputs([5], [200], 1, 1, 16, t)
    k[150, 0] = float("nan")
    assert cross_attention(q, k, v, q_ptr, k_ptr).isnan().all()
    k[150, 0], q[:, 0] = 0.0, 0.0
    k[10:20, 0] = float("-inf")
    q[2, 0] = 1.0                                         # scores of -inf: no weight
    k[10:20, 0, 1:] = 0.0
    q[[0, 1, 3, 4], 0] = 1.0
    out = cross_attention(q, k, v, q_ptr, k_ptr)
    mask = torch.ones(200, dtype=torch.bool, device=DEV)
    mask[10:20] = False
    assert torch.allclose(out.float(), cross_attention(q, k, v, q_ptr, k_ptr, mask).float(), rtol=1e-2, atol=1e-2)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_scales(scale):
    args = inputs([50], [333], 2, 2, 32, torch.float32, size=0.5)
    check(*both(args, True, scale=scale))
    args = inputs([50], [333], 2, 2, 32, torch.bfloat16, size=0.5)
    check(*both(args, True, scale=scale))


def test_gradient_against_differences():
    q, k, v, q_ptr, k_ptr, _ = inputs([4], [9], 2, 1, 8, torch.float32)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    up = torch.randn(4, 2, 8, device=DEV)
    grads = torch.autograd.grad(cross_attention(*leaves, q_ptr, k_ptr), leaves, up)
    points = [x.detach().double() for x in leaves]
    value = lambda: (attention64(*points, q_ptr, k_ptr)["out"][0] * up.double()).sum().item()  # noqa: E731
    h = 1e-5                                              # h^2 / 6 of the third derivative, 2^-52 / h of the value, 2^-24 of float32
    for x, g in zip(points, grads):
        flat = x.view(-1)
        for i in range(0, flat.numel(), 7):
            keep = flat[i].item()
            flat[i] = keep + h
            above = value()
            flat[i] = keep - h
            below = value()
            flat[i] = keep
            assert abs((above - below) / (2 * h) - g.reshape(-1)[i].item()) < 2e-5


def test_only_some_gradients_are_wanted():
    q, k, v, q_ptr, k_ptr, _ = inputs([40], [90], 2, 2, 32, torch.bfloat16)
    full = [x.detach().requires_grad_() for x in (q, k, v)]
    all_ = torch.autograd.grad(cross_attention(*full, q_ptr, k_ptr).float().sum(), full)
    for i in range(3):
        some = [x.detach().requires_grad_(j == i) for j, x in enumerate((q, k, v))]
        one, = torch.autograd.grad(cross_attention(*some, q_ptr, k_ptr).float().sum(), some[i])
        assert torch.equal(one, all_[i])


@pytest.mark.parametrize("dtype", list(TYPES))
def test_same_bits_on_another_stream_and_in_graphs(dtype):
    t = TYPES[dtype]
    args = inputs([100, 3], [2000, 900], 4, 2, 64, t, masked=True)
    q, k, v = (x.detach().requires_grad_() for x in args[:3])
    d_out = torch.randn(q.shape, device=DEV).to(t)

    def step():
        out = cross_attention(q, k, v, *args[3:])
        return [out.detach()] + list(torch.autograd.grad(out, (q, k, v), d_out))

    first = step()
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))  # noqa: E731
    assert same(first, step())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beside = step()
    side.synchronize()
    assert same(first, beside)
    graphs, results = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            results.append(step())
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert same(first, results[0]) and same(first, results[1])
    sphconv.check_status()


def test_rows_of_a_sparse_tensor():
    shape, B = [4, 5, 8], 3
    idx = torch.tensor([[b, i % 4, i % 5, i % 8] for b in (0, 2) for i in range(20 + b)], dtype=torch.int32, device=DEV)
    x = sphconv.SparseConvTensor(torch.randn(42, 32, device=DEV), shape, B, indices=idx)
    k_ptr = scan_rows(x)
    assert k_ptr.tolist() == [0, 20, 20, 42] and k_ptr.dtype == torch.int32
    rows = x.feature.view(42, 4, 8)
    q = torch.randn(6, 4, 8, device=DEV)
    got = cross_attention(q, rows, rows, ptr([2, 2, 2]), k_ptr)
    check({"out": got}, attention64(q, rows, rows, ptr([2, 2, 2]), k_ptr))


def test_pointers_out_of_order_or_range_are_reported():
    q, k, v, q_ptr, k_ptr, _ = inputs([10, 10], [30, 30], 2, 2, 32, torch.float32)
    for bad in ([0, 40, 30], [0, 30, 61], [-1, 30, 60]):
        cross_attention(q, k, v, q_ptr, torch.tensor(bad, dtype=torch.int32, device=DEV))
        with pytest.raises(RuntimeError, match="index"):
            sphconv.check_status()
    cross_attention(q, k, v, q_ptr, k_ptr)
    sphconv.check_status()


def test_no_rows():
    q, k, v, q_ptr, k_ptr, _ = inputs([0, 0], [30, 30], 2, 2, 32, torch.bfloat16)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = cross_attention(*leaves, q_ptr, k_ptr)
    assert out.shape == (0, 2, 32)
    assert all(not g.any() for g in torch.autograd.grad(out.sum(), leaves))
    q, k, v, q_ptr, k_ptr, _ = inputs([4, 3], [0, 0], 2, 2, 32, torch.bfloat16)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = cross_attention(*leaves, q_ptr, k_ptr)
    assert not out.any() and all(not g.any() for g in torch.autograd.grad(out.sum(), leaves))


def test_refusals():
    q, k, v, q_ptr, k_ptr, _ = inputs([4], [9], 2, 2, 8, torch.float32)
    mask = torch.ones(9, dtype=torch.bool, device=DEV)
    ok = dict(q=q, k=k, v=v, q_ptr=q_ptr, k_ptr=k_ptr)
    for change in (dict(q=q.double()), dict(q=q.half()), dict(k=k[:8]), dict(q=q[..., :4]), dict(q=q.repeat(1, 2, 1)[:, :3]),
                   dict(q=q[0]), dict(q_ptr=q_ptr.long()), dict(q_ptr=q_ptr[:1]), dict(k_ptr=torch.cat([k_ptr, k_ptr])),
                   dict(key_mask=mask[:8]), dict(key_mask=mask.int()), dict(q=q.cpu()), dict(k_ptr=k_ptr.cpu()), dict(scale=math.nan),
                   dict(q=torch.ones(4, 2, 129, device=DEV), k=torch.ones(9, 2, 129, device=DEV), v=torch.ones(9, 2, 129, device=DEV))):
        with pytest.raises(RuntimeError):
            cross_attention(**dict(ok, **change))
    leaf = q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(cross_attention(leaf, k, v, q_ptr, k_ptr).sum(), leaf, create_graph=True)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("hq,hkv,d", [(6, 2, 128), (4, 4, 40), (5, 1, 64)])
def test_many_scans_of_very_different_lengths(hq, hkv, d, dtype):
    """More scans than a warp has lanes, one of them with most of the keys and one with most of the queries."""
    lq = [(7 * i) % 5 for i in range(75)]
    lk = [(11 * i) % 9 for i in range(75)]
    lk[40], lk[74], lq[33], lq[50] = 5000, 700, 400, 130
    got, want = both(inputs(lq, lk, hq, hkv, d, TYPES[dtype], seed=9, extra=(3, 2)), True)
    check(got, want)
    sphconv.check_status()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_one_scan_of_most_keys_and_few_rows_is_split(dtype):
    """A walk in as many parts as there are, on either side."""
    check(*both(inputs([3, 90], [20000, 5], 2, 2, 64, TYPES[dtype], seed=11), True))
    check(*both(inputs([9000, 2], [30, 3], 2, 1, 64, TYPES[dtype], seed=12), True))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_keys_that_are_the_values_and_shared_heads(dtype):
    """One tensor as keys and values, and one head expanded to all: their gradients are the sums."""
    t = TYPES[dtype]
    q, k, _, q_ptr, k_ptr, _ = inputs([70, 9], [200, 31], 4, 4, 32, t, seed=13)
    d_out = torch.randn(q.shape, device=DEV).to(t)
    rows = k.detach().requires_grad_()
    got, = torch.autograd.grad(cross_attention(q, rows, rows, q_ptr, k_ptr), rows, d_out)
    want = attention64(q, k, k, q_ptr, k_ptr, d_out=d_out)
    # each is rounded by itself, and their sum once more
    half = torch.finfo(t).eps / 2
    total = want["d_k"][0] + want["d_v"][0]
    check({"rows": got}, {"rows": (total, want["d_k"][1] + want["d_v"][1] + half * total.abs())})
    one = k[:, :1].detach().requires_grad_()
    k4 = one.expand(-1, 4, -1)
    out = cross_attention(q, k4, k4, q_ptr, k_ptr)
    k4 = k4.detach().contiguous()
    want = attention64(q, k4, k4, q_ptr, k_ptr, d_out=d_out)
    check({"out": out.detach()}, {"out": want["out"]})
    got, = torch.autograd.grad(out, one, d_out)
    parts = torch.cat([want["d_k"][0], want["d_v"][0]], 1)
    total = parts.sum(1, keepdim=True)
    # eight terms: their sums are rounded seven times at most, each time half a step of at most the terms' sizes together
    bound = (want["d_k"][1] + want["d_v"][1]).sum(1, keepdim=True) + 8 * half * parts.abs().sum(1, keepdim=True)
    check({"one": got}, {"one": (total, bound)})


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_rows_far_apart(dtype):
    """Offsets past 2^31 elements."""
    t, n, d, far = TYPES[dtype], 75, 64, 1 << 25
    store = torch.zeros(n * far, dtype=t, device=DEV)
    q, k, v, q_ptr, k_ptr, _ = inputs([40, 3], [50, 25], 2, 1, d, t, seed=14)
    far_k = store.as_strided((n, 1, d), (far, d, 1))
    far_v = store.as_strided((n, 1, d), (far, d, 1), 4 * d)
    far_k.copy_(k)
    far_v.copy_(v)
    assert (n - 1) * far > 2 ** 31
    check(*both((q, far_k, far_v, q_ptr, k_ptr, None), True))
    for lengths in ([1, 1], [300, 0]):
        q = torch.randn(sum(lengths), 2, d, device=DEV).to(t)
        args = (q, far_k, far_v, ptr(lengths), k_ptr, None)
        check(*both(args, False))


def test_more_values_than_31_bits():
    n = (1 << 23) + 1000                        # times 4 heads of 64 channels
    kv = torch.randn(400, 2, 4, 64, device=DEV).bfloat16()
    k, v = (torch.zeros(n, 4, 64, dtype=torch.bfloat16, device=DEV) for _ in "kv")
    k[-400:], v[-400:] = kv[:, 0], kv[:, 1]
    q = torch.randn(3, 4, 64, device=DEV).bfloat16()
    d_out = torch.randn_like(q)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    k_ptr = torch.tensor([0, n - 400, n], dtype=torch.int32, device=DEV)
    out = cross_attention(*leaves, ptr([0, 3]), k_ptr)
    got = dict(zip(("d_q", "d_k", "d_v"), torch.autograd.grad(out, leaves, d_out)), out=out.detach())
    assert not got["d_k"][:-400].any() and not got["d_v"][:-400].any()
    got["d_k"], got["d_v"] = got["d_k"][-400:], got["d_v"][-400:]
    check(got, attention64(q.detach(), kv[:, 0], kv[:, 1], ptr([3]), ptr([400]), d_out=d_out))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("layout", ["apart", "odd"])
def test_gradients_that_are_not_finite_where_nothing_is_read(dtype, layout):
    """NaN on its way back to queries without keys stays away from everything: they have zeros, and so do their scan's keys."""
    q, k, v, q_ptr, k_ptr, _ = inputs([40, 200, 7], [300, 129, 0], 2, 2, 64, TYPES[dtype], layout=layout)
    mask = torch.ones(k.shape[0], dtype=torch.bool, device=DEV)
    mask[300:] = False                                    # every key of the second scan
    mask[7] = False
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = cross_attention(*leaves, q_ptr, k_ptr, mask)
    d_out = torch.randn(out.shape, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).to(out.dtype)
    want = attention64(q, k, v, q_ptr, k_ptr, mask, d_out=d_out)
    d_out[40:] = float("nan")
    d_out[100:120] = float("inf")
    got = dict(zip(("d_q", "d_k", "d_v"), torch.autograd.grad(out, leaves, d_out)), out=out.detach())
    check(got, want)
    assert not got["d_q"][40:].any() and not got["d_k"][~mask].any() and not got["d_v"][~mask].any()
    # and in a scan with keys, whose gradients it spoils, those of what is no key are zeros all the same
    d_out[3] = float("nan")
    _, d_k, d_v = torch.autograd.grad(cross_attention(*leaves, q_ptr, k_ptr, mask), leaves, d_out)
    assert not d_k[~mask].any() and not d_v[~mask].any()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_one_query_row_for_all_and_a_head_for_each(dtype):
    """Queries broadcast over rows and heads (strides of zero), and more query heads of a key head than a tile has rows."""
    t = TYPES[dtype]
    _, k, v, q_ptr, k_ptr, _ = inputs([90, 1, 60], [70, 200, 31], 2, 2, 64, t, seed=21)
    one = torch.randn(1, 1, 64, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).to(t)
    check(*both((one.expand(151, 2, 64), k, v, q_ptr, k_ptr, None), True))
    q, k, v, q_ptr, k_ptr, _ = inputs([3, 0, 2], [70, 200, 31], 300, 1, 48, t, seed=22)
    check(*both((q, k, v, q_ptr, k_ptr, None), True))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_a_thousand_scans(dtype):
    lq, lk = [i % 3 for i in range(1000)], [i % 4 * 5 for i in range(1000)]
    check(*both(inputs(lq, lk, 2, 1, 32, TYPES[dtype], seed=23), True))
    check(*both(inputs([1] * 1000, lk, 2, 2, 64, TYPES[dtype], seed=24), False))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d", [8, 64, 128])
@pytest.mark.parametrize("at", [5, 20000, 39999])
def test_one_key_above_a_long_flat_rest(d, at, dtype):
    """What a key far below the largest one gets is little, but tens of thousands of them are not, and their values are all the same: what is
    lost of them does not average out.  Query i has one key that is 10 + i above the others, whose scores are zero."""
    t, n, rows = TYPES[dtype], 40000, 14
    q, k = torch.zeros(rows, 1, d, device=DEV), torch.zeros(n, 1, d, device=DEV)
    q[:, 0, 0] = 10.0 + torch.arange(rows, device=DEV)    # exact in every type, and so are the scores
    k[at, 0, 0] = 1.0
    v = torch.ones(n, 1, d, device=DEV)
    v[at] = 0.0
    check(*both((q.to(t), k.to(t), v.to(t), ptr([rows]), ptr([n]), None), True, scale=1.0))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d", [8, 64, 128])
def test_a_key_far_below_another_for_many_queries(d, dtype):
    """The value of a key that tens of thousands of queries give the same little weight: what its gradient loses does not average out.  The
    two keys of scan i are 14 + i apart, and the gradient is 40000 times e^-(14 + i).

    Not of d_q and d_k: `out`, here e^-(14 + i) in all channels, is rounded in steps of 2^-24 in float16, delta is the sum of d of them, and
    off by up to d 2^-25 where it is itself no more; the bounds take the rounding for one of half a step relative to `out`."""
    t, n, scans = TYPES[dtype], 40000, 12
    q, k = torch.zeros(scans * n, 1, d, device=DEV), torch.zeros(2 * scans, 1, d, device=DEV)
    q[:, 0, 0] = 14.0 + torch.arange(scans, device=DEV).repeat_interleave(n)
    k[::2, 0, 0] = 1.0
    v = torch.ones(2 * scans, 1, d, device=DEV)
    v[::2] = 0.0
    q, k, v = (x.to(t).requires_grad_() for x in (q, k, v))
    q_ptr, k_ptr = ptr([n] * scans), ptr([2] * scans)
    out = cross_attention(q, k, v, q_ptr, k_ptr, scale=1.0)
    d_out = torch.ones_like(out)
    d_v, = torch.autograd.grad(out, v, d_out)
    check({"out": out, "d_v": d_v}, attention64(q, k, v, q_ptr, k_ptr, scale=1.0, d_out=d_out))


def test_a_walk_longer_than_a_wait_may_take():
    """A tile of rows keeps its place while all of its scan is walked over, and what waits for that place waits as long: 62500 steps of
    about half a microsecond are three times the limit of a wait in the library for tests (10 ms), where this is no failure either.
    Results are those of the shipped library, whose limit is 0.2 s.  300 tiles of keys give some of the blocks three of them; the scans without
    rows make the walk look short to the host, so that it is not split into parts."""
    if not os.path.exists(sph_build.HOOKS_LIB):
        pytest.skip("test-hooks library not built (python -m sphconv_b200.build)")
    B, heads, d, nq, nk = 6000, 64, 8, 62500, 38400
    g = torch.Generator(device=DEV).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()  # noqa: E731
    q, k, v, d_out = r(nq, heads, d), torch.zeros(nk, 1, d, device=DEV).bfloat16(), r(nk, 1, d), r(nq, heads, d)
    ends = [torch.zeros(B + 1, dtype=torch.int32, device=DEV) for _ in "qk"]
    for e, n in zip(ends, (nq, nk)):
        e[3001:] = n
    lse = torch.full((nq, heads), math.log2(nk), device=DEV)            # scores of zero
    out = v.float().mean(0).bfloat16().expand(nq, heads, d).contiguous()
    args = C.Attention(B, heads, 1, d, C.SPH_BF16, 1.0, nq, nk, C.ptr(q), C.ptr(k), C.ptr(v), heads * d, d, d, d, d, d,
                       C.ptr(ends[0]), C.ptr(ends[1]), None)
    results = []
    for lib in (C.lib(), ctypes.CDLL(sph_build.HOOKS_LIB)):
        for name in ("sph_attention_scratch_bytes", "sph_attention_backward"):
            getattr(lib, name).restype, getattr(lib, name).argtypes = C.SIGNATURES[name]
        size = lib.sph_attention_scratch_bytes(ctypes.byref(args), 1)
        assert size == 2 * (B + 2) * 32 + 2 * nq * heads * 4            # plans, delta and counts, and no parts
        scratch = torch.empty(size, dtype=torch.uint8, device=DEV)
        dk, dv, status = torch.full_like(k, 7.0), torch.full_like(v, 7.0), torch.zeros(1, dtype=torch.int32, device=DEV)
        assert lib.sph_attention_backward(ctypes.byref(args), C.ptr(d_out), C.ptr(out), C.ptr(lse), C.ptr(scratch), None, C.ptr(dk),
                                          C.ptr(dv), C.ptr(status), C.stream_ptr(torch.device(DEV))) == 0
        torch.cuda.synchronize()
        assert int(status.item()) == 0
        results.append((dk, dv))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    # every key has a weight of 1 / nk, to 2^-9, from every query: the sum's terms are 4 million of about 1 / nk
    want = d_out.double().sum((0, 1)) / nk
    size = d_out.double().abs().sum((0, 1)) / nk
    assert ((results[0][1].double()[:, 0] - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -9 + 2.0 ** -12) * size).all()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_gradients_of_scores_that_are_no_numbers(dtype):
    """A NaN in a query reaches what that query has a part in: its own result and gradient, and its scan's and key head's keys and values."""
    q, k, v, q_ptr, k_ptr, _ = inputs([140, 9], [200, 31], 4, 2, 64, TYPES[dtype], seed=25)
    q[3, 1, 5] = float("nan")                             # head 1 reads key head 0
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = cross_attention(*leaves, q_ptr, k_ptr)
    d_q, d_k, d_v = torch.autograd.grad(out, leaves, torch.ones_like(out))
    here = torch.zeros(149, 4, dtype=torch.bool, device=DEV)
    here[3, 1] = True
    assert out[here].isnan().all() and torch.isfinite(out[~here]).all() and d_q[here].isnan().all() and torch.isfinite(d_q[~here]).all()
    for g in (d_k, d_v):
        assert g[:200, 0].isnan().all() and torch.isfinite(g[:200, 1]).all() and torch.isfinite(g[200:]).all()
