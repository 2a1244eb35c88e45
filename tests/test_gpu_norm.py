"""Norms before and after a block with gate and residual scale, against the formulas in 64 bits and their 64-bit derivatives."""
import math

import pytest
import torch

import sphconv_b200 as sphconv
from sphconv_b200.norm import ResidualNorm, RowNorm, residual_norm, row_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
NAMES = ("block", "residual", "gate", "weight", "bias", "scale", "next_weight", "next_bias")


def reference(v, eps, center, fixed=False):
    """(out, normed) in 64 bits from a dict of leaves (None: not given); fixed: the norms' statistics taken for constants."""
    hold = lambda x: x.detach() if fixed else x  # noqa: E731
    def norm(x, w, b):
        if w is None:
            return x
        d = x - hold(x.mean(-1, keepdim=True)) if center else x
        y = d / hold(torch.sqrt((d * d).mean(-1, keepdim=True) + eps)) * w
        return y if b is None else y + b

    out = v["residual"]
    if v["block"] is not None:
        inner = norm(v["block"], v["weight"], v["bias"])
        if v["gate"] is not None:
            inner = inner * torch.sigmoid(v["gate"])
        if v["scale"] is not None:
            inner = inner * v["scale"]
        out = out + inner
    return out, None if v["next_weight"] is None else norm(out, v["next_weight"], v["next_bias"])


def make(n, c, t, given, seed=0, param_type=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    v = {"block": r(n, c).to(t), "residual": (2 * r(n, c)).to(t), "gate": r(n, 1).to(t) if "gate_row" in given else r(n, c).to(t)}
    for name, mean in (("weight", 1.0), ("bias", 0.0), ("scale", 0.5), ("next_weight", 1.0), ("next_bias", 0.0)):
        v[name] = (mean + 0.3 * r(c)).to(param_type)
    return {k: (x if k in given or k == "residual" or (k == "gate" and "gate_row" in given) else None) for k, x in v.items()}


def close(got, want, t, terms, what, parts=None):
    """A value rounded once to t from float32 arithmetic of `terms` terms: half a step of t, and of float32 for each term of the
    sums behind it, which come to the size of the largest value of its row (or column).
    parts: a value of the size of what the result is the difference of.  The gradient of a norm is inv (d - n mean(d n)): both terms
    are of the size of inv d, which is its gradient with the statistics fixed, each is rounded to 2^-24 of that, and a row of one
    channel cancels to eps / (x^2 + eps) of it."""
    got, want = got.double(), want.double()
    size = want.abs().amax(-1, keepdim=True).clamp_min(1e-30) if want.dim() > 1 else want.abs().max().clamp_min(1e-30)
    if parts is not None:
        size = torch.maximum(size, parts.abs().amax(-1, keepdim=True))
    tol = torch.finfo(t).eps / 2 * want.abs() + (16 + terms) * torch.finfo(torch.float32).eps / 2 * size + \
        (torch.finfo(t).smallest_normal * torch.finfo(t).eps if t == torch.float16 else 0)      # half a step below the normal range
    bad = ((got - want).abs() - tol).max().item()
    assert bad <= 0, (what, bad, (got - want).abs().max().item())


CASES = [
    # n, c, type, given, center
    (1, 1, "fp32", ("block", "weight", "next_weight"), False),
    (7, 3, "bf16", ("block", "weight", "gate", "scale", "next_weight"), False),
    (33, 16, "fp16", ("block", "weight", "bias", "gate_row", "next_weight", "next_bias"), True),
    (200, 128, "fp16", ("block", "weight", "bias", "next_weight", "next_bias"), True),
    (1031, 64, "bf16", ("block", "weight", "gate_row", "scale", "next_weight"), False),
    (257, 100, "fp32", ("block", "weight", "bias", "gate", "scale", "next_weight", "next_bias"), True),
    (65, 101, "fp16", ("block", "weight", "gate", "next_weight"), False),
    (130, 257, "bf16", ("block", "gate_row", "scale", "next_weight"), False),
    (19, 2048, "bf16", ("block", "weight", "gate", "scale", "next_weight"), False),
    (9, 1000, "fp32", ("block", "weight", "gate", "scale"), True),
    (5, 4097, "fp32", ("block", "weight", "gate", "scale", "next_weight"), False),
    (5, 8192, "fp16", ("block", "weight", "gate_row", "next_weight", "next_bias"), True),
    (300, 40, "bf16", ("next_weight",), False),
    (300, 72, "fp32", ("next_weight", "next_bias"), True),
    (5, 16, "fp32", ("block",), False),
    (100000, 8, "bf16", ("block", "weight", "gate", "scale", "next_weight"), False),
]


@pytest.mark.parametrize("n,c,dtype,given,center", CASES)
def test_forward_and_gradients(n, c, dtype, given, center):
    t = TYPES[dtype]
    v = {k: None if x is None else x.requires_grad_() for k, x in make(n, c, t, given).items()}
    if v["block"] is None:
        out, normed = None, row_norm(v["residual"], v["next_weight"], v["next_bias"], 1e-5, center)
    else:
        out, normed = residual_norm(v["block"], v["residual"], v["weight"], v["bias"], gate=v["gate"], scale=v["scale"],
                                    next_weight=v["next_weight"], next_bias=v["next_bias"], eps=1e-5, center=center)
    v64 = {k: None if x is None else x.detach().double().requires_grad_() for k, x in v.items()}
    out64, normed64 = reference(v64, 1e-5, center)
    log = int(math.log2(c)) + 1
    if out is not None:
        close(out, out64, t, log, "out")
    if normed is not None:
        close(normed, normed64, t, log, "normed")
    g = torch.Generator(device=DEV).manual_seed(9)
    pairs = [(a, b, torch.randn(n, c, generator=g, device=DEV).to(t)) for a, b in ((out, out64), (normed, normed64)) if a is not None]
    names = [k for k in NAMES if v[k] is not None]
    grads = torch.autograd.grad([p[0] for p in pairs], [v[k] for k in names], [p[2] for p in pairs])
    wants = torch.autograd.grad([p[1] for p in pairs], [v64[k] for k in names], [p[2].double() for p in pairs])
    held = [x for x in reference(v64, 1e-5, center, fixed=True) if x is not None]
    parts = torch.autograd.grad(held[-len(pairs):], [v64[k] for k in names], [p[2].double() for p in pairs])
    if v["gate"] is not None and v["gate"].shape != v["residual"].shape:
        # A row's gate has the sum over channels of total_c j_c, where total is the gradient of `out`, which is the residual's, and j_c that
        # of out_c in the logit.  total_c is off by what `close` allows a residual, of the size of the row's largest; the sum and j_c round
        # to 2^-24 of |total_c j_c| a few times: altogether of the size of that largest value times the sum of |j_c|.
        wide = dict(v64, gate=v64["gate"].detach().expand(n, c).contiguous().requires_grad_())
        j, = torch.autograd.grad(reference(wide, 1e-5, center)[0].sum(), wide["gate"])
        at = names.index("residual")
        largest = torch.maximum(wants[at].abs(), parts[at].abs()).amax(-1, keepdim=True)
        parts = [largest * j.abs().sum(-1, keepdim=True) if k == "gate" else x for k, x in zip(names, parts)]
    for k, got, want, part in zip(names, grads, wants, parts):
        assert got.dtype == v[k].dtype and got.shape == v[k].shape
        if k in ("block", "residual", "gate"):
            close(got, want, t, 4 * log, "d_" + k, part)
        else:       # sums of n values of either sign: each 32-bit partial sum rounds to the size that sums of its values have
            scale = max(1.0, want.abs().max().item())
            assert (got.double() - want).abs().max().item() <= 2 ** -24 * 64 * math.sqrt(n) * scale, ("d_" + k)


def test_gradients_against_differences():
    v = {k: None if x is None else x.double() for k, x in make(4, 6, torch.float32, NAMES).items()}
    leaves = {k: x.float().requires_grad_() for k, x in v.items()}
    up = [torch.randn(4, 6, device=DEV) for _ in range(2)]
    out = residual_norm(leaves["block"], leaves["residual"], leaves["weight"], leaves["bias"], gate=leaves["gate"], scale=leaves["scale"],
                        next_weight=leaves["next_weight"], next_bias=leaves["next_bias"], eps=1e-5, center=True)
    grads = torch.autograd.grad(list(out), [leaves[k] for k in NAMES], up)
    value = lambda: sum((a * b.double()).sum() for a, b in zip(reference(v, 1e-5, True), up)).item()  # noqa: E731
    h = 1e-5                                              # central differences: h^2 / 6 of the third derivative, 2^-52 / h of the value
    for k, g in zip(NAMES, grads):
        flat = v[k].view(-1)
        for i in range(0, flat.numel(), 5):
            keep = flat[i].item()
            flat[i] = keep + h
            up_ = value()
            flat[i] = keep - h
            down = value()
            flat[i] = keep
            assert abs((up_ - down) / (2 * h) - g.view(-1)[i].item()) < 1e-4, (k, i)


@pytest.mark.parametrize("param_type", [torch.float16, torch.bfloat16])
def test_parameters_of_16_bits(param_type):
    v = make(50, 64, torch.bfloat16, NAMES, param_type=param_type)
    v = {k: x.requires_grad_() for k, x in v.items()}
    out, normed = residual_norm(v["block"], v["residual"], v["weight"], v["bias"], gate=v["gate"], scale=v["scale"],
                                next_weight=v["next_weight"], next_bias=v["next_bias"], center=True)
    out64, normed64 = reference({k: x.detach().double() for k, x in v.items()}, 1e-6, True)
    close(out, out64, torch.bfloat16, 7, "out")
    close(normed, normed64, torch.bfloat16, 7, "normed")
    d = torch.autograd.grad([out, normed], [v["weight"], v["next_bias"]], [torch.ones_like(out), torch.ones_like(out)])
    assert all(x.dtype == param_type for x in d)
    assert torch.equal(d[1], torch.full_like(d[1], 50.0))


def test_one_output_only_and_no_rows():
    v = {k: x.requires_grad_() for k, x in make(20, 32, torch.float32, NAMES).items()}
    call = lambda: residual_norm(v["block"], v["residual"], v["weight"], v["bias"], gate=v["gate"], scale=v["scale"],  # noqa: E731
                                 next_weight=v["next_weight"], next_bias=v["next_bias"], center=True)
    a = torch.autograd.grad(call()[1].sum(), [v["block"], v["next_bias"]])
    b = torch.autograd.grad(list(call()), [v["block"], v["next_bias"]], [torch.zeros_like(v["block"]), torch.ones_like(v["block"])])
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    d_out = torch.autograd.grad(call()[0].sum(), [v["next_weight"], v["residual"]], allow_unused=True)
    assert torch.equal(d_out[1], torch.ones_like(d_out[1])) and not d_out[0].any()
    empty = torch.empty(0, 32, device=DEV, requires_grad=True)
    w = torch.ones(32, device=DEV, requires_grad=True)
    y = row_norm(empty, w)
    assert y.shape == (0, 32)
    d = torch.autograd.grad(y.sum(), [empty, w])
    assert d[0].shape == (0, 32) and torch.equal(d[1], torch.zeros_like(w))


def test_rows_that_are_not_finite_stay_alone():
    x = torch.randn(9, 64, device=DEV, dtype=torch.bfloat16)
    x[3, 5], x[6, 0] = float("nan"), float("inf")
    y = row_norm(x, torch.ones(64, device=DEV))
    assert torch.isfinite(y[[0, 1, 2, 4, 5, 7, 8]]).all() and y[3].isnan().all() and y[6, 0].isnan()


def test_unaligned_rows_and_parameters_give_the_same():
    x, w = torch.randn(40, 64, device=DEV), torch.rand(64, device=DEV)
    away = torch.empty(40 * 64 + 1, device=DEV)[1:].view(40, 64).copy_(x)
    w_away = torch.empty(65, device=DEV)[1:].copy_(w)
    assert torch.allclose(row_norm(x, w), row_norm(away, w), rtol=1e-6) and torch.equal(row_norm(x, w_away), row_norm(away, w))


def test_same_bits_every_time_on_any_stream_and_in_a_graph():
    v = {k: x.requires_grad_() for k, x in make(3000, 72, torch.bfloat16, NAMES).items()}
    up = [torch.randn(3000, 72, device=DEV, dtype=torch.bfloat16) for _ in range(2)]

    def step():
        out = residual_norm(v["block"], v["residual"], v["weight"], v["bias"], gate=v["gate"], scale=v["scale"],
                            next_weight=v["next_weight"], next_bias=v["next_bias"], center=True)
        return [x.detach() for x in out] + list(torch.autograd.grad(list(out), [v[k] for k in NAMES], up))

    first = step()
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beside = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, beside))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, captured))


def test_modules_in_a_sequential():
    B, shape = 1, [4, 5, 8]
    idx = torch.tensor([[0, i % 4, i % 5, i % 8] for i in range(20)], dtype=torch.int32, device=DEV)
    x = sphconv.SparseConvTensor(torch.randn(20, 8, device=DEV), shape, B, indices=idx)
    net = sphconv.Sequential(RowNorm(8), sphconv.SubMConv3d(8, 16, 3), RowNorm(16, center=True)).to(DEV)
    y = net(x)
    assert y.feature.shape == (20, 16)
    layer = ResidualNorm(16, initial_scale=0.1).to(DEV)
    out, normed = layer(y.feature, y.feature.detach().clone())
    (out.sum() + normed.sum()).backward()
    assert all(p.grad is not None for p in list(net.parameters()) + list(layer.parameters()))


def test_refusals():
    x, w = torch.randn(6, 8, device=DEV), torch.ones(8, device=DEV)
    for call in (lambda: row_norm(x.t(), w[:6]), lambda: row_norm(x, w[:7]), lambda: row_norm(x.double(), w), lambda: row_norm(x.cpu(), w.cpu()),
                 lambda: row_norm(x, w.double()), lambda: row_norm(x, w, eps=-1.0), lambda: row_norm(torch.ones(2, 8193, device=DEV), torch.ones(8193, device=DEV)),
                 lambda: residual_norm(x, x.half(), w), lambda: residual_norm(x, x[:5], w), lambda: residual_norm(x, x, None, w),
                 lambda: residual_norm(x, x, w, gate=x[:, :2].contiguous()), lambda: residual_norm(x, x, w, next_bias=w)):
        with pytest.raises(RuntimeError):
            call()
    leaf = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(row_norm(leaf, w).sum(), leaf, create_graph=True)


@pytest.mark.parametrize("n,c,dtype,given,center", [
    # as many values a thread and threads a row as there are kinds of either, with rows enough that blocks have several
    (700, 1024, "fp32", ("block", "weight", "gate", "scale", "next_weight"), False),
    (500, 2048, "fp32", ("block", "weight", "bias", "gate", "scale", "next_weight", "next_bias"), True),
    (400, 4096, "fp32", ("block", "weight", "gate_row", "scale", "next_weight"), False),
    (400, 8192, "fp32", ("block", "weight", "bias", "gate", "scale", "next_weight", "next_bias"), True),
    (400, 8190, "bf16", ("block", "weight", "gate", "scale", "next_weight", "next_bias"), False),
    (400, 4104, "bf16", ("block", "weight", "gate_row", "scale", "next_weight"), False),
    (500, 1999, "fp16", ("block", "weight", "bias", "gate", "next_weight", "next_bias"), True),
    (500, 2100, "bf16", ("block", "gate", "scale", "next_weight"), False),
    (450, 3001, "fp32", ("block", "weight", "gate_row", "scale", "next_weight"), False),
])
def test_wide_rows(n, c, dtype, given, center):
    test_forward_and_gradients(n, c, dtype, given, center)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_gates_at_their_ends(dtype):
    """Logits whose exponential is zero or infinite: a gate of exactly one or zero, and gradients without NaN."""
    t = TYPES[dtype]
    end = 6e4 if t == torch.float16 else 3e38
    gate = torch.tensor([[-end], [-200.0], [0.0], [200.0], [end]], device=DEV).to(t).expand(5, 40).contiguous().requires_grad_()
    block, residual = torch.full((5, 40), 2.0, device=DEV).to(t).requires_grad_(), torch.ones(5, 40, device=DEV).to(t)
    out, _ = residual_norm(block, residual, gate=gate)
    assert torch.equal(out[:, 0].float(), torch.tensor([1.0, 1.0, 2.0, 3.0, 3.0], device=DEV))
    d_block, d_gate = torch.autograd.grad(out.float().sum(), (block, gate))
    assert torch.equal(d_block[:, 0].float(), torch.tensor([0.0, 0.0, 0.5, 1.0, 1.0], device=DEV))
    assert torch.equal(d_gate[:, 0].float(), torch.tensor([0.0, 0.0, 0.5, 0.0, 0.0], device=DEV))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("c", [64, 2048])
def test_layer_norm_of_rows_whose_values_are_all_alike(c, dtype):
    """Sums of 2^k equal values are exact, and so is their mean: every deviation is zero, far from zero as near to it, and what it is
    multiplied with, 1 / sqrt(eps), must not bring anything back."""
    t = TYPES[dtype]
    x = torch.tensor([0.0, 0.1, -3.3, 1000.1, 30011.0], device=DEV).to(t)[:, None].expand(5, c).contiguous().requires_grad_()
    w, b = torch.full((c,), 1.5, device=DEV, requires_grad=True), torch.linspace(-1, 1, c, device=DEV, requires_grad=True)
    y = row_norm(x, w, b, center=True)
    assert torch.equal(y, b.detach().to(t).expand(5, c))
    d_w, = torch.autograd.grad(y.float().square().sum(), w)
    assert not d_w.any()
    gate = torch.zeros(5, 1, device=DEV, dtype=t)
    out, normed = residual_norm(x, x.detach(), w, b, gate=gate, next_weight=w, center=True)
    want = (x.detach().float() + 0.5 * b.detach()).to(t)
    assert torch.equal(out, want)
    d_w, = torch.autograd.grad(out.float().sum(), w)
    assert not d_w.any()
