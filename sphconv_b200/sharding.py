"""Batch sharding across GPUs: scans are independent (a scan never interacts with another one: tiles are
shared across the batch only as a list index, row ids and z_ptr are per-tensor prefix sums,
src/sphconv/rules.cu:72-80,204-227), so rank r of R takes a contiguous slice of the batch, builds its own
SparseConvTensor (its z_ptr starts at 0) and runs the path locally.  Forward needs no collective; training
adds ONE all-reduce over a flat fp32 buffer holding every layer's weight gradient."""
import math
from typing import Iterable, List, Optional, Sequence, Tuple, Union

import torch


def shard_range(n_scans: int, world: int, rank: int) -> Tuple[int, int]:
    """[first, last) scan ids of `rank`; sizes differ by at most one."""
    if world < 1 or not (0 <= rank < world):
        raise ValueError("bad world/rank %d/%d" % (world, rank))
    base, extra = divmod(n_scans, world)
    first = rank * base + min(rank, extra)
    return first, first + base + (1 if rank < extra else 0)


def slice_batch(z_idx: torch.Tensor, z_ptr: torch.Tensor, feature: torch.Tensor, first: int, last: int):
    """Scans [first, last) of a range-voxel batch as a self-contained batch (z_ptr re-based to start at 0)."""
    B, H, W = z_ptr.shape
    flat = z_ptr.reshape(B, -1)
    row0 = 0 if first == 0 else int(flat[first - 1, -1])
    row1 = row0 if last == first else int(flat[last - 1, -1])
    zp = (z_ptr[first:last] - row0).contiguous()
    return z_idx[row0:row1].contiguous(), zp, feature[row0:row1].contiguous()


class GradBuffer:
    """One flat fp32 buffer that holds the gradient of every parameter of a model, written in place by the
    backward kernels and all-reduced in place with ONE collective.

    The weight-gradient kernels accumulate in fp32 (the reference sums fp32 per-tile partials,
    src/sphconv/rule_conv.cu:483-484,517).  Handing that result to autograd as `.grad` of a bf16/fp16 parameter
    rounds each rank's contribution to 8 or 11 mantissa bits BEFORE the cross-rank sum; here each convolution
    writes its fp32 result straight into its slice of this buffer (the parameter gets no `.grad` from autograd),
    the buffer is summed over the ranks as fp32, and `to_grads()` rounds once at the end.

        gb = GradBuffer(net.parameters())          # attaches a slice to every parameter
        gb.zero(); loss.backward(); gb.all_reduce(); gb.to_grads(); optimizer.step()

    Works with CPU tensors too (host-side tests over gloo)."""

    def __init__(self, params: Iterable[torch.nn.Parameter]):
        self.params = [p for p in params if p.requires_grad]
        total = sum(p.numel() for p in self.params)
        dev = self.params[0].device if self.params else torch.device("cpu")
        self.flat = torch.zeros(total, dtype=torch.float32, device=dev)
        self.views = []
        off = 0
        for p in self.params:
            v = self.flat[off:off + p.numel()].view(p.shape)
            p._sph_master_grad = v          # read by Conv3d.forward / ConvFunction.backward
            self.views.append(v)
            off += p.numel()

    def zero(self) -> None:
        self.flat.zero_()

    def all_reduce(self, group=None, average: bool = False) -> int:
        """Sum (or average) over the process group, in place; returns the number of fp32 elements reduced."""
        import torch.distributed as dist
        if dist.is_available() and dist.is_initialized() and dist.get_world_size(group) > 1:
            dist.all_reduce(self.flat, op=dist.ReduceOp.SUM, group=group)
            if average:
                self.flat /= dist.get_world_size(group)
        return int(self.flat.numel())

    def absorb_autograd(self) -> None:
        """Adds (and clears) `.grad` of parameters whose gradient came through autograd instead of a kernel that
        writes the buffer (dense layers mixed into the model)."""
        for p, v in zip(self.params, self.views):
            if p.grad is not None:
                v.add_(p.grad.float())
                p.grad = None

    def to_grads(self, max_norm: Optional[float] = None, norm_type: float = 2.0) -> Optional[torch.Tensor]:
        """`.grad` of every parameter = its slice, rounded once to the parameter's dtype.  With `max_norm` the gradients are
        clipped on the way (the buffer itself stays as it is), and their norm before that is returned: after all_reduce it is the
        norm over all ranks, the same on each."""
        if max_norm is not None:
            with torch.no_grad():
                for p in self.params:
                    if p.grad is None or p.grad.dtype != p.dtype or not p.grad.is_contiguous():
                        p.grad = torch.empty_like(p, memory_format=torch.contiguous_format)
                return clip_gradients(self.views, max_norm, out=[p.grad for p in self.params], norm_type=norm_type)
        for p, v in zip(self.params, self.views):
            if p.grad is None or p.grad.dtype != p.dtype:
                p.grad = v.to(p.dtype)
            else:
                p.grad.copy_(v)

    def norm(self, norm_type: float = 2.0) -> torch.Tensor:
        """Norm over all gradients in the buffer (a float32 scalar on its device)."""
        return grad_norm([self.flat], norm_type)

    def detach(self) -> None:
        for p in self.params:
            if hasattr(p, "_sph_master_grad"):
                del p._sph_master_grad


def flatten_grads(params: Iterable[torch.nn.Parameter]) -> Tuple[torch.Tensor, List[torch.nn.Parameter]]:
    """One flat fp32 buffer with every parameter's gradient (zeros where a parameter has none)."""
    plist = [p for p in params if p.requires_grad]
    total = sum(p.numel() for p in plist)
    dev = plist[0].device if plist else torch.device("cpu")
    flat = torch.zeros(total, dtype=torch.float32, device=dev)
    off = 0
    for p in plist:
        if p.grad is not None:
            flat[off:off + p.numel()] = p.grad.reshape(-1).float()
        off += p.numel()
    return flat, plist


def unflatten_grads(flat: torch.Tensor, plist: List[torch.nn.Parameter]) -> None:
    off = 0
    for p in plist:
        g = flat[off:off + p.numel()].reshape(p.shape).to(p.dtype)
        if p.grad is None:
            p.grad = g.clone()
        else:
            p.grad.copy_(g)
        off += p.numel()


def allreduce_gradients(params: Iterable[torch.nn.Parameter], group=None, average: bool = False) -> int:
    """Sum (or average) the gradients of `params` over the process group with a single all-reduce.
    Returns the number of fp32 elements reduced."""
    import torch.distributed as dist
    flat, plist = flatten_grads(params)
    if dist.is_available() and dist.is_initialized() and dist.get_world_size(group) > 1:
        dist.all_reduce(flat, op=dist.ReduceOp.SUM, group=group)
        if average:
            flat /= dist.get_world_size(group)
    unflatten_grads(flat, plist)
    return int(flat.numel())


def _largest(norm_type: float) -> bool:
    if norm_type not in (2.0, math.inf):
        raise ValueError("the norm is 2 or inf, got %r" % (norm_type,))
    return norm_type == math.inf


def grad_norm(grads: Sequence[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """sqrt(sum g^2) over every value of every tensor (norm_type 2), or max |g| (inf; NaN if any is): a float32 scalar on their
    device, nothing is read back.  float32, float16 and bfloat16 tensors, mixed; sums are held in 64 bits, in a fixed order."""
    largest, grads = _largest(norm_type), list(grads)
    if grads and grads[0].is_cuda:
        from . import _capi
        return _capi.host().grad_clip(grads, None, None, largest)
    if not grads:
        return torch.zeros(())
    with torch.no_grad():
        if largest:
            return torch.stack([g.abs().max().float() if g.numel() else torch.zeros(()) for g in grads]).max()
        return torch.stack([g.double().square().sum() for g in grads]).sum().sqrt().float()


def _dense(t: torch.Tensor) -> bool:
    """Whether the values fill their memory, in any order of the dimensions."""
    expected = 1
    for stride, size in sorted((stride, size) for stride, size in zip(t.stride(), t.shape) if size != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _check_clip(grads: Sequence[torch.Tensor], out: Sequence[torch.Tensor]) -> None:
    """What clipping refuses, on the CPU as the native call does it for tensors on a GPU."""
    spans = []                                       # (begin, end, written) of memory that is read or written
    for g, o in zip(grads, out):
        for t in (g, o):
            if t.device != grads[0].device:
                raise RuntimeError("gradients on several devices: take their norms apart")
            if t.dtype not in (torch.float32, torch.float16, torch.bfloat16):
                raise RuntimeError("gradients are float32, float16 or bfloat16")
            if t.numel() and not _dense(t):
                raise RuntimeError("sphconv_b200 ops need contiguous tensors")
        if g.shape != o.shape or (g.stride() != o.stride() and not (g.is_contiguous() and o.is_contiguous())):
            raise RuntimeError("a destination must have its gradient's shape and layout")
        if not g.numel():
            continue
        spans.append((o.data_ptr(), o.data_ptr() + o.numel() * o.element_size(), True))
        if o.data_ptr() != g.data_ptr() or o.dtype != g.dtype:
            spans.append((g.data_ptr(), g.data_ptr() + g.numel() * g.element_size(), False))
    ends = {True: 0, False: 0}                       # of what is written, and of what is read, so far
    for begin, end, written in sorted(spans):
        if begin < ends[True] or (written and begin < ends[False]):
            raise RuntimeError("a gradient is in the list twice, or overlaps another one or a destination")
        ends[written] = max(ends[written], end)


def clip_gradients(grads: Sequence[torch.Tensor], max_norm: float, out: Optional[Sequence[torch.Tensor]] = None,
                   norm_type: float = 2.0) -> torch.Tensor:
    """Every gradient times min(1, max_norm / (norm + 1e-6)), in place or into `out` (tensors of the same shapes, of any of the
    dtypes: rounded once); returns the norm before clipping.  A norm that is NaN makes all gradients NaN; an infinite one makes them zero
    and those that are infinite NaN, as torch.nn.utils.clip_grad_norm_ does.  Tensors are dense, on one device (the CPU too), float32,
    float16 or bfloat16.  One that is listed twice, or that overlaps another one or a destination, is refused."""
    largest, grads = _largest(norm_type), list(grads)
    if not max_norm >= 0:
        raise ValueError("max_norm must not be negative")
    out = None if out is None else list(out)
    if out is not None and len(out) != len(grads):
        raise ValueError("as many destinations as gradients are needed")
    if grads and grads[0].is_cuda:
        from . import _capi
        return _capi.host().grad_clip(grads, out, float(max_norm), largest)
    to = grads if out is None else out
    _check_clip(grads, to)
    norm = grad_norm(grads, norm_type)
    with torch.no_grad():
        by = torch.clamp(max_norm / (norm + 1e-6), max=1.0)
        for g, o in zip(grads, to):
            o.copy_(g.float() * by)
    return norm


def clip_grad_norm_(params: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0) -> torch.Tensor:
    """Clips the `.grad`s of `params` in place by their global norm, and returns it; parameters without a gradient are passed
    over, one given twice counts once.  For a model whose gradients are in a GradBuffer: `GradBuffer.to_grads(max_norm)`."""
    params = [params] if isinstance(params, torch.Tensor) else params
    grads = {id(p): p.grad for p in params if p.grad is not None}
    if not grads:
        return torch.zeros(())
    return clip_gradients(list(grads.values()), max_norm, norm_type=norm_type)
