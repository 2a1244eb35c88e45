"""Cross attention of a head's queries to the rows of a sparse tensor: with ``SparseConvTensor.dense()``, which feeds a dense head, the
other way out of the encoder.  Rows stay as they are, ragged over the scans.  No reference counterpart."""
import math
from typing import Optional

import torch

from . import _capi as C


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_ptr: torch.Tensor, k_ptr: torch.Tensor,
                    key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """softmax(scale q k^T) v, scan by scan -> [n, heads, channels].

    q [n, heads, channels]; k, v [m, key heads, channels]; float32, float16 or bfloat16, at most 128 channels, any strides (read in
    place where channels are consecutive: slices of one projection need no copy).  Query head h reads key head h // (heads / key heads).
    q_ptr, k_ptr: int32 [B+1] on the device; scan b has the queries q_ptr[b] .. q_ptr[b+1]-1 and the keys k_ptr[b] .. k_ptr[b+1]-1,
    any number of each.  One query a scan (q_ptr = 0, 1, ..., B) is a decoding step.
    key_mask: bool [m]; rows where it is False are no keys and may hold anything.  A query whose scan has no key, and a row that
    belongs to no scan, get zeros, and so do their gradients.  scale: 1 / sqrt(channels) by default.

    Scores, softmax and sums are float32; 16-bit rows have their probabilities rounded to their type in front of the product with v.
    Differentiable once, in q, k and v; results do not depend on the run.  Pointers out of order or out of range are
    reported by check_status()."""
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1]) if q.dim() and q.shape[-1] else 1.0
    return C.host().cross_attention(q, k, v, q_ptr, k_ptr, key_mask, scale)


def scan_rows(x) -> torch.Tensor:
    """k_ptr of a SparseConvTensor: int32 [B+1], where the rows of every scan begin and end."""
    ends = x.z_ptr.reshape(x.B, -1)[:, -1]
    return torch.cat([ends.new_zeros(1), ends]).to(torch.int32)
