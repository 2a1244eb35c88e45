"""Cross attention of a head's queries to the rows of a sparse tensor: with ``SparseConvTensor.dense()``, which feeds a dense head, the
other way out of the encoder.  Rows stay as they are, ragged over the scans.  No reference counterpart."""
import math
from typing import Optional, Tuple

import torch
from torch import nn

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

    Scores, softmax and sums are float32; 16-bit rows have their probabilities rounded to their type in front of the product with v, and
    gradients take their part of `out` from the rounded one.  Scores of some millions and more have lost their differences to float32's
    rounding, and the probabilities with them.

    How fast: 16-bit rows run on the tensor cores where channels are a multiple of 8, rows and heads begin on 16-byte boundaries and the
    scale is positive.  Others take the CUDA cores and many times as long (256 queries and 20 k keys a scan, 8 scans, 4 heads: 85 us with
    64 channels, 2.8 ms with 60), so projections are better padded.  Where scans have a query row for each key head or less on average, it is
    taken for a decoding step, which reads a scan's keys once for each of its query rows: queries that are all in one of many scans are
    better asked by themselves (64 over 87 k keys: 1.6 ms beside 63 scans without any, 48 us alone).

    Differentiable once, backward, in q, k and v; results do not depend on the run.  Pointers out of order or out of range are
    reported by check_status()."""
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1]) if q.dim() and q.shape[-1] else 1.0
    return C.host().cross_attention(q, k, v, q_ptr, k_ptr, key_mask, scale)


def scan_rows(x) -> torch.Tensor:
    """k_ptr of a SparseConvTensor: int32 [B+1], where the rows of every scan begin and end."""
    ends = x.z_ptr.reshape(x.B, -1)[:, -1]
    return torch.cat([ends.new_zeros(1), ends]).to(torch.int32)


class CrossAttention(nn.Module):
    """cross_attention between its linear projections: forward(queries [n, channels], rows [m, row_channels], q_ptr, k_ptr,
    key_mask=None) -> [n, channels].

    The rows' keys and values are one product, read in place.  What asks the same rows again (a decoder's next token) keeps them:
    k, v = project(rows) once, then attend(queries, k, v, q_ptr, k_ptr) for each."""

    def __init__(self, channels: int, row_channels: int, heads: int, key_heads: Optional[int] = None,
                 head_channels: Optional[int] = None, bias: bool = False):
        super().__init__()
        self.heads, self.key_heads = heads, heads if key_heads is None else key_heads
        if self.heads < 1 or self.key_heads < 1 or self.heads % self.key_heads:
            raise ValueError("{} heads are not a multiple of {} key heads".format(heads, self.key_heads))
        if head_channels is None and channels % heads:
            raise ValueError("{} channels are not a multiple of {} heads".format(channels, heads))
        self.head_channels = channels // heads if head_channels is None else head_channels
        self.to_q = nn.Linear(channels, self.heads * self.head_channels, bias)
        self.to_kv = nn.Linear(row_channels, 2 * self.key_heads * self.head_channels, bias)
        self.to_out = nn.Linear(self.heads * self.head_channels, channels, bias)

    def extra_repr(self):
        return "heads={}, key_heads={}, head_channels={}".format(self.heads, self.key_heads, self.head_channels)

    def project(self, rows: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """Keys and values of rows [m, row_channels]: two views of one [m, 2, key heads, head channels]."""
        return self.to_kv(rows).view(rows.shape[0], 2, self.key_heads, self.head_channels).unbind(1)

    def attend(self, queries, k, v, q_ptr, k_ptr, key_mask=None):
        q = self.to_q(queries).view(queries.shape[0], self.heads, self.head_channels)
        return self.to_out(cross_attention(q, k, v, q_ptr, k_ptr, key_mask).flatten(1))

    def forward(self, queries, rows, q_ptr, k_ptr, key_mask=None):
        return self.attend(queries, *self.project(rows), q_ptr, k_ptr, key_mask)
