"""A head of queries on the encoder: layers of cross attention to a sparse tensor's rows and an MLP, each followed by its gate, residual
scale and the next norm in one pass.  Scans stay ragged, nothing is made dense.  No reference counterpart."""
from typing import List, Optional, Tuple

import torch
from torch import nn

from .attention import CrossAttention, scan_rows
from .norm import ResidualNorm, RowNorm
from .tensor import SparseConvTensor

KeysAndValues = Tuple[torch.Tensor, torch.Tensor]


class DecoderLayer(nn.Module):
    """forward(x, normed, k, v, q_ptr, k_ptr, key_mask=None) -> (x, normed): attention and MLP, each on the normed rows, gated by a
    linear layer of them and added to x."""

    def __init__(self, channels, row_channels, heads, key_heads, hidden, eps, center, initial_scale):
        super().__init__()
        self.attention = CrossAttention(channels, row_channels, heads, key_heads)
        self.gate = nn.Linear(channels, channels)
        self.after_attention = ResidualNorm(channels, eps, center, norm_block=False, initial_scale=initial_scale)
        self.mlp = nn.Sequential(nn.Linear(channels, hidden), nn.GELU(), nn.Linear(hidden, channels))
        self.after_mlp = ResidualNorm(channels, eps, center, norm_block=False, initial_scale=initial_scale)

    def forward(self, x, normed, k, v, q_ptr, k_ptr, key_mask=None):
        x, normed = self.after_attention(self.attention.attend(normed, k, v, q_ptr, k_ptr, key_mask), x, self.gate(normed))
        return self.after_mlp(self.mlp(normed), x)


class QueryDecoder(nn.Module):
    """`layers` DecoderLayers on a SparseConvTensor; the result is normed.

    forward(x): the decoder's own `queries` for every scan -> [B, queries, channels].
    forward(x, rows, q_ptr): any number of queries a scan, rows [n, channels] with scan b's from q_ptr[b] to q_ptr[b+1] -> [n, channels].
    key_mask bool [NNZ]: rows of the tensor that are left out where False.
    Step after step on the same scans (tokens of a sequence): memory(x) once, then decode(rows, q_ptr, memory) each time.

    Keys and values are made of x.feature alone: where a row lies in its scan is known to the head as far as the features say it, so a caller
    that needs positions adds them to the features (an embedding of x.z_idx and of the column, say).  Queries of a scan do not see
    one another."""

    def __init__(self, channels: int, row_channels: int, heads: int, layers: int, queries: int = 0, key_heads: Optional[int] = None,
                 hidden: Optional[int] = None, eps: float = 1e-6, center: bool = False, initial_scale: Optional[float] = None):
        super().__init__()
        self.queries = nn.Parameter(torch.randn(queries, channels)) if queries else None
        self.norm_rows = RowNorm(row_channels, eps, center)
        self.norm = RowNorm(channels, eps, center)
        self.layers = nn.ModuleList(DecoderLayer(channels, row_channels, heads, key_heads, hidden or 4 * channels, eps, center,
                                                 initial_scale) for _ in range(layers))

    def memory(self, x: SparseConvTensor) -> Tuple[torch.Tensor, List[KeysAndValues]]:
        """Where the scans' rows begin and end, and each layer's keys and values of them."""
        rows = self.norm_rows(x.feature)
        return scan_rows(x), [layer.attention.project(rows) for layer in self.layers]

    def decode(self, rows: torch.Tensor, q_ptr: torch.Tensor, memory: Tuple[torch.Tensor, List[KeysAndValues]],
               key_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        k_ptr, projected = memory
        normed = self.norm(rows)
        for layer, (k, v) in zip(self.layers, projected):
            rows, normed = layer(rows, normed, k, v, q_ptr, k_ptr, key_mask)
        return normed

    def forward(self, x: SparseConvTensor, rows: Optional[torch.Tensor] = None, q_ptr: Optional[torch.Tensor] = None,
                key_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        if rows is not None:
            if q_ptr is None:
                raise ValueError("rows of queries need q_ptr: where those of each scan begin and end")
            return self.decode(rows, q_ptr, self.memory(x), key_mask)
        if self.queries is None:
            raise ValueError("the decoder has no queries of its own: give rows and q_ptr")
        n = self.queries.shape[0]
        own = self.queries.expand(x.B, -1, -1).reshape(x.B * n, -1)
        q_ptr = torch.arange(0, (x.B + 1) * n, n, dtype=torch.int32, device=own.device)
        return self.decode(own, q_ptr, self.memory(x), key_mask).view(x.B, n, -1)
