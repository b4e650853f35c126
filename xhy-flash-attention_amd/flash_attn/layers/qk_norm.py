"""Per-head RMS norm of queries and keys with the rotary embedding in the same pass.

The norm that current attention blocks put on q and k before the rotary embedding: each head's row
is scaled by ``weight / sqrt(mean(x^2) + eps)`` and its first ``rotary_dim`` columns are rotated, in one
read and one write (the HIP kernels behind ``flash_attn_qk_norm_rotary``, csrc/fa_qknorm.hip), instead
of a norm, two casts and ``apply_rotary_emb_func`` after each other.  Beside
``flash_attn.layers.rotary``, which rotates without a norm; no reference counterpart.  The checks,
allocations and the autograd function are in C++ (csrc/fa_host.cpp).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

import flash_attn_2_cuda as _ext

__all__ = ["apply_qk_norm_rotary_func", "QKNormRotary"]


def apply_qk_norm_rotary_func(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                              k_weight: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
                              sin: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                              interleaved: bool = False, eps: float = 1e-6,
                              inplace: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of each head of q and k, then the rotary embedding of their first columns.

    Arguments:
        q, k: (batch, seqlen, nheads, headdim) and (batch, seqlen, nheads_k, headdim), or without
            the batch dimension; fp16 or bf16, headdim <= 256, any strides with a contiguous last dim.
        q_weight, k_weight: (headdim,), fp32 or q's dtype; None: 1.
        cos, sin: (rows, rotary_dim / 2), fp32 or q's dtype; None: no rotation.
        positions: int32, the shape of q without its last two dims: the row of cos / sin for each
            token; None: 0 .. seqlen - 1.  A token whose position is outside the table gives NaN.
        interleaved: rotate adjacent columns (GPT-J) instead of the two halves (GPT-NeoX).
        inplace: write over q and k (inference: refused when a gradient is asked for).
    Returns q and k normalised and rotated, one rounding from fp32.  Differentiable (once) in q, k and
    the weights; the weights' gradients are summed in a fixed order.  Forward and backward can be captured in
    a graph; a capture is refused while an eager graph of the same leaves that was made on the default stream is
    alive (its gradient accumulators would draw that stream into the capture)."""
    return _ext.host_module().norm_rotary(q, k, q_weight, k_weight, cos, sin, positions, interleaved, eps,
                                          inplace)


class QKNormRotary(torch.nn.Module):
    """The weights of ``apply_qk_norm_rotary_func`` and, with rotary_dim > 0, its cos / sin table.

    The table is fp32, computed in fp64 (angles of far positions keep their digits) for as many rows
    as asked for, and grows by doubling (the host then waits for it: any stream may use it next); XPos
    scaling is not part of it.  Tables that were outgrown are kept (all of them together are smaller than
    the last one): graphs captured with them read them at every replay.  A call in a capture that needs a
    longer table fills one of its own at every replay; call ``table(rows, device)``, or the step itself,
    before the capture."""

    def __init__(self, headdim: int, rotary_dim: int = 0, base: float = 10000.0, interleaved: bool = False,
                 eps: float = 1e-6, device=None, dtype=None):
        super().__init__()
        self.rotary_dim, self.base, self.interleaved, self.eps = rotary_dim, float(base), interleaved, eps
        self.q_weight = torch.nn.Parameter(torch.ones(headdim, device=device, dtype=dtype))
        self.k_weight = torch.nn.Parameter(torch.ones(headdim, device=device, dtype=dtype))
        self._tables = {}                          # device: its tables, the last one in use

    def table(self, rows: int, device) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
        """cos, sin of at least ``rows`` rows on ``device``."""
        if self.rotary_dim == 0:
            return None, None
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        tables = self._tables.setdefault(device, [])
        have = tables[-1][0].shape[0] if tables else 0
        if have < rows:
            # (a table made under inference_mode could not be saved for a later backward)
            with torch.inference_mode(False):
                inv = self.base ** (-torch.arange(0, self.rotary_dim, 2, device=device, dtype=torch.float64)
                                    / self.rotary_dim)
                angle = torch.outer(torch.arange(max(rows, 2 * have), device=device, dtype=torch.float64), inv)
                made = angle.cos().float(), angle.sin().float()
            if device.type == "cuda":
                with torch.cuda.device(device):
                    if torch.cuda.is_current_stream_capturing():
                        return made                # filled by the replays, in the graph's memory: for this call alone
                    torch.cuda.current_stream().synchronize()   # whole for calls on other streams
            tables.append(made)
        return tables[-1]

    def forward(self, q, k, positions=None, max_position=None):
        """q, k as apply_qk_norm_rotary_func; with positions, max_position bounds them (rows of the table)."""
        rows = q.shape[-3] if positions is None else max_position
        assert self.rotary_dim == 0 or rows is not None, "positions need max_position, the rows of the table"
        cos, sin = self.table(rows, q.device) if self.rotary_dim else (None, None)
        return apply_qk_norm_rotary_func(q, k, self.q_weight, self.k_weight, cos, sin,
                                         positions if self.rotary_dim else None, self.interleaved, self.eps)
