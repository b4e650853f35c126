"""Per-head RMS norm of queries and keys with the rotary embedding in the same pass.

The norm that current attention blocks put on q and k before the rotary embedding: each head's row
is scaled by ``weight / sqrt(mean(x^2) + eps)`` and its first ``rotary_dim`` columns are rotated, in one
read and one write (the HIP kernels behind ``flash_attn_qk_norm_rotary``, csrc/fa_qknorm.hip), instead
of a norm, two casts and ``apply_rotary_emb_func`` after each other.  Beside
``flash_attn.layers.rotary``, which rotates without a norm; no reference counterpart.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

import flash_attn_2_cuda as _ext

__all__ = ["apply_qk_norm_rotary_func", "QKNormRotary"]

_lib = _ext._lib
_P, _I, _I64, _F, _B = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_bool
_lib.flash_attn_qk_norm_rotary.argtypes = [_P] * 9 + [_I] * 7 + [_F] + [_P] * 4 + [_I64] * 2 + [_B] * 4 + [_P]
_lib.flash_attn_qk_norm_rotary.restype = _B
_lib.flash_attn_qk_norm_rotary_bwd.argtypes = ([_P] * 14 + [_I] * 7 + [_F] + [_P] * 6 + [_I64] * 2 + [_B] * 4
                                               + [_P])
_lib.flash_attn_qk_norm_rotary_bwd.restype = _B
_lib.flash_attn_qk_norm_rotary_workspace.argtypes = [_I]
_lib.flash_attn_qk_norm_rotary_workspace.restype = ctypes.c_size_t


def _strides(t: torch.Tensor):
    return (_I64 * 3)(t.stride(0), t.stride(1), t.stride(2))


def _rows(t: torch.Tensor) -> torch.Tensor:
    """(b, s, h, d) view of a fixed-length or (total, h, d) tensor."""
    return t if t.dim() == 4 else t.unsqueeze(0)


def _check_args(q, k, q_weight, k_weight, cos, sin, positions):
    check = _ext._check
    check(q.dtype in (torch.float16, torch.bfloat16), "qk_norm_rotary: only fp16 and bf16 are supported")
    check(k.dtype == q.dtype, "qk_norm_rotary: q and k must have the same dtype")
    check(q.dim() in (3, 4) and k.dim() == q.dim(),
          "qk_norm_rotary: q and k must be (batch, seqlen, nheads, headdim) or (total, nheads, headdim)")
    check(q.shape[:-2] == k.shape[:-2] and q.shape[-1] == k.shape[-1],
          "qk_norm_rotary: q and k must agree in batch, seqlen and headdim")
    check(q.shape[-2] > 0 and k.shape[-2] > 0, "qk_norm_rotary: q and k need a head each")
    check(0 < q.shape[-1] <= 256, "qk_norm_rotary: headdim must be at most 256")
    check(q.stride(-1) == 1 and k.stride(-1) == 1, "qk_norm_rotary: last dim must be contiguous")
    d = q.shape[-1]
    for w in (q_weight, k_weight):
        if w is not None:
            check(tuple(w.shape) == (d,), "qk_norm_rotary: weights must have shape (headdim,)")
            check(w.dtype in (q.dtype, torch.float32), "qk_norm_rotary: weights must be fp32 or of q's dtype")
    if q_weight is not None and k_weight is not None:
        check(q_weight.dtype == k_weight.dtype, "qk_norm_rotary: weights must share a dtype")
    check((cos is None) == (sin is None), "qk_norm_rotary: cos and sin come together")
    if cos is None:
        check(positions is None, "qk_norm_rotary: positions without cos and sin")
    else:
        _check_table(q, cos, sin, positions)
    tensors = [t for t in (q, k, q_weight, k_weight, cos, sin, positions) if t is not None]
    check(all(t.is_cuda for t in tensors), "qk_norm_rotary: tensors must be on the GPU")
    check(all(t.device == q.device for t in tensors), "qk_norm_rotary: tensors must share a device")
    check(_ext._is_gfx950(q.device), "qk_norm_rotary: only gfx950 (MI355X) GPUs are supported")


def _check_table(q, cos, sin, positions):
    check, d = _ext._check, q.shape[-1]
    check(cos.dim() == 2 and cos.shape == sin.shape and cos.dtype == sin.dtype, "qk_norm_rotary: bad cos/sin shape")
    check(cos.dtype in (q.dtype, torch.float32), "qk_norm_rotary: cos and sin must be fp32 or of q's dtype")
    check(0 < 2 * cos.shape[1] <= d and cos.shape[0] > 0, "qk_norm_rotary: bad cos/sin shape")
    if positions is None:
        check(cos.shape[0] >= q.shape[-3], "qk_norm_rotary: cos/sin have fewer rows than the sequence")
    else:
        check(positions.dtype == torch.int32, "qk_norm_rotary: positions must have dtype int32")
        check(positions.shape == q.shape[:-2], "qk_norm_rotary: positions must have the shape of q's tokens")


def _common(q4, k4, q_weight, k_weight, cos, sin, positions):
    """Contiguous vectors, table and positions, and the arguments that both directions end with."""
    if cos is not None and (cos.stride(1) != 1 or sin.stride() != cos.stride()):
        cos, sin = cos.contiguous(), sin.contiguous()
    if positions is not None:
        positions = positions.reshape(q4.shape[:2])
        if positions.stride(1) != 1:
            positions = positions.contiguous()
    q_weight, k_weight = (None if w is None else w.contiguous() for w in (q_weight, k_weight))
    return q_weight, k_weight, cos, sin, positions


def _sizes(q4, k4, cos):
    b, s, h, d = q4.shape
    return b, s, h, k4.shape[2], d, 0 if cos is None else 2 * cos.shape[1], 0 if cos is None else cos.shape[0]


def _flags(q4, q_weight, k_weight, cos, positions, interleaved):
    w = q_weight if q_weight is not None else k_weight
    return (0 if positions is None else positions.stride(0), 0 if cos is None else cos.stride(0),
            w is not None and w.dtype == torch.float32, cos is not None and cos.dtype == torch.float32,
            bool(interleaved), q4.dtype == torch.bfloat16, _ext._stream(q4))


def _forward(q, k, q_out, k_out, q_weight, k_weight, cos, sin, positions, interleaved, eps):
    q4, k4, qo4, ko4 = _rows(q), _rows(k), _rows(q_out), _rows(k_out)
    q_weight, k_weight, cos, sin, positions = _common(q4, k4, q_weight, k_weight, cos, sin, positions)
    if q4.numel() == 0:
        return
    ptr = _ext._ptr
    with _ext._device_guard(q.device):
        ok = _lib.flash_attn_qk_norm_rotary(
            ptr(q4), ptr(k4), ptr(qo4), ptr(ko4), ptr(q_weight), ptr(k_weight), ptr(cos), ptr(sin), ptr(positions),
            *_sizes(q4, k4, cos), float(eps), _strides(q4), _strides(k4), _strides(qo4), _strides(ko4),
            *_flags(q4, q_weight, k_weight, cos, positions, interleaved))
    if not ok:
        _ext._raise_lib_error("flash_attn_qk_norm_rotary")


class ApplyQKNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, interleaved, eps):
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        _forward(q, k, q_out, k_out, q_weight, k_weight, cos, sin, positions, interleaved, eps)
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.interleaved, ctx.eps = interleaved, eps
        return q_out, k_out

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        # (a sum's gradient is an expanded scalar, for instance)
        dq_out, dk_out = (t if t.stride(-1) == 1 else t.contiguous() for t in (dq_out, dk_out))
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        q4, k4 = _rows(q), _rows(k)
        qw, kw, cos, sin, positions = _common(q4, k4, q_weight, k_weight, cos, sin, positions)
        want = q4.numel() > 0
        make = torch.empty_like if want else torch.zeros_like
        dqw = make(qw) if qw is not None and ctx.needs_input_grad[2] else None
        dkw = make(kw) if kw is not None and ctx.needs_input_grad[3] else None
        if want:
            ptr = _ext._ptr
            with _ext._device_guard(q.device):
                work = None
                if dqw is not None or dkw is not None:
                    size = _lib.flash_attn_qk_norm_rotary_workspace(q.shape[-1])
                    work = torch.empty(size, dtype=torch.uint8, device=q.device)
                ok = _lib.flash_attn_qk_norm_rotary_bwd(
                    ptr(dq_out), ptr(dk_out), ptr(q4), ptr(k4), ptr(dq), ptr(dk), ptr(qw), ptr(kw), ptr(dqw), ptr(dkw),
                    ptr(cos), ptr(sin), ptr(positions), ptr(work), *_sizes(q4, k4, cos), float(ctx.eps),
                    _strides(_rows(dq_out)), _strides(_rows(dk_out)), _strides(q4), _strides(k4), _strides(_rows(dq)),
                    _strides(_rows(dk)), *_flags(q4, qw, kw, cos, positions, ctx.interleaved))
            if not ok:
                _ext._raise_lib_error("flash_attn_qk_norm_rotary_bwd")
        return dq, dk, dqw, dkw, None, None, None, None, None


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
    the weights; the weights' gradients are summed in a fixed order."""
    _ext._check(eps >= 0.0, "qk_norm_rotary: eps must not be negative")
    _check_args(q, k, q_weight, k_weight, cos, sin, positions)
    if not inplace:
        return ApplyQKNormRotary.apply(q, k, q_weight, k_weight, cos, sin, positions, interleaved, eps)
    leaves = (q, k, q_weight, k_weight)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in leaves):
        raise RuntimeError("qk_norm_rotary: inplace=True is for inference; the backward needs the inputs")
    _forward(q, k, q, k, q_weight, k_weight, cos, sin, positions, interleaved, eps)
    return q, k


class QKNormRotary(torch.nn.Module):
    """The weights of ``apply_qk_norm_rotary_func`` and, with rotary_dim > 0, its cos / sin table.

    The table is fp32, computed in fp64 (angles of far positions keep their digits) for as many rows
    as asked for, and grows by doubling; XPos scaling is not part of it."""

    def __init__(self, headdim: int, rotary_dim: int = 0, base: float = 10000.0, interleaved: bool = False,
                 eps: float = 1e-6, device=None, dtype=None):
        super().__init__()
        self.rotary_dim, self.base, self.interleaved, self.eps = rotary_dim, float(base), interleaved, eps
        self.q_weight = torch.nn.Parameter(torch.ones(headdim, device=device, dtype=dtype))
        self.k_weight = torch.nn.Parameter(torch.ones(headdim, device=device, dtype=dtype))
        self._cos = self._sin = None

    def table(self, rows: int, device) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
        if self.rotary_dim == 0:
            return None, None
        if self._cos is None or self._cos.shape[0] < rows or self._cos.device != device:
            have = 0 if self._cos is None or self._cos.device != device else self._cos.shape[0]
            n = max(rows, 2 * have)
            inv = self.base ** (-torch.arange(0, self.rotary_dim, 2, device=device, dtype=torch.float64)
                                / self.rotary_dim)
            angle = torch.outer(torch.arange(n, device=device, dtype=torch.float64), inv)
            self._cos, self._sin = angle.cos().float(), angle.sin().float()
        return self._cos, self._sin

    def forward(self, q, k, positions=None, max_position=None):
        """q, k as apply_qk_norm_rotary_func; with positions, max_position bounds them (rows of the table)."""
        rows = q.shape[-3] if positions is None else max_position
        assert self.rotary_dim == 0 or rows is not None, "positions need max_position, the rows of the table"
        cos, sin = self.table(rows, q.device) if self.rotary_dim else (None, None)
        return apply_qk_norm_rotary_func(q, k, self.q_weight, self.k_weight, cos, sin,
                                         positions if self.rotary_dim else None, self.interleaved, self.eps)
