"""The step between two blocks of a residual network as one kernel (sbq_residual_norm).

The reference adds each block's output to the residual stream and normalises the sum for the next block
in separate operations (RMSNorm, spikingbrain_cpu/model.py:30-39; Block.forward, model.py:388-392).
``residual_norm`` does the step in one pass, with the optional parts models add to it: a norm of the
block's own output, a gate on it, and scales on both terms.  It hands the next projection its input in
16 bits while the residual stays in its own type.  Like the projections it sits between, it is not
differentiable.
"""

from __future__ import annotations

import ctypes

import torch
import torch.nn as nn

from . import _lib as L
from .quant import _DTYPE_CODE, _current


def _rows(t: torch.Tensor, d: int, what: str, dev: torch.device) -> torch.Tensor:
    """t as [m, d] with unit column stride on ``dev`` (a copy only if its rows are not evenly strided)."""
    if t.device != dev:
        raise ValueError("%s must be on the residual's device %s, got %s" % (what, dev, t.device))
    if t.dtype not in _DTYPE_CODE:
        raise ValueError("%s must be fp32, fp16 or bf16, got %s" % (what, t.dtype))
    t = t if t.dim() == 2 else t.reshape(-1, d)
    return t if (t.stride(1) == 1 or d == 1) and (t.shape[0] <= 1 or t.stride(0) >= d) else t.contiguous()


def _weight(w: torch.Tensor, d: int, what: str, dev: torch.device) -> torch.Tensor:
    if tuple(w.shape) != (d,):
        raise ValueError("%s must have shape (%d,), got %s" % (what, d, tuple(w.shape)))
    if w.device != dev:
        raise ValueError("%s must be on the residual's device %s, got %s" % (what, dev, w.device))
    w = w if w.dtype == torch.float32 else w.float()
    return w if d == 1 or w.stride(0) == 1 else w.contiguous()


def residual_norm(branch: torch.Tensor | None, residual: torch.Tensor, pre_weight: torch.Tensor | None = None, *,
                  post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, gate_act: str = "none",
                  residual_scale: float = 1.0, branch_scale: float = 1.0, eps: float = 1e-6,
                  out_dtype: torch.dtype = torch.float16, residual_out: torch.Tensor | None = None):
    """``(r', x)`` of the step after a block, over the last dimension:

        h  = branch                      or branch * rsqrt(mean(branch^2) + eps) * post_weight
        r' = residual_scale * residual + branch_scale * act(gate) * h
        x  = r' * rsqrt(mean(r'^2) + eps) * pre_weight

    ``residual`` [..., d] and ``branch`` (the block's output, same shape, or None: no branch) are fp32, fp16 or
    bf16 on one CUDA device; r' has the residual's type, x ``out_dtype``, and x is taken from r' before it is
    rounded.  ``gate``: [d], [..., 1] or [..., d]; ``gate_act``: none, sigmoid, silu or tanh.  Statistics are
    fp32.  Without ``pre_weight`` there is no x (None is returned for it).  ``residual_out`` receives r' ([..., d] in
    the residual's type; it may be the residual itself); with no branch, a residual_scale of 1 and no
    ``residual_out`` the residual is returned as it is.
    """
    if not residual.is_cuda:
        raise ValueError("residual_norm runs on a CUDA device, got " + str(residual.device))
    if residual.dim() == 0 or residual.shape[-1] == 0:
        raise ValueError("residual must have a last dimension to normalise over, got shape %s" % (tuple(residual.shape),))
    dev, shape, d = residual.device, residual.shape, residual.shape[-1]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (branch, residual, gate)):
        raise ValueError("residual_norm has no gradient: call it under torch.no_grad() or detach its inputs")
    if gate_act not in L.GATE_ACTS:
        raise ValueError("unknown gate activation %s (one of %s)" % (gate_act, ", ".join(L.GATE_ACTS)))
    if out_dtype not in _DTYPE_CODE:
        raise ValueError("output dtype must be fp32, fp16 or bf16, got %s" % out_dtype)
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    if branch is None and (gate is not None or post_weight is not None):
        raise ValueError("a gate or post_weight needs a branch")
    if branch is not None and branch.shape != shape:
        raise ValueError("branch %s and residual %s must have the same shape" % (tuple(branch.shape), tuple(shape)))
    r = _rows(residual, d, "residual", dev)
    m = r.shape[0]
    a = L.ResidualNormArgs(residual=r.data_ptr(), ld_residual=r.stride(0), residual_dtype=_DTYPE_CODE[r.dtype], m=m, d=d,
                           gate_act=L.GATE_ACTS[gate_act], residual_scale=residual_scale, branch_scale=branch_scale,
                           eps=eps, out_dtype=_DTYPE_CODE[out_dtype])
    keep = [r]  # operands that may be copies live until the launch is queued
    if branch is not None:
        y = _rows(branch, d, "branch", dev)
        keep.append(y)
        a.branch, a.ld_branch, a.branch_dtype = y.data_ptr(), y.stride(0), _DTYPE_CODE[y.dtype]
    if gate is not None:
        if tuple(gate.shape) == (d,) and gate.dim() == 1:
            g = _rows(gate.view(1, d) if gate.stride(0) == 1 or d == 1 else gate.reshape(1, d), d, "gate", dev)
            a.gate_mode = L.GATE_PER_COLUMN
        elif gate.shape == shape:
            g = _rows(gate, d, "gate", dev)
            a.gate_mode = L.GATE_FULL
        elif gate.shape == (*shape[:-1], 1):
            g = _rows(gate, 1, "gate", dev)
            a.gate_mode = L.GATE_PER_ROW
        else:
            raise ValueError("gate must have shape (%d,), %s or %s, got %s" % (d, (*shape[:-1], 1), tuple(shape), tuple(gate.shape)))
        keep.append(g)
        a.gate, a.ld_gate, a.gate_dtype = g.data_ptr(), g.stride(0), _DTYPE_CODE[g.dtype]
    if post_weight is not None:
        w = _weight(post_weight, d, "post_weight", dev)
        keep.append(w)
        a.post_weight = w.data_ptr()
    x = None
    if pre_weight is not None:
        w = _weight(pre_weight, d, "pre_weight", dev)
        keep.append(w)
        x = torch.empty(shape, dtype=out_dtype, device=dev)
        a.pre_weight, a.out, a.ld_out = w.data_ptr(), x.data_ptr(), d
    if residual_out is None and branch is None and residual_scale == 1.0:
        new = residual
    else:
        new = torch.empty(shape, dtype=residual.dtype, device=dev) if residual_out is None else residual_out
        if new.shape != shape or new.dtype != residual.dtype or new.device != dev:
            raise ValueError("residual_out must be a %s tensor of shape %s on %s" % (residual.dtype, tuple(shape), dev))
        if m > 0:
            o = new if new.dim() == 2 else new.reshape(-1, d)
            if o.data_ptr() != new.data_ptr() or (d > 1 and o.stride(1) != 1) or (m > 1 and o.stride(0) < d):
                raise ValueError("residual_out must be rows of unit stride at an even distance")
            a.residual_out, a.ld_residual_out = o.data_ptr(), o.stride(0)
    if m > 0 and (a.out or a.residual_out):
        with _current(dev):
            L.call("sbq_residual_norm", ctypes.byref(a), torch.cuda.current_stream(dev).cuda_stream)
    return new, x


class ResidualNorm(nn.Module):
    """``residual_norm`` with its weights: the step after a block, ``forward(branch, residual, gate=None)``.

    ``pre_weight`` [d] normalises for the next block (None: only the residual is updated), ``post_weight`` [d] the
    block's own output.  Both are kept as fp32 buffers.
    """

    def __init__(self, pre_weight: torch.Tensor | None, post_weight: torch.Tensor | None = None, gate_act: str = "none",
                 residual_scale: float = 1.0, branch_scale: float = 1.0, eps: float = 1e-6,
                 out_dtype: torch.dtype = torch.float16):
        super().__init__()
        if gate_act not in L.GATE_ACTS:
            raise ValueError("unknown gate activation %s (one of %s)" % (gate_act, ", ".join(L.GATE_ACTS)))
        self.register_buffer("pre_weight", None if pre_weight is None else pre_weight.detach().float())
        self.register_buffer("post_weight", None if post_weight is None else post_weight.detach().float())
        self.gate_act, self.out_dtype = gate_act, out_dtype
        self.residual_scale, self.branch_scale, self.eps = float(residual_scale), float(branch_scale), float(eps)

    def forward(self, branch: torch.Tensor | None, residual: torch.Tensor, gate: torch.Tensor | None = None):
        b = self._buffers
        return residual_norm(branch, residual, b["pre_weight"], post_weight=b["post_weight"], gate=gate,
                             gate_act=self.gate_act, residual_scale=self.residual_scale, branch_scale=self.branch_scale,
                             eps=self.eps, out_dtype=self.out_dtype)
