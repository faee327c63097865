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
from torch.autograd import forward_ad

from . import _lib as L
from .quant import _DTYPE_CODE, _raw_stream, _written


def _rows(t: torch.Tensor, d: int, what: str, dev: torch.device) -> tuple[torch.Tensor, int]:
    """(t, row stride) of t as [m, d] with unit column stride (t is a copy only if its rows are not evenly strided)."""
    if t.device != dev:
        raise ValueError("%s must be on the residual's device %s, got %s" % (what, dev, t.device))
    if t.dtype not in _DTYPE_CODE:
        raise ValueError("%s must be fp32, fp16 or bf16, got %s" % (what, t.dtype))
    if t.is_contiguous():
        return t, d
    t = t if t.dim() == 2 else t.reshape(-1, d)
    if (t.stride(1) == 1 or d == 1) and (t.shape[0] <= 1 or t.stride(0) >= d):
        return t, t.stride(0) if t.shape[0] > 1 else d
    return t.contiguous(), d


def _weight(w: torch.Tensor, d: int, what: str, dev: torch.device) -> torch.Tensor:
    if w.shape != (d,):
        raise ValueError("%s must have shape (%d,), got %s" % (what, d, tuple(w.shape)))
    if w.device != dev:
        raise ValueError("%s must be on the residual's device %s, got %s" % (what, dev, w.device))
    if w.dtype != torch.float32:
        w = w.float()
    return w if w.is_contiguous() else w.contiguous()


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
    the residual's type; it may be the residual itself, other overlaps with it, the branch or a full gate are
    refused unless they are the same elements, and so is every overlap with a weight or another gate); with no branch, a residual_scale of 1 and no
    ``residual_out`` the residual is returned as it is.
    """
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                              for t in (branch, residual, gate, pre_weight, post_weight)):
        raise ValueError("residual_norm has no gradient: its inputs must not carry forward-mode tangents")
    dev, shape = residual.device, residual.shape
    if dev.type != "cuda":
        raise ValueError("residual_norm runs on a CUDA device, got " + str(dev))
    if not shape or shape[-1] == 0:
        raise ValueError("residual must have a last dimension to normalise over, got shape %s" % (tuple(shape),))
    if dev.index != torch._C._cuda_getDevice():  # the library launches on the current device
        with torch.cuda.device(dev):
            return residual_norm(branch, residual, pre_weight, post_weight=post_weight, gate=gate, gate_act=gate_act,
                                 residual_scale=residual_scale, branch_scale=branch_scale, eps=eps, out_dtype=out_dtype,
                                 residual_out=residual_out)
    if torch.is_grad_enabled() and (residual.requires_grad or (branch is not None and branch.requires_grad) or
                                    (gate is not None and gate.requires_grad) or
                                    (pre_weight is not None and pre_weight.requires_grad) or
                                    (post_weight is not None and post_weight.requires_grad)):
        raise ValueError("residual_norm has no gradient: call it under torch.no_grad() or detach its inputs")
    act = L.GATE_ACTS.get(gate_act)
    if act is None:
        raise ValueError("unknown gate activation %s (one of %s)" % (gate_act, ", ".join(L.GATE_ACTS)))
    out_code = _DTYPE_CODE.get(out_dtype)
    if out_code is None:
        raise ValueError("output dtype must be fp32, fp16 or bf16, got %s" % out_dtype)
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    d = shape[-1]
    a = L.ResidualNormArgs()
    # every operand (`r`, `y`, `g` and the weights) may be a copy: it stays referenced until the launch is queued
    r, a.ld_residual = _rows(residual, d, "residual", dev)
    a.residual, a.residual_dtype = r.data_ptr(), _DTYPE_CODE[r.dtype]
    m = residual.numel() // d
    a.m, a.d = m, d
    a.gate_act, a.residual_scale, a.branch_scale, a.eps, a.out_dtype = act, residual_scale, branch_scale, eps, out_code
    if branch is not None:
        if branch.shape != shape:
            raise ValueError("branch %s and residual %s must have the same shape" % (tuple(branch.shape), tuple(shape)))
        y, a.ld_branch = _rows(branch, d, "branch", dev)
        a.branch, a.branch_dtype = y.data_ptr(), _DTYPE_CODE[y.dtype]
    elif gate is not None or post_weight is not None:
        raise ValueError("a gate or post_weight needs a branch")
    if gate is not None:
        if gate.dim() == 1 and gate.shape[0] == d:
            g, a.ld_gate = _rows(gate.view(1, d), d, "gate", dev)
            a.gate_mode = L.GATE_PER_COLUMN
        elif gate.shape == shape:
            g, a.ld_gate = _rows(gate, d, "gate", dev)
            a.gate_mode = L.GATE_FULL
        elif gate.shape == (*shape[:-1], 1):
            g, a.ld_gate = _rows(gate, 1, "gate", dev)
            a.gate_mode = L.GATE_PER_ROW
        else:
            raise ValueError("gate must have shape (%d,), %s or %s, got %s" % (d, (*shape[:-1], 1), tuple(shape), tuple(gate.shape)))
        a.gate, a.gate_dtype = g.data_ptr(), _DTYPE_CODE[g.dtype]
    if post_weight is not None:
        wp = _weight(post_weight, d, "post_weight", dev)
        a.post_weight = wp.data_ptr()
    x = None
    if pre_weight is not None:
        w = _weight(pre_weight, d, "pre_weight", dev)
        x = torch.empty(*shape, dtype=out_dtype, device=dev)
        a.pre_weight, a.out, a.ld_out = w.data_ptr(), x.data_ptr(), d
    if residual_out is not None:
        if residual_out.shape != shape or residual_out.dtype != residual.dtype or residual_out.device != dev:
            raise ValueError("residual_out must be a %s tensor of shape %s on %s" % (residual.dtype, tuple(shape), dev))
        new = residual_out
        if m > 0:
            o = new if new.dim() == 2 else new.reshape(-1, d)
            if o.data_ptr() != new.data_ptr() or (d > 1 and o.stride(1) != 1) or (m > 1 and o.stride(0) < d):
                raise ValueError("residual_out must be rows of unit stride at an even distance")
            a.residual_out, a.ld_residual_out = new.data_ptr(), o.stride(0) if m > 1 else d
    elif branch is None and residual_scale == 1.0:
        new = residual
    else:
        new = torch.empty_like(residual, memory_format=torch.contiguous_format)
        a.residual_out, a.ld_residual_out = new.data_ptr(), d
    if m > 0 and (x is not None or new is not residual or residual_out is not None):
        status = L.load().sbq_residual_norm(ctypes.byref(a), _raw_stream(dev))
        if status:
            L.check(status, "sbq_residual_norm")
        if residual_out is not None:
            _written(residual_out)
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
