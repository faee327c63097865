"""The blocks of the model with residual stream and norms (ResidualStack): eager and captured, against 64 bits.

Each half of a block rounds its input, and the tensors between its projections, to fp16 (2^-11 of each value, at most five
roundings in a row), and its output is normalised, so the term it adds to the residual is off by at most about
5 * 2^-11 of its norm, independently for each half; the residual itself is fp32.  The bound takes 8 * 2^-11 per half.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu


def dense(lin):
    q, s = lin.qweight.double(), lin.scale.double()
    return q * (s[:, None] if s.dim() == 1 else s.repeat_interleave(lin.group, 1)[:, :q.shape[1]])


def rms(v, w):
    return v / (v.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()


def reference(stack, x):
    r = x.double()
    x = rms(r, stack.first.pre_weight)
    for b in stack.layers:
        a = (x @ dense(b.qkv).t())[:, 2 * stack.hidden:] @ dense(b.o).t()
        r = r + torch.sigmoid(b.gate_attention.double()) * rms(a, b.after_attention.post_weight)
        x = rms(r, b.after_attention.pre_weight)
        g = x @ dense(b.mlp.gate_proj).t()
        y = (g * g.sigmoid() * (x @ dense(b.mlp.up_proj).t())) @ dense(b.mlp.down_proj).t()
        r = r + torch.sigmoid(b.gate_mlp.double()) * rms(y, b.after_mlp.post_weight)
        x = rms(r, b.after_mlp.pre_weight)
    return x


@pytest.mark.parametrize("fmt", ["int8", "int4-g32", "int4-g128"])
@pytest.mark.parametrize("m", [1, 16, 40, 200])
def test_residual_stack(sbq, fmt, m):
    layers, hidden, inter = 3, 256, 640
    stack = sbq.stack.ResidualStack(layers, hidden, inter, seed=5, fmt=fmt)
    x = sbq.workloads.activation(m, hidden, seed=6).cuda()
    y, want = stack(x), reference(stack, x)
    assert y.dtype == torch.float16 and y.shape == (m, hidden)
    assert (y.double() - want).norm() <= 2 * layers * 8 * 2.0 ** -11 * want.norm()
    captured = sbq.stack.CapturedStack(stack, m)
    assert torch.equal(captured(x), y)
    assert torch.equal(captured(x.cpu()), y.cpu())
    captured.release()


def test_refusals(sbq):
    with pytest.raises(ValueError, match="int8 or int4"):
        sbq.stack.ResidualStack(1, 64, 64, fmt="int8-dyn")
