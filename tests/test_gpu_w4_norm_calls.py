"""Calls of the 4-bit entry points and of residual_norm beside the ordinary ones: operands that lie in one buffer, calls
that follow one another closely, sizes at the limits of a launch."""

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def rand(*shape, seed, dtype=F32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


@pytest.mark.parametrize("m,d", [(1, 320), (6, 96), (6, 333), (700, 2560), (3, 20000)])
def test_gates_and_weights_in_one_buffer(sbq, m, d):
    """A gate or a weight under an output is refused (its readers and the writer are not ordered); beside the output's
    rows, in the same buffer, it is read as anywhere else."""
    y, w = rand(m, d, seed=1), rand(d, seed=2)
    buf = rand(m + 2, d + 8, seed=3)
    r, kept = buf[:m, 4:4 + d], buf.clone()
    for kw in ({"gate": r[:, :1]}, {"gate": r[:, d - 1:]}, {"post_weight": r[0]}, {"pre_weight": r[m - 1]}):
        kw = {"pre_weight": w, **kw}
        with pytest.raises(ValueError, match="overlaps"):
            sbq.residual_norm(y, r, gate_act="sigmoid" if "gate" in kw else "none", residual_out=r, **kw)
    if m > 1:
        with pytest.raises(ValueError, match="overlaps"):
            sbq.residual_norm(y, r, w, gate=r[0], residual_out=r)
    assert torch.equal(buf, kept)
    # the same call on three buffers of the same layout: one for the rows, one for the output, one for the rest
    out = torch.empty_like(buf)[:m, 4:4 + d]
    apart, own = ({"gate": b[:m, :1], "pre_weight": b[m, 4:4 + d], "post_weight": b[m + 1, 4:4 + d]} for b in (kept, buf))
    want = sbq.residual_norm(y, r, gate_act="tanh", residual_out=out, **apart)
    got = sbq.residual_norm(y, r, gate_act="tanh", residual_out=r, **own)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(buf[m:], kept[m:]) and torch.equal(buf[:, :4], kept[:, :4]) and torch.equal(buf[:, 4 + d:], kept[:, 4 + d:])
