"""Argument checks of the 4-bit entry points and of sbq_residual_norm, before any launch (no GPU needed).

The calls below carry made-up addresses: each of them has to be refused on the host.  Where a call next to a
refused one is to be let through, the host's answer is looked at only for the refusal's words.
"""

import ctypes

import pytest
import torch

BASE = 1 << 20  # an address no test reads


def norm_status(sbq, m, d, **fields):
    """(status, message) of sbq_residual_norm on fp32 rows: a branch, a residual and both outputs in buffers of
    their own, 16 MiB apart, with `fields` on top."""
    L = sbq._lib
    a = L.ResidualNormArgs()
    step = 1 << 24
    a.branch, a.residual, a.residual_out, a.out = (BASE + i * step for i in range(4))
    a.pre_weight = BASE + 4 * step
    a.ld_branch = a.ld_residual = a.ld_residual_out = a.ld_out = d
    a.m, a.d = m, d
    a.residual_scale = a.branch_scale = 1.0
    a.eps = 1e-6
    for name, value in fields.items():
        setattr(a, name, value)
    status = L.load().sbq_residual_norm(ctypes.byref(a), None)
    return status, L.load().sbq_last_error().decode()


def refused(sbq, m, d, **fields):
    status, message = norm_status(sbq, m, d, **fields)
    return status == sbq._lib.ERR_INVALID_ARGUMENT and "overlaps" in message


RES, FREE = BASE + (1 << 24), BASE + 6 * (1 << 24)
OUTPUTS = {"residual_out": BASE + 2 * (1 << 24), "out": BASE + 3 * (1 << 24)}


@pytest.fixture
def no_device():
    if torch.cuda.is_available():
        pytest.skip("made-up addresses, some of which pass the checks: only where nothing can be launched")


@pytest.mark.parametrize("m,d", [(1, 8), (5, 96), (300, 333)])
def test_norm_outputs_over_a_vector(sbq, no_device, m, d):
    """No output may lie on a weight or a gate per column: every row reads them, whenever another row is stored."""
    L = sbq._lib
    last = (m - 1) * d * 4
    for name in ("pre_weight", "post_weight", "gate"):
        mode = {"gate_mode": L.GATE_PER_COLUMN} if name == "gate" else {}
        for out, at in OUTPUTS.items():
            for off in (0, last, last + 4 * (d - 1), -4 * (d - 1)):
                if name == "gate" and m == 1 and off == 0:
                    continue  # one row: the gate's elements are those of a full gate
                assert refused(sbq, m, d, **{name: at + off}, **mode), (name, out, off)
            for off in (last + 4 * d, -4 * d):
                assert not refused(sbq, m, d, **{name: at + off}, **mode), (name, out, off)


def test_norm_outputs_around_a_vector(sbq, no_device):
    """A vector that lies between the rows of an output shares nothing with it; one that reaches a row does."""
    L = sbq._lib
    m, d, ld = 7, 40, 128
    for name, mode in (("pre_weight", {}), ("post_weight", {}), ("gate", {"gate_mode": L.GATE_PER_COLUMN})):
        for out, at in OUTPUTS.items():
            wide = {"ld_" + out: ld}
            for col, bad in ((40, False), (88, False), (39, True), (89, True), (0, True)):
                assert refused(sbq, m, d, **{name: at + 4 * (3 * ld + col)}, **mode, **wide) == bad, (name, out, col)


@pytest.mark.parametrize("m,d", [(1, 300), (4, 96), (4, 600)])
def test_norm_outputs_over_a_gate_per_row(sbq, no_device, m, d):
    """A gate per row that is a column of an output is refused, in place or not; a column beside it is not."""
    L = sbq._lib
    ld = d + 16
    for out, at in OUTPUTS.items():
        wide = {"ld_" + out: ld, "gate_mode": L.GATE_PER_ROW, "ld_gate": ld}
        for col, bad in ((0, True), (d - 1, True), (d, False), (d + 15, False)):
            assert refused(sbq, m, d, gate=at + 4 * col, **wide) == bad, (out, col)
        # gates next to each other, inside a row of the output and outside of all of them
        wide["ld_gate"] = 1
        assert refused(sbq, m, d, gate=at, **wide)
        assert not refused(sbq, m, d, gate=FREE, **wide)
    assert refused(sbq, m, d, gate=RES, gate_mode=L.GATE_PER_ROW, ld_gate=d, residual_out=RES)
    assert not refused(sbq, m, d, gate=RES, gate_mode=L.GATE_PER_ROW, ld_gate=d)


def plan(sbq, m, n, k, x_dtype="F32", matrices=1):
    L = sbq._lib
    out = (ctypes.c_int * 4)()
    L.call("sbq_linear_w4_plan", m, n, k, getattr(L, x_dtype), matrices, out)
    return list(out)


def test_plan_of_a_call(sbq):
    L = sbq._lib
    assert plan(sbq, 1, 4096, 4096) == [0, 8, 0, 0] and plan(sbq, 16, 4096, 4096)[:2] == [0, 16]
    assert plan(sbq, 17, 4096, 4096, "F16")[:2] == [1, 64]
    assert plan(sbq, 4096, 12288, 4096, "F16")[:2] == [2, 256]
    for m, n, k in ((0, 16, 16), (16, -1, 16), (16, 16, 0)):
        assert L.load().sbq_linear_w4_plan(m, n, k, L.F16, 1, (ctypes.c_int * 4)()) == L.ERR_INVALID_ARGUMENT
    assert L.load().sbq_linear_w4_plan(16, 16, 16, L.F16, 1, None) == L.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("matrices", [1, 2])
@pytest.mark.parametrize("x_dtype", ["F16", "BF16", "F32"])
def test_every_row_count_fits_its_launch(sbq, x_dtype, matrices):
    """The CTA kernel's 64-row tiles are the y dimension of its grid, which ends at 65535."""
    for m in (65535 * 64, 65535 * 64 + 1, 1 << 23, 1 << 27, (1 << 31) - 257):
        for n in (1, 16, 64, 128, 129, 1024):
            for k in (16, 100, 512, 2560):
                kernel, tokens, parts, _ = plan(sbq, m, n, k, x_dtype, matrices)
                assert kernel == 2 or -(-m // tokens) <= 65535, (m, n, k)
                assert kernel == 1 or tokens == 256 and parts >= 1


def int4(sbq, n, k, device, group=64):
    """An Int4Linear around buffers of the right sizes on any device, which cannot be run."""
    lib = sbq._lib.load()
    mod = sbq.Int4Linear.__new__(sbq.Int4Linear)
    torch.nn.Module.__init__(mod)
    mod._adopt((torch.zeros(lib.sbq_w4_packed_bytes(n, k), dtype=torch.uint8, device=device),
                torch.zeros(lib.sbq_w4_scale_bytes(n, k, group), dtype=torch.uint8, device=device),
                torch.zeros((n + 15) // 16 * 16, dtype=torch.int32, device=device)), (n, k), None, group)
    return mod


def int8(sbq, n, k, device):
    return sbq.Int8Linear.from_packed(torch.zeros(sbq._lib.packed_bytes(n, k), dtype=torch.int8, device=device),
                                      torch.zeros(n, device=device), None, n, k)


@pytest.mark.parametrize("make", [int4, int8])
def test_gate_and_up_on_different_devices(sbq, make):
    """One launch reads both weights: both have to be on its device, also when a module was moved later."""
    down = make(sbq, 64, 128, "cpu")
    with pytest.raises(ValueError, match="same device"):
        sbq.FusedGatedMLP(make(sbq, 128, 64, "cpu"), make(sbq, 128, 64, "meta"), down)
    mlp = sbq.FusedGatedMLP(make(sbq, 128, 64, "cpu"), make(sbq, 128, 64, "cpu"), down)
    mlp.up_proj.to("meta")
    x = torch.zeros(2, 64)
    for call in (mlp, mlp.gateup, lambda t: mlp.gateup_into(t, torch.zeros(2, 128))):
        with pytest.raises(ValueError, match="same device"):
            call(x)


def test_buffers_of_another_size_are_not_unpacked(sbq):
    """unpack_int4 reads what n, k and group say: the buffers have to be those of such a weight, on one CUDA device."""
    n, k, group = 40, 200, 64
    lin = int4(sbq, n, k, "cpu", group)
    bad = [(lin.packed, lin.scales, 56, k, group), (lin.packed, lin.scales, n, 300, group), (lin.packed, lin.scales, n, k, 32),
           (lin.packed[:-1024], lin.scales, n, k, group), (lin.packed, lin.scales[1:], n, k, group),
           (lin.packed.view(torch.int8), lin.scales, n, k, group), (lin.packed, lin.scales.view(torch.bfloat16), n, k, group),
           (torch.zeros(2 * lin.packed.numel(), dtype=torch.uint8)[::2], lin.scales, n, k, group),
           (lin.packed[:0], lin.scales[:0], 0, k, group), (lin.packed[:0], lin.scales[:0], n, 0, group)]
    for args in bad:
        with pytest.raises(ValueError, match="do not match"):
            sbq.unpack_int4(*args)
    with pytest.raises(ValueError, match="group size"):
        sbq.unpack_int4(lin.packed, lin.scales, n, k, 48)
    with pytest.raises(ValueError, match="one CUDA device"):
        sbq.unpack_int4(lin.packed, lin.scales, n, k, group)
    for args in bad:
        args = (*args[:2], lin.rowmul, *args[2:4], None, args[4])
        with pytest.raises(ValueError, match="do not match"):
            sbq.Int4Linear.from_packed(*args)
    with pytest.raises(ValueError, match="do not match"):
        sbq.Int4Linear.from_packed(lin.packed, lin.scales, lin.rowmul[:-1], n, k, None, group)
    with pytest.raises(ValueError, match="one CUDA device"):
        sbq.Int4Linear.from_packed(lin.packed, lin.scales, lin.rowmul, n, k, None, group)


def test_packing_of_misaligned_operands(sbq, no_device):
    """Addresses that are not multiples of the element size are refused, as the products refuse them."""
    L, at = sbq._lib, BASE
    bufs = (at, at + 4096, at + 8192)  # packed, scales, rowmul

    def refused(name, *args):
        status, message = getattr(L.load(), name)(*args, None), L.load().sbq_last_error().decode()
        return status == L.ERR_ALIGNMENT and "aligned" in message

    w = at + 65536
    for dtype, off, bad in ((L.F32, 2, True), (L.F32, 4, False), (L.F16, 1, True), (L.BF16, 3, True), (L.BF16, 2, False)):
        assert refused("sbq_w4_quantize_pack", w + off, dtype, 16, 32, 32, 32, *bufs) == bad
    assert refused("sbq_w4_quantize_pack", w, L.F32, 16, 32, 32, 32, *bufs[:2], bufs[2] + 2)
    for scale, row, bad in ((1, 0, True), (2, 0, False), (0, 2, True), (0, 4, False)):
        assert refused("sbq_w4_pack", w + 1, 32, w + 4096 + scale, 1, 16, 32, 32, *bufs[:2], bufs[2] + row) == bad
    assert refused("sbq_w4_unpack", *bufs[:2], 16, 32, 32, w + 1, 32, w + 4097, 1)
    assert not refused("sbq_w4_unpack", *bufs[:2], 16, 32, 32, w + 1, 32, w + 4098, 1)


def test_norm_refuses_forward_mode_tangents(sbq):
    """residual_norm has no gradient in either mode: a dual tensor is refused, whichever operand it is."""
    import torch.autograd.forward_ad as fwd

    with fwd.dual_level():
        rows, vec = torch.randn(3, 8), torch.randn(8)
        dual = fwd.make_dual(rows, torch.ones(3, 8)), fwd.make_dual(vec, torch.ones(8))
        for branch, residual, kw in ((dual[0], rows, {}), (rows, dual[0], {}), (rows, rows, {"gate": dual[0]}),
                                     (rows, rows, {"pre_weight": dual[1]}), (rows, rows, {"post_weight": dual[1]})):
            with pytest.raises(ValueError, match="no gradient"):
                sbq.residual_norm(branch, residual, **kw)
        with pytest.raises(ValueError, match="CUDA device"):  # plain tensors within a dual level
            sbq.residual_norm(rows, rows, vec)


@pytest.mark.parametrize("make", [int4, int8])
def test_fusing_leaves_a_block_spread_over_devices_alone(sbq, make):
    model = torch.nn.Module()
    for name, device in (("together", "cpu"), ("apart", "meta")):
        block = torch.nn.Module()
        block.gate_proj, block.up_proj, block.down_proj = make(sbq, 128, 64, "cpu"), make(sbq, 128, 64, device), make(sbq, 64, 128, "cpu")
        setattr(model, name, block)
    apart = model.apart
    assert sbq.fuse_gated_mlp(model) == 1
    assert isinstance(model.together, sbq.FusedGatedMLP) and model.apart is apart
