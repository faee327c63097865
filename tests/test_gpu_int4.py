"""4-bit weights with group scales against plain 64-bit products.

Tolerances.  q * s and a 16-bit x enter the kernels exactly (fp32 x with 22 bits: 2^-23 of each element),
so what is left is the fp32 summation and the rounding of the result.  Every accumulation step loses at
most 2^-22 of the sum of magnitudes S = sum |x w| (a tensor-core step may truncate, one bit more than
half a step), and no element sees more than STEPS of them in a chain: ceil(k / 16) tensor-core steps for
each part of x, the joining of the partial sums, the scale and the bias.  The result is then rounded once: eps / 2 of its
value (2^-25 absolute for an fp16 result below the normal range).
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def weight(n, k, group, seed, spread=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(-8, 8, (n, k), generator=g, device="cuda", dtype=torch.int8)
    s = torch.rand(n, -(-k // group), generator=g, device="cuda") * 0.01 + 0.002
    if spread:  # scales of a row over many powers of two
        s = s * torch.exp2(torch.randint(-12, 12, s.shape, generator=g, device="cuda").float())
    return q, s.to(BF16)


def dense(q, s, group):
    return q.double() * s.double().repeat_interleave(group, dim=1)[:, :q.shape[1]]


def tolerance(x, w, y_dtype, ref, extra=0.0):
    k = x.shape[1]
    parts = 2 if x.dtype == F32 else 1
    steps = parts * -(-k // 16) + -(-k // 128) + 16
    mags = x.double().abs() @ w.abs().t()
    tol = (steps * 2.0 ** -22 + (2.0 ** -23 if x.dtype == F32 else 0.0)) * mags + extra
    return tol + ref.abs() * (torch.finfo(y_dtype).eps / 2) + (2.0 ** -25 if y_dtype == F16 else 0.0)


def acts(m, k, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(m, k, generator=g, device="cuda").to(dtype)


def check(y, x, q, s, group, bias=None):
    w = dense(q, s, group)
    ref = x.double() @ w.t()
    if bias is not None:
        ref = ref + bias.double()
    err = (y.double() - ref).abs()
    tol = tolerance(x, w, y.dtype, ref, 0.0 if bias is None else bias.double().abs() * 2.0 ** -23)
    worst = (err - tol).max().item()
    assert worst <= 0, "off by %g over the tolerance" % worst
    if y.dtype == F32 and ref.norm() > 0 and min(x.shape) > 1 and y.shape[1] > 8:
        # as a whole: sums are cut into pieces of at most 32 tensor-core steps, each off by at most 2^-23
        assert err.norm() <= 2.0 ** -18 * ref.norm(), (err.norm() / ref.norm()).item()


ROWS = [1, 2, 7, 8, 9, 16, 17, 33, 64, 65, 128, 129, 300]


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("x_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_rows_types_groups(sbq, m, x_dtype, group):
    n, k = 272, 640
    q, s = weight(n, k, group, seed=m)
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=group)
    x = acts(m, k, x_dtype, seed=100 + m)
    for y_dtype in (F32, F16, BF16):
        lin.out_dtype = y_dtype
        y = lin(x)
        assert y.dtype == y_dtype and y.shape == (m, n)
        check(y, x, q, s, group)


@pytest.mark.parametrize("n,k", [(1, 1), (1, 16), (3, 8), (15, 31), (16, 128), (17, 129), (100, 257), (255, 96), (513, 1000),
                                 (64, 2560), (2560, 64), (4099, 2500), (33, 12288)])
@pytest.mark.parametrize("m", [1, 5, 12, 20, 77, 200])
def test_odd_sizes(sbq, m, n, k):
    group = (32, 64, 128)[(n + k + m) % 3]
    x_dtype = (F16, BF16, F32)[(n + m) % 3]
    q, s = weight(n, k, group, seed=n + k)
    bias = acts(1, n, F32, seed=3)[0] if n % 2 else None
    lin = sbq.Int4Linear.from_quantized(q, s, bias, group=group)
    x = acts(m, k, x_dtype, seed=m)
    check(lin(x), x, q, s, group, bias)


@pytest.mark.parametrize("m", [3, 16, 40, 260])
def test_scales_over_many_powers_of_two(sbq, m):
    q, s = weight(144, 512, 32, seed=5, spread=True)
    s[3, :] = 0.0          # a row of zeros
    s[4, 1:] = 0.0
    s[5] = -s[5]           # negative scales are scales too
    s[6] = s[6].float().mul(2.0 ** -100).to(BF16)
    s[7] = s[7].float().mul(2.0 ** 90).to(BF16)
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=32)
    for dt in (F16, BF16, F32):
        x = acts(m, 512, dt, seed=8)
        y, w = lin(x), dense(q, s, 32)
        ref = x.double() @ w.t()
        assert ((y.double() - ref).abs() <= tolerance(x, w, F32, ref)).all()


@pytest.mark.parametrize("m", [2, 16, 31, 130])
@pytest.mark.parametrize("x_dtype", [BF16, F32])
def test_activations_of_any_range(sbq, m, x_dtype):
    """Rows far outside fp16's range, a row of zeros, and elements far below the row's largest."""
    q, s = weight(64, 384, 64, seed=6)
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=64)
    x = acts(m, 384, F32, seed=9)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[-1, ::2] *= 1e-12
    if m > 2:
        x[2] = 0.0
    x = x.to(x_dtype)
    y, w = lin(x), dense(q, s, 64)
    ref = x.double() @ w.t()
    assert ((y.double() - ref).abs() <= tolerance(x, w, F32, ref)).all()


@pytest.mark.parametrize("m", [4, 20, 140])
@pytest.mark.parametrize("x_dtype", [F16, BF16, F32])
def test_infinities_and_nan_stay_in_their_rows(sbq, m, x_dtype):
    q, s = weight(48, 256, 128, seed=7)
    q[:, 17] = 3
    q[:, 40] = 2
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=128)
    x = acts(m, 256, x_dtype, seed=10)
    x[1, 17] = float("inf")
    x[2, 40] = float("nan")
    y = lin(x)
    assert torch.equal(y[1], torch.full_like(y[1], float("inf")))
    assert torch.isnan(y[2]).all()
    rest = [i for i in range(m) if i not in (1, 2)]
    check(y[rest], x[rest], q, s, 128)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("shape", [(5, 7), (33, 130), (16, 640)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_quantiser(sbq, group, shape, dtype):
    """Scales and codes by their formula, in fp32 as the definition says."""
    n, k = shape
    w = (acts(n, k, F32, seed=11) * 0.02).to(dtype)
    w[0] = 0.0
    q, s = sbq.quantize_per_group(w, group)
    groups = -(-k // group)
    wf = torch.zeros(n, groups * group, device="cuda")
    wf[:, :k] = w.float()
    wf = wf.view(n, groups, group)
    s_ref = (wf.abs().amax(2).clamp_min(1e-8) / 7.0).to(BF16)
    q_ref = (wf / s_ref.float()[:, :, None]).round().clamp(-7, 7).to(torch.int8).view(n, -1)[:, :k]
    assert torch.equal(s, s_ref) and torch.equal(q, q_ref)


@pytest.mark.parametrize("m", [2, 30, 200])
def test_weights_that_are_not_finite(sbq, m):
    """An infinity or a NaN in a group makes its channel's results NaN, and no other's."""
    w = acts(40, 256, F32, seed=50) * 0.02
    clean = sbq.Int4Linear(w, None, group=64)
    w[3, 70], w[17, 255], w[39, 0] = float("nan"), float("inf"), -float("inf")
    lin = sbq.Int4Linear(w, None, group=64)
    nan = torch.isnan(lin.scale)
    assert nan.nonzero().tolist() == [[3, 1], [17, 3], [39, 0]]
    x = acts(m, 256, F16, seed=51)
    y, want = lin(x), clean(x)
    bad = [3, 17, 39]
    assert torch.isnan(y[:, bad]).all()
    keep = [i for i in range(40) if i not in bad]
    assert torch.equal(y[:, keep], want[:, keep])


def test_pack_unpack_round_trip(sbq):
    for n, k, group in ((1, 1, 32), (31, 200, 64), (130, 1025, 128)):
        q, s = weight(n, k, group, seed=12)
        packed, scales, _ = sbq.pack_int4(q, s, group)
        q2, s2 = sbq.unpack_int4(packed, scales, n, k, group)
        assert torch.equal(q, q2) and torch.equal(s, s2)


@pytest.mark.parametrize("m", [1, 8, 16, 17, 128, 129, 400])
@pytest.mark.parametrize("x_dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n,k,group", [(96, 256, 32), (64, 640, 128), (201, 72, 64)])
def test_gateup(sbq, m, x_dtype, n, k, group):
    qg, sg = weight(n, k, group, seed=13)
    qu, su = weight(n, k, group, seed=14)
    gate, up = (sbq.Int4Linear.from_quantized(q, s, None, group=group) for q, s in ((qg, sg), (qu, su)))
    down = sbq.Int4Linear.from_quantized(*weight(32, n, group, seed=15), None, group=group)
    x = acts(m, k, x_dtype, seed=16)
    wg, wu = dense(qg, sg, group), dense(qu, su, group)
    g, u = x.double() @ wg.t(), x.double() @ wu.t()
    ref = g * g.sigmoid() * u
    tg, tu = tolerance(x, wg, F32, g), tolerance(x, wu, F32, u)
    # d silu / d gate is at most 1.1; expf, the division and the products add a few fp32 roundings
    err = 1.1 * tg * u.abs() + (g * g.sigmoid()).abs() * tu + 1.1 * tg * tu + 8 * 2.0 ** -23 * ref.abs()
    for h_dtype in (F32, F16, BF16):
        mlp = sbq.FusedGatedMLP(gate, up, down, h_dtype=h_dtype)
        h = mlp.gateup(x)
        assert h.dtype == h_dtype
        tol = err + ref.abs() * torch.finfo(h_dtype).eps / 2 + (2.0 ** -25 if h_dtype == F16 else 0.0)
        assert ((h.double() - ref).abs() <= tol).all()
        assert torch.equal(mlp(x), down(h))


# tiles of 96 to 256 tokens, less and more than one for every pair of SMs, whole and cut along k
MANY = [(2100, 2001, 640), (1300, 5003, 515), (200, 12100, 900), (512, 9500, 2600), (300, 4100, 4100), (90, 900, 9000), (4000, 2500, 700),
        (77, 40000, 300), (333, 700, 4001), (2500, 2100, 130)]


@pytest.mark.parametrize("m,n,k", MANY)
@pytest.mark.parametrize("x_dtype", [F16, BF16, F32])
def test_many_rows(sbq, m, n, k, x_dtype):
    q, s = weight(n, k, 64, seed=60)
    lin = sbq.Int4Linear.from_quantized(q, s, acts(1, n, F32, seed=61)[0], group=64)
    x = acts(m, k, x_dtype, seed=62)
    for y_dtype in (F32, F16):
        lin.out_dtype = y_dtype
        y = lin(x)
        check(y, x, q, s, 64, bias=lin.bias)
        assert torch.equal(y, lin(x))


@pytest.mark.parametrize("m,n,k", MANY)
@pytest.mark.parametrize("x_dtype", [BF16, F32])
def test_gateup_many_rows(sbq, m, n, k, x_dtype):
    qg, sg = weight(n, k, 128, seed=63)
    qu, su = weight(n, k, 128, seed=64)
    gate, up = (sbq.Int4Linear.from_quantized(q, s, None, group=128) for q, s in ((qg, sg), (qu, su)))
    down = sbq.Int4Linear.from_quantized(*weight(16, n, 128, seed=65), None, group=128)
    x = acts(m, k, x_dtype, seed=66)
    wg, wu = dense(qg, sg, 128), dense(qu, su, 128)
    g, u = x.double() @ wg.t(), x.double() @ wu.t()
    ref = g * g.sigmoid() * u
    tg, tu = tolerance(x, wg, F32, g), tolerance(x, wu, F32, u)
    err = 1.1 * tg * u.abs() + (g * g.sigmoid()).abs() * tu + 1.1 * tg * tu + 8 * 2.0 ** -23 * ref.abs()  # as in test_gateup
    for h_dtype in (F32, F16):
        h = sbq.FusedGatedMLP(gate, up, down, h_dtype=h_dtype).gateup(x)
        tol = err + ref.abs() * torch.finfo(h_dtype).eps / 2 + (2.0 ** -25 if h_dtype == F16 else 0.0)
        bad = ((h.double() - ref).abs() - tol).max().item()
        assert bad <= 0, bad


@pytest.mark.parametrize("m", [3, 16, 24, 150])
def test_strided_rows_and_untouched_surroundings(sbq, m):
    q, s = weight(40, 96, 32, seed=17)
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=32)
    for x_dtype in (F16, BF16, F32):
        big = acts(m, 160, x_dtype, seed=18)
        x = big[:, 32:128]
        for y_dtype in (F32, F16, BF16):
            frame = torch.full((m + 2, 64), 7.0, dtype=y_dtype, device="cuda")
            lin.forward_into(x, frame[1:m + 1, 3:43])
            check(frame[1:m + 1, 3:43], x, q, s, 32)
            frame[1:m + 1, 3:43] = 7.0
            assert (frame == 7.0).all()
    # a transposed view and a leading shape
    xt = acts(96, m, F16, seed=19).t()
    check(lin(xt), xt.contiguous(), q, s, 32)
    x3 = acts(2 * m, 96, F16, seed=20).view(2, m, 96)
    assert torch.equal(lin(x3), lin(x3.view(-1, 96)).view(2, m, 40))


@pytest.mark.parametrize("m", [1, 12, 30, 140])
@pytest.mark.parametrize("k", [1, 7, 64, 90, 333, 4100, 13001])
def test_rows_at_any_address(sbq, m, k):
    """Widths that are multiples of nothing, rows at odd distances and odd first addresses; what lies beside the rows
    (infinities here) has no part in the result."""
    q, s = weight(33, k, 32, seed=50)
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=32)
    for x_dtype in (F16, BF16, F32):
        wide = torch.full((m, k + 5), float("inf"), dtype=x_dtype, device="cuda")
        x = acts(m, k, x_dtype, seed=51)
        wide[:, 3:3 + k] = x
        check(lin(wide[:, 3:3 + k]), x, q, s, 32)
        flat = torch.full((m * k + 1,), float("inf"), dtype=x_dtype, device="cuda")
        flat[1:] = x.flatten()
        check(lin(flat[1:].view(m, k)), x, q, s, 32)
        check(lin(x.t().contiguous().t()), x, q, s, 32)
        check(lin(x[:1].expand(m, k)), x[:1].expand(m, k).contiguous(), q, s, 32)


def test_empty_and_host_inputs(sbq):
    q, s = weight(24, 64, 64, seed=21)
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=64)
    assert lin(torch.empty(0, 64, device="cuda", dtype=F16)).shape == (0, 24)
    assert lin(torch.empty(3, 0, 64, device="cuda")).shape == (3, 0, 24)
    x = acts(5, 64, F32, seed=22)
    assert torch.equal(lin(x.cpu()), lin(x).cpu())
    assert lin(x[0]).shape == (24,) and torch.equal(lin(x[0]), lin(x[:1])[0])


@pytest.mark.parametrize("m", [1, 16, 100, 300])
def test_same_results_every_time(sbq, m):
    q, s = weight(300, 1024, 128, seed=23)
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=128)
    for dt in (F16, F32):
        x = acts(m, 1024, dt, seed=24)
        first = lin(x)
        for _ in range(5):
            assert torch.equal(lin(x), first)


@pytest.mark.parametrize("m", [1, 9, 48, 200])
@pytest.mark.parametrize("x_dtype", [F16, BF16, F32])
def test_streams_and_graphs(sbq, m, x_dtype):
    """The same weights on two streams at once, and captured; a replay reads what its input holds then."""
    q, s = weight(208, 512, 64, seed=25)
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=64)
    xs = [acts(m, 512, x_dtype, seed=26 + i) for i in range(2)]
    want = [lin(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(lin(xs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])
    buf = xs[0].clone()
    graphs, outs = [], []
    for _ in range(2):  # two graphs of the same module, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = lin(buf)
            outs.append(lin(buf) + y)
        graphs.append(graph)
    for i in (0, 1, 0):
        buf.copy_(xs[i])
        for graph, out in zip(graphs, outs):
            graph.replay()
            assert torch.equal(out, want[i] + want[i])


def test_state_dict_round_trip(sbq):
    w = acts(70, 200, F32, seed=28) * 0.02
    a = sbq.make_linear("int4-g64", w, torch.ones(70))
    state = a.state_dict()
    assert set(state) == {"qweight", "scale", "bias"} and state["qweight"].dtype == torch.int8
    b = sbq.make_linear("int4-g64", torch.zeros(70, 200), torch.zeros(70))
    b.load_state_dict(state)
    x = acts(21, 200, F16, seed=29)
    assert torch.equal(a(x), b(x)) and torch.equal(b(x[:3]), a(x[:3]))
    for bad in ({**state, "qweight": state["qweight"][:, :100]}, {**state, "qweight": state["qweight"] * 2},
                {k: v for k, v in state.items() if k != "scale"}):
        with pytest.raises(RuntimeError):
            b.load_state_dict(bad)


def test_converted_modules(sbq):
    """.half() and .to(dtype) on a model leave the packed weight and the results as they were (the bias is rounded)."""
    q, s = weight(40, 96, 32, seed=40)
    bias = torch.arange(40.0) / 8  # exact in fp16
    lin = sbq.Int4Linear.from_quantized(q, s, bias, group=32)
    xs = [acts(m, 96, F16, seed=41) for m in (3, 30)]
    want = [lin(x) for x in xs]
    for convert in (lambda m: m.half(), lambda m: m.to(BF16), lambda m: m.to("cuda")):
        box = convert(torch.nn.Sequential(sbq.Int4Linear.from_quantized(q, s, bias, group=32)))
        assert all(torch.equal(box(x), w) for x, w in zip(xs, want))
    with pytest.raises(ValueError, match="do not match"):
        sbq.Int4Linear.from_packed(lin.packed, lin.scales, lin.rowmul.float(), 40, 96, None, 32)
    with pytest.raises(ValueError, match="do not match"):
        sbq.Int4Linear.from_packed(lin.packed, lin.scales, lin.rowmul, 40, 96, None, 64)


def test_first_call_may_be_a_captured_one(sbq):
    """Nothing needs a warm-up: kernels that have not run in this process, captured first (a process of its own)."""
    import subprocess
    import sys

    from conftest import ROOT

    code = """
import importlib, torch
sbq = importlib.import_module("spikingbrain-cpu_b200")
q = torch.randint(-8, 8, (300, 512), dtype=torch.int8, device="cuda")
s = torch.ones(300, 8, dtype=torch.bfloat16, device="cuda")
lin = sbq.Int4Linear.from_quantized(q, s, None, group=64)
w = torch.ones(300, device="cuda")
for m in (1, 40, 300):
    x = torch.randn(m, 512, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = lin(x)
        r, n = sbq.residual_norm(y, y, w)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, lin(x)) and torch.equal(n, sbq.residual_norm(y, y, w)[1])
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=str(ROOT), capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_formats_loader_and_groups(sbq):
    """Every way a user gets to the format: make_linear, the streaming loader, the module fusions."""
    for fmt in sbq.INT4_FORMATS:
        w = acts(48, 160, F32, seed=30).cpu() * 0.02
        a = sbq.make_linear(fmt, w)
        packer = sbq.loader.StreamingPacker(staging_bytes=1 << 20)
        b = packer.make_linear(fmt, w)
        packer.finish()
        assert isinstance(a, sbq.Int4Linear) and a.group == int(fmt[6:]) and torch.equal(a.packed, b.packed)
    parent = torch.nn.Module()
    parent.q_proj = sbq.make_linear("int4-g32", acts(40, 96, F32, seed=31), torch.arange(40.0))
    parent.k_proj = sbq.make_linear("int4-g32", acts(17, 96, F32, seed=32))
    parent.v_proj = sbq.make_linear("int4-g32", acts(16, 96, F32, seed=33))
    for m in (2, 30):
        x = acts(m, 96, F16, seed=34)
        want = [getattr(parent, n)(x) for n in sbq.groups.ATTENTION_SHARED_INPUTS]
        got = sbq.groups.SharedInputGroup([getattr(parent, n) for n in sbq.groups.ATTENTION_SHARED_INPUTS]).forward_all(x)
        for a, b in zip(want, got):
            assert torch.allclose(a, b, rtol=0, atol=2.0 ** -18 * float(a.abs().max()))
    sbq.groups.fuse_shared_inputs(parent, sbq.groups.ATTENTION_SHARED_INPUTS)
    x = acts(2, 96, F16, seed=34)
    assert [parent.get_submodule(n)(x).shape[1] for n in sbq.groups.ATTENTION_SHARED_INPUTS] == [40, 17, 16]
    block = torch.nn.Module()
    block.mlp = torch.nn.Module()
    for n, shape in (("gate_proj", (64, 96)), ("up_proj", (64, 96)), ("down_proj", (96, 64))):
        setattr(block.mlp, n, sbq.make_linear("int4-g64", acts(*shape, F32, seed=35) * 0.02))
    assert sbq.fuse_gated_mlp(block) == 1 and isinstance(block.mlp, sbq.FusedGatedMLP)
    assert block.mlp(x).shape == (2, 96)


@pytest.mark.parametrize("m,ld", [(3, 1 << 30), (40, 1 << 26), (140, 1 << 24)])
def test_offsets_past_32_bits(sbq, m, ld):
    """Rows so far apart that element offsets pass 2^31: the activation's and the result's."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    q, s = weight(72, 192, 64, seed=56)
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=64)
    far = torch.empty((m - 1) * ld + 512, dtype=F16, device="cuda")
    x, y = (far[o:].as_strided((m, c), (ld, 1)) for o, c in ((0, 192), (256, 72)))
    x.copy_(acts(m, 192, F16, seed=57))
    lin.forward_into(x, y)
    check(y, x.contiguous(), q, s, 64)


@pytest.mark.parametrize("m", [4, 20, 200])
def test_gateup_of_far_gates(sbq, m):
    """Gates far out on both sides: silu is 0 or the gate itself, and nothing overflows on the way."""
    k = 64
    q = torch.zeros(32, k, dtype=torch.int8, device="cuda")
    q[:, 0] = 7
    s = torch.full((32, 1), 0.5, dtype=BF16, device="cuda")
    up_q = torch.zeros_like(q)
    up_q[:, 1] = 2
    gate, up = (sbq.Int4Linear.from_quantized(t, s, None, group=64) for t in (q, up_q))
    down = sbq.Int4Linear.from_quantized(*weight(k, 32, 32, seed=58), None, group=32)
    x = torch.zeros(m, k, device="cuda", dtype=F16)
    x[:, 0] = torch.tensor([-10000.0, -30.0, -24.5, 8.0], device="cuda").repeat(m // 4)  # gates -35000, -105, -86, 28
    x[:, 1] = 1.0                                                                       # up 1
    g = x[:, :1].double() * 3.5
    ref = (g * g.sigmoid()).expand(m, 32)
    for h_dtype in (F32, F16, BF16):
        h = sbq.FusedGatedMLP(gate, up, down, h_dtype=h_dtype).gateup(x)
        # as in test_gateup, with exact gates; silu below 2^-120 may be 0
        tol = ref.abs() * (8 * 2.0 ** -23 + torch.finfo(h_dtype).eps / 2) + 2.0 ** -118 + (2.0 ** -25 if h_dtype == F16 else 0.0)
        assert ((h.double() - ref).abs() <= tol).all(), h_dtype


@pytest.mark.parametrize("m", [3, 20, 150])
def test_output_beside_the_activation(sbq, m):
    """Columns of one buffer as activation and output; shared bytes are refused."""
    q, s = weight(64, 128, 64, seed=52)
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=64)
    lin.out_dtype = F16
    both = acts(m, 192, F16, seed=53)
    x = both[:, :128].clone()
    lin.forward_into(both[:, :128], both[:, 128:])
    assert torch.equal(both[:, 128:], lin(x)) and torch.equal(both[:, :128], x)
    for out in (both[:, :64], both[:, 127:191], both.view(-1)[1:m * 64 + 1].view(m, 64)):
        with pytest.raises(ValueError, match="overlap"):
            lin.forward_into(both[:, :128], out)
    mlp = sbq.FusedGatedMLP(lin, lin, sbq.Int4Linear.from_quantized(*weight(128, 64, 64, seed=54), None, group=64))
    with pytest.raises(ValueError, match="overlap"):
        mlp.gateup_into(both[:, :128], both[:, 100:164])


def test_refusals(sbq):
    L = sbq._lib
    q, s = weight(32, 64, 32, seed=36)
    with pytest.raises(ValueError, match="group size"):
        sbq.Int4Linear.from_quantized(q, s, None, group=48)
    with pytest.raises(ValueError, match="bf16"):
        sbq.Int4Linear.from_quantized(q, s.float(), None, group=32)
    with pytest.raises(ValueError, match="bf16"):
        sbq.Int4Linear.from_quantized(q, s, None, group=64)
    with pytest.raises(ValueError, match=r"\[-8, 7\]"):
        sbq.Int4Linear.from_quantized(q + 8, s, None, group=32)
    with pytest.raises(ValueError, match="finite"):
        sbq.Int4Linear.from_quantized(q, s * float("inf"), None, group=32)
    with pytest.raises(ValueError, match="bias"):
        sbq.Int4Linear.from_quantized(q, s, torch.zeros(31), group=32)
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=32)
    with pytest.raises(ValueError, match="feature size"):
        lin(torch.zeros(2, 48, device="cuda"))
    with pytest.raises(ValueError, match="feature size"):
        lin(torch.zeros((), device="cuda"))
    with pytest.raises(ValueError, match="output must be"):
        lin.forward_into(torch.zeros(2, 64, device="cuda"), torch.zeros(2, 31, device="cuda"))
    with pytest.raises(ValueError, match="input must be"):
        lin.forward_into(torch.zeros(2, 80, device="cuda")[:, :48], torch.zeros(2, 32, device="cuda"))
    with pytest.raises(ValueError, match="ALIGNMENT"):
        lin.forward_into(torch.zeros(2, 80, device="cuda")[:, 1:65], torch.zeros(2, 32, device="cuda"))
    with pytest.raises(ValueError, match="int4"):
        sbq.FusedGatedMLP(lin, sbq.Int8Linear(torch.zeros(32, 64), None), lin)
    with pytest.raises(ValueError, match="grouped decode"):
        down = sbq.Int4Linear.from_quantized(*weight(64, 32, 32, seed=1), None, group=32)
        sbq.FusedGatedMLP(lin, lin, down).gateup_job(torch.zeros(1, 64, device="cuda"), torch.zeros(1, 32, device="cuda"))
    x = torch.zeros(2, 64, device="cuda")
    y = torch.zeros(2, 32, device="cuda")
    args = [x.data_ptr(), L.F32, 64, lin.packed.data_ptr(), lin.scales.data_ptr(), lin.rowmul.data_ptr(), 32, None, 2, 32, 64,
            y.data_ptr(), L.F32, 32, None, 0, None]
    for at, value, name in ((14, None, "INVALID"), (0, x.data_ptr() + 4, "ALIGNMENT"), (1, 3, "UNSUPPORTED"), (6, 16, "UNSUPPORTED"),
                            (10, 72, "INVALID"), (13, 31, "INVALID"), (3, lin.packed.data_ptr() + 16, "ALIGNMENT")):
        bad = list(args)
        bad[at] = value
        with pytest.raises(ValueError, match=name):
            L.call("sbq_linear_w4", *bad)
    ws = torch.empty(256, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError, match="WORKSPACE"):
        L.call("sbq_linear_w4", *args[:14], ws.data_ptr(), 256, None)
    assert L.load().sbq_check_device_error() == 0
