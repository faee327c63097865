"""4-bit products on CTA pairs: sizes that the schedule gives to that kernel, whole and cut along k, and on them every
type, group size and kind of data.  (Small products with the same row counts run a kernel of single CTAs, which the
tests beside these reach.)

Tolerances as derived in test_gpu_int4.py.
"""

import ctypes

import pytest
import torch

from test_gpu_int4 import acts, check, dense, tolerance, weight

gpu = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
# m, n, k: one tile for some pairs; a full round of tiles and a rest; 96-token tiles cut in four; tiles of 192 tokens and, of
# gate and up with fp32 rows, a full round with cut tiles behind it; the same of a linear
SHAPES = [(405, 5433, 262), (1647, 2956, 129), (69, 4196, 3250), (1884, 1266, 1439), (264, 9707, 2903)]
GATEUP_SHAPES = SHAPES + [(67, 9636, 2981)]  # the same of gate and up, any rows


def plan(sbq, m, n, k, x_dtype, matrices):
    out = (ctypes.c_int * 4)()
    sbq._lib.call("sbq_linear_w4_plan", m, n, k, {F32: sbq._lib.F32, F16: sbq._lib.F16, BF16: sbq._lib.BF16}[x_dtype], matrices, out)
    return list(out)


def on_pairs(sbq, x, n, matrices=1):
    assert plan(sbq, x.shape[0], n, x.shape[1], x.dtype, matrices)[0] == 2


@pytest.mark.parametrize("matrices", [1, 2])
@pytest.mark.parametrize("x_dtype", [F16, F32])
def test_shapes_reach_every_form(sbq, x_dtype, matrices):
    """Evaluated for 148 SMs where there is no GPU."""
    plans = [plan(sbq, *s, x_dtype, matrices) for s in (GATEUP_SHAPES if matrices == 2 else SHAPES)]
    assert all(p[0] == 2 for p in plans)
    forms = {(parts > 1, rounds > 0) for _, _, parts, rounds in plans}
    assert {(False, True), (True, False), (True, True)} <= forms
    assert matrices == 2 or (False, False) in forms
    assert {p[1] for p in plans} & {96, 128} and {p[1] for p in plans} & {192, 256}


@gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("x_dtype", [F16, BF16, F32])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear(sbq, m, n, k, x_dtype, group):
    q, s = weight(n, k, group, seed=m)
    lin = sbq.Int4Linear.from_quantized(q, s, acts(1, n, F32, seed=1)[0] if group == 64 else None, group=group)
    x = acts(m, k, x_dtype, seed=2)
    on_pairs(sbq, x, n)
    for y_dtype in (F32, F16, BF16):
        lin.out_dtype = y_dtype
        y = lin(x)
        check(y, x, q, s, group, lin.bias)
        assert torch.equal(lin(x), y)


def mlp_of(sbq, n, k, group, seed, h_dtype=F16):
    pairs = [weight(n, k, group, seed=seed + i) for i in range(2)]
    gate, up = (sbq.Int4Linear.from_quantized(*p, None, group=group) for p in pairs)
    down = sbq.Int4Linear.from_quantized(*weight(16, n, group, seed=seed + 2), None, group=group)
    return sbq.FusedGatedMLP(gate, up, down, h_dtype=h_dtype), [dense(*p, group) for p in pairs]


def check_gateup(h, x, wg, wu):
    g, u = x.double() @ wg.t(), x.double() @ wu.t()
    ref = g * g.sigmoid() * u
    tg, tu = tolerance(x, wg, F32, g), tolerance(x, wu, F32, u)
    tol = 1.1 * tg * u.abs() + (g * g.sigmoid()).abs() * tu + 1.1 * tg * tu + 8 * 2.0 ** -23 * ref.abs()
    tol = tol + ref.abs() * torch.finfo(h.dtype).eps / 2 + (2.0 ** -25 if h.dtype == F16 else 0.0)
    worst = ((h.double() - ref).abs() - tol).max().item()
    assert worst <= 0, worst


@gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("x_dtype", [F16, BF16, F32])
@pytest.mark.parametrize("m,n,k", GATEUP_SHAPES)
def test_gateup(sbq, m, n, k, x_dtype, group):
    mlp, ws = mlp_of(sbq, n, k, group, seed=m)
    x = acts(m, k, x_dtype, seed=3) * 0.125  # products of a few units: fp16 results stay in range
    on_pairs(sbq, x, n, 2)
    for h_dtype in (F32, F16, BF16):
        mlp.h_dtype = h_dtype
        h = mlp.gateup(x)
        check_gateup(h, x, *ws)
        assert torch.equal(mlp.gateup(x), h)


FEW = [(405, 5433, 272), (69, 4196, 3264)]  # whole and cut, of a width that is read in place


def test_few_shapes_are_whole_and_cut(sbq):
    for x_dtype in (F16, F32):
        for matrices in (1, 2):
            (k0, _, parts0, _), (k1, _, parts1, _) = (plan(sbq, *s, x_dtype, matrices) for s in FEW)
            assert (k0, k1) == (2, 2) and parts0 == 1 < parts1


@gpu
@pytest.mark.parametrize("m,n,k", FEW)
@pytest.mark.parametrize("x_dtype", [F16, BF16, F32])
def test_infinities_and_nan_stay_in_their_rows(sbq, m, n, k, x_dtype):
    q, s = weight(n, k, 128, seed=7)
    q[:, 17], q[:, 40] = 3, 2
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=128)
    x = acts(m, k, x_dtype, seed=10)
    x[1, 17], x[m - 1, 17], x[2, 40] = float("inf"), -float("inf"), float("nan")
    on_pairs(sbq, x, n)
    y = lin(x)
    assert (y[1] == float("inf")).all() and (y[m - 1] == -float("inf")).all() and torch.isnan(y[2]).all()
    rest = [i for i in range(m - 1) if i not in (1, 2)]
    check(y[rest], x[rest], q, s, 128)


@gpu
@pytest.mark.parametrize("m,n,k", FEW)
@pytest.mark.parametrize("x_dtype", [BF16, F32])
def test_activations_of_any_range(sbq, m, n, k, x_dtype):
    q, s = weight(n, k, 64, seed=6)
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=64)
    x = acts(m, k, F32, seed=9)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2] = 0.0
    x[-1, ::2] *= 1e-12
    x = x.to(x_dtype)
    on_pairs(sbq, x, n)
    y, w = lin(x), dense(q, s, 64)
    ref = x.double() @ w.t()
    assert ((y.double() - ref).abs() <= tolerance(x, w, F32, ref)).all()


@gpu
@pytest.mark.parametrize("m,n,k", FEW)
def test_scales_over_many_powers_of_two(sbq, m, n, k):
    q, s = weight(n, k, 32, seed=5, spread=True)
    s[3, :] = 0.0
    s[4, 1:] = 0.0
    s[5] = -s[5]
    s[6] = s[6].float().mul(2.0 ** -100).to(BF16)
    s[7] = s[7].float().mul(2.0 ** 90).to(BF16)
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=32)
    for dt in (F16, BF16, F32):
        x = acts(m, k, dt, seed=8)
        on_pairs(sbq, x, n)
        y, w = lin(x), dense(q, s, 32)
        ref = x.double() @ w.t()
        assert ((y.double() - ref).abs() <= tolerance(x, w, F32, ref)).all()


@gpu
@pytest.mark.parametrize("m,n,k", [(405, 5433, 320), (69, 4196, 3264)])
@pytest.mark.parametrize("x_dtype", [F16, BF16, F32])
def test_sums_that_cancel(sbq, m, n, k, x_dtype):
    """The first half of every row of x against the second half: partial sums hundreds of times the result.  16-bit
    results are summed in one truncating piece, fp32 ones in segments; both within the bound of their steps."""
    q, s = weight(n, k // 2, 32, seed=11)
    q, s = torch.cat([q, -q.clamp(min=-7)], 1), torch.cat([s, s], 1)
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=32)
    x = acts(m, k // 2, F32, seed=12).abs() + 1.0
    x = torch.cat([x, x + acts(m, k // 2, F32, seed=13) * 2.0 ** -8], 1).to(x_dtype)
    on_pairs(sbq, x, n)
    for y_dtype in (F32, F16, BF16):
        lin.out_dtype = y_dtype
        y, w = lin(x), dense(q, s, 32)
        ref = x.double() @ w.t()
        assert ((y.double() - ref).abs() <= tolerance(x, w, y_dtype, ref)).all()


@gpu
@pytest.mark.parametrize("m,n,k", FEW)
@pytest.mark.parametrize("x_dtype", [F16, BF16, F32])
def test_strided_rows_and_untouched_surroundings(sbq, m, n, k, x_dtype):
    q, s = weight(n, k, 64, seed=17)
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=64)
    mlp, ws = mlp_of(sbq, n, k, 32, seed=18)
    x = (acts(m, k + 64, x_dtype, seed=20) * 0.125)[:, 32:32 + k]
    on_pairs(sbq, x, n)
    on_pairs(sbq, x, n, 2)
    for y_dtype in (F32, F16, BF16):
        frame = torch.full((m + 2, n + 24), 7.0, dtype=y_dtype, device="cuda")
        inner = frame[1:m + 1, 3:3 + n]
        lin.forward_into(x, inner)
        check(inner, x, q, s, 64)
        mlp.gateup_into(x, inner)
        check_gateup(inner, x, *ws)
        inner.fill_(7.0)
        assert (frame == 7.0).all()


@gpu
@pytest.mark.parametrize("m,n,k", FEW)
@pytest.mark.parametrize("x_dtype", [F16, F32])
def test_streams_and_graphs(sbq, m, n, k, x_dtype):
    """Two streams at once, each call with a workspace of its own; two graphs replayed in turn with new inputs."""
    q, s = weight(n, k, 64, seed=25)
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=64)
    xs = [acts(m, k, x_dtype, seed=26 + i) for i in range(2)]
    on_pairs(sbq, xs[0], n)
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
    for _ in range(2):
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


@gpu
def test_offsets_past_32_bits(sbq):
    """Rows so far apart that element offsets pass 2^31: the activation's and the result's."""
    m, n, k = FEW[1]
    ld = 1 << 25
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    q, s = weight(n, k, 64, seed=56)
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=64)
    far = torch.empty((m - 1) * ld + 16384, dtype=F16, device="cuda")
    x, y = (far[o:].as_strided((m, c), (ld, 1)) for o, c in ((0, k), (8192, n)))
    x.copy_(acts(m, k, F16, seed=57))
    on_pairs(sbq, x, n)
    lin.forward_into(x, y)
    check(y, x.contiguous(), q, s, 64)


@gpu
@pytest.mark.parametrize("m,n,k", FEW)
def test_gateup_of_far_gates(sbq, m, n, k):
    """Gates far out on both sides: silu is 0 or the gate itself, and nothing overflows on the way."""
    q = torch.zeros(n, k, dtype=torch.int8, device="cuda")
    q[:, 0] = 7
    s = torch.full((n, -(-k // 64)), 0.5, dtype=BF16, device="cuda")
    up_q = torch.zeros_like(q)
    up_q[:, 1] = 2
    gate, up = (sbq.Int4Linear.from_quantized(t, s, None, group=64) for t in (q, up_q))
    down = sbq.Int4Linear.from_quantized(*weight(16, n, 32, seed=58), None, group=32)
    x = torch.zeros(m, k, device="cuda", dtype=F16)
    x[:, 0] = torch.tensor([-10000.0, -30.0, -24.5, 8.0], device="cuda").repeat(m // 4 + 1)[:m]  # gates -35000, -105, -86, 28
    x[:, 1] = 1.0                                                                                # up 1
    on_pairs(sbq, x, n, 2)
    g = x[:, :1].double() * 3.5
    ref = (g * g.sigmoid()).expand(m, n)
    for h_dtype in (F32, F16, BF16):
        h = sbq.FusedGatedMLP(gate, up, down, h_dtype=h_dtype).gateup(x)
        tol = ref.abs() * (8 * 2.0 ** -23 + torch.finfo(h_dtype).eps / 2) + 2.0 ** -118 + (2.0 ** -25 if h_dtype == F16 else 0.0)
        assert ((h.double() - ref).abs() <= tol).all(), h_dtype
