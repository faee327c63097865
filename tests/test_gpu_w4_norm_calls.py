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


@pytest.mark.parametrize("m,n,k", [(1, 512, 2048), (20, 512, 2048), (300, 4096, 4096)])
@pytest.mark.parametrize("x_dtype", [F16, F32])
def test_product_right_behind_the_packing(sbq, m, n, k, x_dtype):
    """Products read their weight before they wait for the kernel before them: one that follows the packing of its
    weight at once finds it complete, eager and in a graph, also where the buffers held another weight before."""
    L = sbq._lib
    ws = [rand(n, k, seed=10 + i, scale=0.02) for i in range(3)]
    x = rand(m, k, seed=20, dtype=x_dtype)
    lin = sbq.Int4Linear(ws[0], None, group=64)
    quantised = [sbq.quantize_per_group(w, 64) for w in ws]
    wants = []
    for q, s in quantised:
        other = sbq.Int4Linear.from_quantized(q, s, None, group=64)
        torch.cuda.synchronize()
        wants.append(other(x))

    def pack(i, kind):
        w, (q, s) = ws[i], quantised[i]
        bufs = (lin.packed.data_ptr(), lin.scales.data_ptr(), lin.rowmul.data_ptr(), torch.cuda.current_stream().cuda_stream)
        if kind:
            L.call("sbq_w4_pack", q.data_ptr(), k, s.data_ptr(), s.shape[1], n, k, 64, *bufs)
        else:
            L.call("sbq_w4_quantize_pack", w.data_ptr(), L.F32, n, k, k, 64, *bufs)

    torch.cuda.synchronize()
    got = []
    for i in range(60):
        pack(i % 3, i & 1)
        got.append((lin(x), wants[i % 3]))
    assert all(torch.equal(a, b) for a, b in got)
    graph, outs = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph):
        for i in range(6):
            pack(i % 3, i & 1)
            outs.append(lin(x))
    for _ in range(3):
        graph.replay()
        assert all(torch.equal(o, wants[i % 3]) for i, o in enumerate(outs))
    fresh = sbq.Int4Linear(ws[1], None, group=64)(x)  # as a user writes it
    assert torch.equal(fresh, wants[1])


@pytest.mark.parametrize("m", [1, 40, 300])
def test_int8_product_right_behind_the_packing(sbq, m):
    """The same for the int8 formats, whose products read their weight as early."""
    n, k = 1024, 2048
    ws, x = [rand(n, k, seed=30 + i, scale=0.02) for i in range(2)], rand(m, k, seed=33, dtype=F16)
    for kind in (sbq.Int8Linear, sbq.DynamicInt8Linear):
        lins = [kind(w, None) for w in ws]
        torch.cuda.synchronize()
        wants = [lin(x) for lin in lins]
        got = [(kind(ws[i & 1], None)(x), wants[i & 1]) for i in range(40)]
        assert all(torch.equal(a, b) for a, b in got)


@pytest.mark.parametrize("m", [65535 * 64, 65535 * 64 + 1])
def test_more_rows_than_a_grid_dimension(sbq, m):
    """64-row tiles beyond 65535, which is what a grid has in y: the linear and the gate/up form."""
    n, k = 16, 32
    q, s = torch.randint(-8, 8, (n, k), device="cuda", dtype=torch.int8), rand(n, 1, seed=40).abs().add(0.5).to(BF16)
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=32)
    x = rand(m, k, seed=41)
    w = q.double() * s.double()
    ref, mags = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    # fp32 x has 22 bits (2^-23 of each element); 4 tensor-core steps, the factor and the rounding of the result
    tol = mags * (2.0 ** -23 + 8 * 2.0 ** -22)
    assert ((lin(x).double() - ref).abs() <= tol).all()
    del mags
    down = sbq.Int4Linear.from_quantized(q.t().contiguous(), torch.ones(k, 1, dtype=BF16, device="cuda"), None, group=32)
    mlp = sbq.FusedGatedMLP(lin, lin, down, h_dtype=F32)
    h = ref * ref.sigmoid() * ref
    # d (silu(g) u) with g = u: at most 2.1 |g| of the product's error, and a few roundings
    assert ((mlp.gateup(x).double() - h).abs() <= 2.2 * tol * (ref.abs() + tol) + 8 * 2.0 ** -23 * h.abs()).all()


@pytest.mark.parametrize("fmt", ["int4-g64", "int8"])
def test_group_members_called_with_different_inputs(sbq, fmt):
    """A step that calls some members of a group only, and the next one that begins with another member."""
    parent = torch.nn.Module()
    names = ["q_proj", "k_proj"]
    lins = [sbq.make_linear(fmt, rand(48, 128, seed=50 + i)) for i in range(2)]
    for name, lin in zip(names, lins):
        setattr(parent, name, lin)
    sbq.groups.fuse_shared_inputs(parent, names)
    for i in range(10):
        for name, lin in (("q_proj", lins[0]), ("k_proj", lins[1])):
            x = rand(3, 128, seed=60 + 2 * i + (name == "k_proj"), dtype=F16)
            got, want = parent.get_submodule(name)(x), lin(x)
            assert (got - want).norm() <= 2.0 ** -18 * want.norm()
            del x


@pytest.mark.parametrize("writer", ["int4", "int8", "gateup int4", "gateup int8", "residual_norm"])
def test_calls_that_write_into_a_tensor_count_as_changes_of_it(sbq, writer):
    """The kernels write through addresses; the tensor's version moves all the same, and a group whose x was refilled
    this way computes anew."""
    parent = torch.nn.Module()
    parent.q_proj, parent.k_proj = lins = [sbq.make_linear("int4-g64", rand(48, 128, seed=70 + i)) for i in range(2)]
    sbq.groups.fuse_shared_inputs(parent, ["q_proj", "k_proj"])
    fmt = "int8" if writer.endswith("int8") else "int4-g64"
    step = sbq.make_linear(fmt, rand(128, 128, seed=72))
    mlp = sbq.FusedGatedMLP(*(sbq.make_linear(fmt, rand(128, 128, seed=73 + i)) for i in range(3)))
    src, x = rand(3, 128, seed=76, dtype=F16), rand(3, 128, seed=77, dtype=F16)
    write = {"int4": lambda: step.forward_into(src, x), "int8": lambda: step.forward_into(src, x),
             "gateup int4": lambda: mlp.gateup_into(src, x), "gateup int8": lambda: mlp.gateup_into(src, x),
             "residual_norm": lambda: sbq.residual_norm(src, x, residual_out=x)}[writer]
    parent.q_proj(x)
    version, before = x._version, x.clone()
    write()
    assert x._version > version and not torch.equal(x, before)
    got, want = parent.k_proj(x), lins[1](x)
    assert (got - want).norm() <= 2.0 ** -18 * want.norm()
    with torch.inference_mode():  # tensors without a version
        x = x.clone()
        write()


@pytest.mark.parametrize("act", ["sigmoid", "silu"])
@pytest.mark.parametrize("d", [680, 681, 5441])
def test_gates_towards_zero(sbq, act, d):
    """The gated term alone, fp32, for gates whose weight beside a residual would hide their error."""
    m = 4
    g = torch.linspace(-85.0, 0.0, m * d, device="cuda").view(m, d)
    y = 1.0 + rand(m, d, seed=90).abs()
    r, _ = sbq.residual_norm(y, torch.zeros_like(y), gate=g, gate_act=act, residual_scale=0.0)
    gd = g.double()
    ref = y.double() * torch.sigmoid(gd) * (gd if act == "silu" else 1.0)
    # the exponent -g log2 e is rounded (2^-24) and so is log2 e (2^-26): |g| (2^-24 + 2^-26) = 0.3125 |g| 2^-22 of the power
    # of two, which is good to 2^-22; the sum, the reciprocal and the products add at most 2^-22 together
    tol = ref.abs() * (2.0 + 0.32 * gd.abs()) * 2.0 ** -22
    assert ((r.double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("m,n,k", [(4, 64, 384), (40, 64, 384), (405, 5433, 272)])
@pytest.mark.parametrize("x_dtype", [F16, BF16, F32])
def test_elements_far_below_their_rows_largest(sbq, m, n, k, x_dtype):
    """A row whose largest element meets zero weights only.  fp32 rows, and bf16 ones of more than 16, are read as fp16
    parts of the scaled row: what lies far below the largest keeps an absolute 2^-39 of it, and no more."""
    q = torch.randint(-8, 8, (n, k), device="cuda", dtype=torch.int8, generator=torch.Generator(device="cuda").manual_seed(91))
    s = (rand(n, -(-k // 64), seed=92).abs() * 0.01 + 0.002).to(BF16)
    q[:, 5] = 0
    lin = sbq.Int4Linear.from_quantized(q, s, None, group=64)
    w = q.double() * s.double().repeat_interleave(64, dim=1)[:, :k]
    for far in (2.0 ** 10, 2.0 ** 15, 2.0 ** 20, 2.0 ** 30, 2.0 ** 45, 2.0 ** 90):
        x = rand(m, k, seed=93)
        x[:, 5] = far if x_dtype != F16 else min(far, 2.0 ** 15)
        x = x.to(x_dtype)
        ref = x.double() @ w.t()
        mags = x.double().abs() @ w.abs().t()
        steps = (2 if x_dtype == F32 else 1) * -(-k // 16) + -(-k // 128) + 16
        tol = mags * steps * 2.0 ** -22 + ref.abs() * 2.0 ** -24
        if x_dtype == F32 or (x_dtype == BF16 and m > 16):
            tol = tol + mags * 2.0 ** -23 + 2.0 ** -39 * x[:, 5:6].double() * w.abs().sum(1)
        assert ((lin(x).double() - ref).abs() <= tol).all(), far


@pytest.mark.parametrize("fmt", ["int4-g64", "int8"])
def test_group_members_called_on_streams_and_in_graphs(sbq, fmt):
    """A kept result belongs to the stream, and the graph or not, that it was computed in: elsewhere a member computes anew."""
    parent, names = torch.nn.Module(), ["q_proj", "k_proj"]
    lins = [sbq.make_linear(fmt, rand(48, 128, seed=80 + i)) for i in range(2)]
    for name, lin in zip(names, lins):
        setattr(parent, name, lin)
    group = sbq.groups.fuse_shared_inputs(parent, names)
    computed = []
    forward_all = group.forward_all
    group.forward_all = lambda x: computed.append(x) or forward_all(x)

    def same(got, want):
        return (got - want).norm() <= 2.0 ** -18 * want.norm()

    x, side = rand(3, 128, seed=82, dtype=F16), torch.cuda.Stream()
    parent.q_proj(x)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = parent.k_proj(x)
    torch.cuda.synchronize()
    assert len(computed) == 2 and same(got, lins[1](x))
    # one member before the capture, the other one in it: the graph holds the product, of x as it is at each replay
    y = rand(3, 128, seed=83, dtype=F16)
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        parent.q_proj(y)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        out = parent.k_proj(y)
    with torch.cuda.stream(side):
        after = parent.q_proj(y)  # and nothing of the graph's goes to an eager call
    torch.cuda.synchronize()
    assert same(after, lins[0](y))
    for seed in (84, 85):
        y.copy_(rand(3, 128, seed=seed, dtype=F16))
        graph.replay()
        assert same(out, lins[1](y))
