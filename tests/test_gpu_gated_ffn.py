"""GPU tests of the gated feed-forward block and its gradients against float64 (bounds carried through every rounding: tests/token_reference.py)."""
import pytest
import torch

import token_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.fixture(scope="module")
def dev(native_lib):
    assert torch.cuda.is_available(), "GPU tests need a visible MI355X"
    return torch.device("cuda", 0)


def _inputs(dev, M, D, F, O, dtype, seed=0):
    g = torch.Generator(dev).manual_seed(seed)
    n = lambda *s, scale=1.0: (torch.randn(s, generator=g, device=dev) * scale).to(dtype)
    return n(M, D), n(F, D, scale=D ** -0.5), n(F, D, scale=D ** -0.5), n(O, F, scale=F ** -0.5), n(M, O)


def _check(got, want, what):
    got = got.double()
    assert got.shape == want.val.shape, (what, got.shape, want.val.shape)
    bad = ~((got - want.val).abs() <= want.err)
    assert not bad.any(), "%s: %d of %d outside their bound, worst %.2f of it, first at %s" % (
        what, int(bad.sum()), bad.numel(), float(((got - want.val).abs() / want.err).max()), bad.nonzero()[0].tolist())


def _run(x, wg, wu, wd, dy, kind):
    from gddim_amd import ops
    y, saved = ops.gated_ffn(x, wg, wu, wd, act=kind, save=True)
    return (y,) + ops.gated_ffn_backward(dy, x, wg, wu, wd, saved, act=kind)


SIZES = [
    # M, D, F, O
    (1, 1, 1, 1), (1, 64, 64, 64), (1, 512, 96, 40), (2, 8, 16, 8), (3, 40, 72, 24), (5, 33, 17, 9), (16, 128, 256, 128), (17, 136, 88, 264),
    (31, 7, 130, 3), (33, 256, 344, 256), (64, 72, 520, 72), (65, 100, 30, 101), (130, 64, 129, 66), (257, 200, 136, 96), (300, 96, 700, 250),
    (1000, 24, 24, 24), (12, 1032, 24, 16), (700, 16, 1032, 8),
]


@pytest.mark.parametrize("typ", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_forward_and_gradients(dev, size, typ):
    from gddim_amd import ops
    kind = ("silu", "gelu", "gelu_tanh")[SIZES.index(size) % 3]
    x, wg, wu, wd, dy = _inputs(dev, *size, TYPES[typ])
    want = ref.gated_ffn(x, wg, wu, wd, kind, TYPES[typ], dy)
    got = _run(x, wg, wu, wd, dy, kind)
    for g, w, what in zip(got, want, ("y", "dx", "dw_gate", "dw_up", "dw_down")):
        assert g.dtype == TYPES[typ]
        _check(g, w, what)
    assert torch.equal(ops.gated_ffn(x, wg, wu, wd, act=kind), got[0])
    for a, b in zip(got, _run(x, wg, wu, wd, dy, kind)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("typ", ["f32", "bf16", "f16"])
def test_activations_over_their_range(dev, typ, kind):
    """projections from -30 to 30, where exponentials over- and underflow"""
    x, wg, wu, wd, dy = _inputs(dev, 70, 16, 40, 24, TYPES[typ], 3)
    x = x * torch.linspace(0, 12, 70, device=dev, dtype=torch.float32)[:, None].to(x.dtype)
    want = ref.gated_ffn(x, wg, wu, wd, kind, TYPES[typ], dy)
    for g, w, what in zip(_run(x, wg, wu, wd, dy, kind), want, ("y", "dx", "dw_gate", "dw_up", "dw_down")):
        _check(g, w, what)


@pytest.mark.parametrize("typ", ["bf16", "f32"])
@pytest.mark.parametrize("size", [(4100, 72, 1560, 64), (4100, 2888, 136, 2888), (264, 2888, 1288, 2888), (8200, 64, 264, 1352)], ids=str)
def test_tiles_that_fill_the_chip(dev, size, typ):
    x, wg, wu, wd, dy = _inputs(dev, *size, TYPES[typ], 1)
    want = ref.gated_ffn(x, wg, wu, wd, "silu", TYPES[typ], dy)
    for g, w, what in zip(_run(x, wg, wu, wd, dy, "silu"), want, ("y", "dx", "dw_gate", "dw_up", "dw_down")):
        _check(g, w, what)


@pytest.mark.parametrize("typ", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("size", [(2048, 1024, 2048, 1024), (2100, 1001, 2003, 999), (429, 884, 2764, 188), (3133, 328, 280, 328), (1500, 80, 291, 80)], ids=str)
def test_tiles_of_each_width(dev, size, typ):
    """square matrices and narrow ones, aligned and not"""
    x, wg, wu, wd, dy = _inputs(dev, *size, TYPES[typ], 6)
    want = ref.gated_ffn(x, wg, wu, wd, "gelu", TYPES[typ], dy)
    got = _run(x, wg, wu, wd, dy, "gelu")
    for g, w, what in zip(got, want, ("y", "dx", "dw_gate", "dw_up", "dw_down")):
        _check(g, w, what)
    for a, b in zip(got, _run(x, wg, wu, wd, dy, "gelu")):
        assert torch.equal(a, b)


@pytest.mark.parametrize("typ", ["bf16", "f32"])
@pytest.mark.parametrize("size", [(8200, 64, 2600, 64), (8200, 72, 2600, 72), (8200, 200, 1304, 1304), (8200, 65, 1301, 67), (16000, 24, 2056, 24)], ids=str)
def test_more_tiles_than_workgroups(dev, size, typ):
    """a workgroup walks several tiles, of one stage of k and of more"""
    x, wg, wu, wd, dy = _inputs(dev, *size, TYPES[typ], 2)
    want = ref.gated_ffn(x, wg, wu, wd, "gelu_tanh", TYPES[typ], dy)
    got = _run(x, wg, wu, wd, dy, "gelu_tanh")
    for g, w, what in zip(got, want, ("y", "dx", "dw_gate", "dw_up", "dw_down")):
        _check(g, w, what)
    for a, b in zip(got, _run(x, wg, wu, wd, dy, "gelu_tanh")):
        assert torch.equal(a, b)


@pytest.mark.parametrize("typ", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("size", [(1, 8, 8, 8), (1, 520, 4104, 1032), (4, 1024, 40, 8), (16, 264, 4104, 2056), (17, 64, 2064, 1032), (48, 72, 136, 24), (64, 1000, 1024, 4104),
                                  (100, 64, 136, 72), (256, 64, 200, 64), (255, 128, 352, 128), (16, 2048, 8200, 2048), (40, 1032, 6152, 1032), (90, 1024, 4096, 1024)], ids=str)
def test_few_rows(dev, size, typ):
    from gddim_amd import ops
    x, wg, wu, wd, _ = _inputs(dev, *size, TYPES[typ], 4)
    for kind in ("silu", "gelu"):
        y, saved = ops.gated_ffn(x, wg, wu, wd, act=kind, save=True)
        _check(y, ref.gated_ffn(x, wg, wu, wd, kind, TYPES[typ]), "y")
        gate, up = ref.product(ref.V(x.double()), ref.V(wg.double())), ref.product(ref.V(x.double()), ref.V(wu.double()))
        _check(saved[0], gate, "gate")
        _check(saved[1], up, "up")
        _check(saved[2], (ref.act(gate, kind)[0] * up).rounded(TYPES[typ]), "hidden")


@pytest.mark.parametrize("typ", ["bf16", "f32"])
@pytest.mark.parametrize("size", [(1, 64, 72, 40), (65, 72, 130, 66), (300, 33, 17, 9), (4100, 72, 520, 64)], ids=str)
def test_nothing_is_written_beside_the_results(dev, native_lib, size, typ):
    """the C entry points on buffers between guard values"""
    from gddim_amd._abi import FfnDesc
    M, D, F, O = size
    dtype = TYPES[typ]
    x, wg, wu, wd, dy = _inputs(dev, *size, dtype, 9)
    pad = 1024

    def guarded(rows, cols, dt=dtype):
        buf = torch.full((rows * cols + 2 * pad,), 12345.0, dtype=dt, device=dev)
        return buf, buf[pad:pad + rows * cols].view(rows, cols)

    for unaligned in (0, 1):
        d = bytes(FfnDesc(0 if typ == "f32" else 1, 0, M, D, F, O, unaligned, D, D, F))
        s = torch.cuda.current_stream().cuda_stream
        bufs = [guarded(M, F, torch.float32), guarded(M, F, torch.float32), guarded(M, F), guarded(M, O), guarded(M, D), guarded(F, D), guarded(F, D), guarded(O, F)]
        ws = [guarded(1, max(4, native_lib.gd_gated_ffn_workspace(d, b) // 4), torch.float32) for b in (0, 1)]
        p = [v.data_ptr() for _, v in bufs]
        assert native_lib.gd_gated_ffn(d, x.data_ptr(), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), p[0], p[1], p[2], p[3], ws[0][1].data_ptr(), s) == 0
        assert native_lib.gd_gated_ffn_backward(d, dy.data_ptr(), O, x.data_ptr(), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), p[0], p[1], p[2], p[4], p[5], p[6], p[7],
                                                ws[1][1].data_ptr(), s) == 0
        torch.cuda.synchronize()
        for buf, v in bufs + ws:
            assert (buf[:pad] == buf[0]).all() and (buf[-pad:] == buf[0]).all() and buf[0] == torch.tensor(12345.0, dtype=buf.dtype)
        want = ref.gated_ffn(x, wg, wu, wd, "silu", dtype, dy)
        for i, w in zip((3, 4, 5, 6, 7), want):
            _check(bufs[i][1], w, "result %d" % i)


def test_offsets_past_32_bits(dev):
    """hidden rows past 2^31 elements, first and last rows checked, all others zero"""
    from gddim_amd import ops
    M, D, F, O = 540000, 64, 4096, 64
    rows = torch.tensor([0, 1, 255, 256, 300000, M - 2, M - 1], device=dev)
    x, wg, wu, wd, dy = _inputs(dev, len(rows), D, F, O, torch.bfloat16, 10)
    want = ref.gated_ffn(x, wg, wu, wd, "silu", torch.bfloat16, dy)
    big_x, big_dy = torch.zeros(M, D, dtype=x.dtype, device=dev), torch.zeros(M, O, dtype=x.dtype, device=dev)
    big_x[rows], big_dy[rows] = x, dy
    y, saved = ops.gated_ffn(big_x, wg, wu, wd, save=True)
    assert saved[0].numel() > 1 << 31
    dx, *dw = ops.gated_ffn_backward(big_dy, big_x, wg, wu, wd, saved)
    _check(y[rows], want[0], "y")
    _check(dx[rows], want[1], "dx")
    for g, w, what in zip(dw, want[2:], ("dw_gate", "dw_up", "dw_down")):
        _check(g, w, what)
    others = torch.ones(M, dtype=torch.bool, device=dev)
    others[rows] = False
    assert (y[others] == 0).all() and (dx[others] == 0).all()


def test_two_streams_at_once(dev):
    a, b = _inputs(dev, 700, 256, 688, 256, torch.bfloat16, 11), _inputs(dev, 700, 256, 688, 256, torch.bfloat16, 12)
    want = [_run(*t, "silu") for t in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, t in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(_run(*t, "silu"))
    torch.cuda.synchronize()
    for i in range(2):
        for run in got[i]:
            assert all(torch.equal(p, q) for p, q in zip(run, want[i]))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs a second GPU")
def test_tensors_of_another_device():
    from gddim_amd import ops
    other = torch.device("cuda", 1)
    x, wg, wu, wd, dy = _inputs(other, 70, 64, 136, 64, torch.bfloat16)
    with torch.cuda.device(0):
        got = _run(x, wg, wu, wd, dy, "silu")
    for g, w in zip(got, ref.gated_ffn(x, wg, wu, wd, "silu", torch.bfloat16, dy)):
        assert g.device == other
        _check(g, w, "on the second device")


@pytest.mark.parametrize("typ", ["bf16", "f32"])
def test_strides_and_batches(dev, typ):
    """rows and weights seen through larger matrices, both projections packed, channels not adjacent, batches of any rank, rows off any alignment"""
    from gddim_amd import ops
    dtype, M, D, F, O = TYPES[typ], 30, 48, 56, 40
    x, wg, wu, wd, dy = _inputs(dev, M, D, F, O, dtype, 5)
    want = ref.gated_ffn(x, wg, wu, wd, "gelu", dtype, dy)
    nan = lambda *s: torch.full(s, float("nan"), dtype=dtype, device=dev)
    packed = torch.cat((wg, wu))
    wide_x, wide_w, wide_y = nan(M + 2, D + 16), nan(O + 1, F + 8), nan(M, O + 3)
    wide_x[1:M + 1, 8:8 + D], wide_w[:O, :F], wide_y[:, 1:1 + O] = x, wd, dy
    forms = [
        (wide_x[1:M + 1, 8:8 + D], packed[:F], packed[F:], wide_w[:O, :F], wide_y[:, 1:1 + O]),
        (x.t().contiguous().t(), wg.t().contiguous().t(), wu, wd.t().contiguous().t(), dy.t().contiguous().t()),
        (x.view(2, 3, 5, D), wg, wu, wd, dy.view(2, 3, 5, O)),
    ]
    odd = nan(M * (D + 1) + 1)[1:].view(M, D + 1)
    odd[:, :D] = x
    forms.append((odd[:, :D], wg, wu, wd, dy))
    for i, f in enumerate(forms):
        got = _run(*f, "gelu")
        assert got[0].shape == f[0].shape[:-1] + (O,) and got[1].shape == f[0].shape
        for g, w, what in zip(got, want, ("y", "dx", "dw_gate", "dw_up", "dw_down")):
            _check(g.reshape(w.val.shape), w, "%s of form %d" % (what, i))
    one = x[:1].expand(M, D)  # one row seen as many
    _check(ops.gated_ffn(one, wg, wu, wd, act="gelu"), ref.gated_ffn(one, wg, wu, wd, "gelu", dtype), "expanded")


@pytest.mark.parametrize("typ", ["bf16", "f32"])
@pytest.mark.parametrize("size,apart", [((70, 64, 72, 100), 104), ((70, 64, 72, 98), 104), ((300, 40, 264, 13), 16), ((70, 64, 72, 96), 99), ((70, 63, 72, 96), 104), ((3, 64, 72, 96), (1 << 21) + 8)], ids=str)
def test_rows_of_dy_apart(dev, size, apart, typ):
    """dense rows of dy would not be aligned, these are; and the other way round"""
    from gddim_amd import ops
    x, wg, wu, wd, dy = _inputs(dev, *size, TYPES[typ], 7)
    wide = torch.full((size[0], apart), 7.0, dtype=TYPES[typ], device=dev)
    wide[:, :size[3]] = dy
    want = _run(x, wg, wu, wd, dy, "silu")
    got = _run(x, wg, wu, wd, wide[:, :size[3]], "silu")
    for g, w, f64, what in zip(got, want, ref.gated_ffn(x, wg, wu, wd, "silu", TYPES[typ], dy), ("y", "dx", "dw_gate", "dw_up", "dw_down")):
        _check(g, f64, what)
        _check(w, f64, what)


@pytest.mark.parametrize("typ", ["bf16", "f32"])
@pytest.mark.parametrize("apart", [0, 1, 24, 1 << 40])
def test_row_stride_of_a_single_row_means_nothing(dev, apart, typ):
    size = (1, 64, 72, 40)
    x, wg, wu, wd, dy = _inputs(dev, *size, TYPES[typ], 8)
    x[0, 5] = float("inf")  # padded rows of the sums over rows must not meet it
    wg[:, 5] = wg[:, 5].abs() * 1e-3
    want = _run(x, wg, wu, wd, dy, "silu")
    for g, w in zip(_run(x.as_strided((1, 64), (apart, 1)), wg, wu, wd, dy.as_strided((1, 40), (apart, 1)), "silu"), want):
        assert torch.equal(g.nan_to_num(123.0), w.nan_to_num(123.0))
    one = _inputs(dev, 5, 64, 1, 1, TYPES[typ], 8)  # weights of one row
    want = _run(*one, "gelu")
    w = [t.as_strided(t.shape, (apart + i, 1)) for i, t in enumerate(one[1:4])]
    for g, v in zip(_run(one[0], *w, one[4], "gelu"), want):
        assert torch.equal(g, v)


@pytest.mark.parametrize("typ", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M", [1, 7, 40, 200])
def test_infinities_and_nan_stay_in_their_row(dev, typ, M):
    from gddim_amd import ops
    x, wg, wu, wd, dy = _inputs(dev, M + 2, 72, 80, 64, TYPES[typ], 6)
    clean = ops.gated_ffn(x, wg, wu, wd)
    bad = x.clone()
    bad[0] = float("nan")
    bad[M + 1, 3] = float("inf")
    got = ops.gated_ffn(bad, wg, wu, wd)
    assert torch.isnan(got[0]).all() and not torch.isfinite(got[M + 1]).all()
    assert torch.equal(got[1:M + 1], clean[1:M + 1])


@pytest.mark.parametrize("typ", ["bf16", "f32"])
def test_gradients_against_differences(dev, typ):
    """a directional difference of the float64 form, step 1e-6: its own error is under 1e-8 of the sums' magnitude, the kernels' under their types' bounds"""
    dtype = TYPES[typ]
    x, wg, wu, wd, dy = _inputs(dev, 9, 24, 40, 16, dtype, 7)
    got = _run(x, wg, wu, wd, dy, "gelu_tanh")
    want = ref.gated_ffn(x, wg, wu, wd, "gelu_tanh", dtype, dy)
    leaves = [t.double() for t in (x, wg, wu, wd)]
    loss = lambda l: (ref.product(ref.act(ref.product(ref.V(l[0]), ref.V(l[1])), "gelu_tanh")[0] * ref.product(ref.V(l[0]), ref.V(l[2])), ref.V(l[3])).val * dy.double()).sum()
    for i in range(4):
        d = torch.randn(leaves[i].shape, generator=torch.Generator(dev).manual_seed(i), device=dev, dtype=torch.float64)
        up, dn = list(leaves), list(leaves)
        up[i], dn[i] = leaves[i] + 1e-6 * d, leaves[i] - 1e-6 * d
        num = (loss(up) - loss(dn)) / 2e-6
        assert abs(float(num - (got[i + 1].double() * d).sum())) <= float((want[i + 1].err * d.abs()).sum()) + 1e-6


def test_no_rows(dev):
    from gddim_amd import ops
    for dtype in TYPES.values():
        _, wg, wu, wd, _ = _inputs(dev, 1, 24, 40, 16, dtype)
        x, dy = torch.empty(0, 24, dtype=dtype, device=dev), torch.empty(0, 16, dtype=dtype, device=dev)
        y, saved = ops.gated_ffn(x, wg, wu, wd, save=True)
        assert y.shape == (0, 16)
        dx, *dw = ops.gated_ffn_backward(dy, x, wg, wu, wd, saved)
        assert dx.shape == (0, 24) and all((g == 0).all() for g in dw)


@pytest.mark.parametrize("M", [3, 300])
def test_other_streams_and_graph_replays(dev, M):
    x, wg, wu, wd, dy = _inputs(dev, M, 64, 136, 64, torch.bfloat16, 8)
    eager = _run(x, wg, wu, wd, dy, "silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _run(x, wg, wu, wd, dy, "silu")
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graphs = []
    for _ in range(2):  # two captured calls: workspaces of their own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, _run(x, wg, wu, wd, dy, "silu")))
        graphs[-1] = (graph, graphs[-1][1])
    for trial in range(4):
        x.copy_(torch.randn(x.shape, generator=torch.Generator(dev).manual_seed(trial), device=dev).to(x.dtype))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        now = _run(x, wg, wu, wd, dy, "silu")
        for _, captured in graphs:
            assert all(torch.equal(a, b) for a, b in zip(now, captured))


def test_refusals_on_the_gpu(dev):
    from gddim_amd import ops
    from gddim_amd._abi import GddimError
    x, wg, wu, wd, dy = _inputs(dev, 6, 24, 40, 16, torch.float32)
    y, saved = ops.gated_ffn(x, wg, wu, wd, save=True)
    bad = [
        lambda: ops.gated_ffn(x, wg, wu, wd, act="relu"),
        lambda: ops.gated_ffn(x.double(), wg.double(), wu.double(), wd.double()),
        lambda: ops.gated_ffn(x, wg.half(), wu, wd),
        lambda: ops.gated_ffn(x, wg.cpu(), wu, wd),
        lambda: ops.gated_ffn(x, wg[:8], wu, wd),
        lambda: ops.gated_ffn(x[:, :8], wg, wu, wd),
        lambda: ops.gated_ffn(x, wg, wu, wd[:, :8]),
        lambda: ops.gated_ffn(x, wg[None], wu[None], wd),
        lambda: ops.gated_ffn(x, wg[:0], wu[:0], wd[:, :0]),
        lambda: ops.gated_ffn(x, wg.clone().requires_grad_(), wu, wd),
        lambda: ops.gated_ffn_backward(dy[:3], x, wg, wu, wd, saved),
        lambda: ops.gated_ffn_backward(dy, x, wg, wu, wd, saved[:2]),
        lambda: ops.gated_ffn_backward(dy, x, wg, wu, wd, y),
        lambda: ops.gated_ffn_backward(dy, x, wg, wu, wd, tuple(t[:3] for t in saved)),
        lambda: ops.gated_ffn_backward(dy.half(), x, wg, wu, wd, saved),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(GddimError):
            call()
            pytest.fail("call %d was not refused" % i)


@pytest.mark.parametrize("typ", ["bf16", "f16"])
@pytest.mark.parametrize("columns", [49, 50, 51, 129, 130, 255])
@pytest.mark.parametrize("which", ["x", "w_gate and w_up", "w_down"])
def test_odd_columns_of_padded_rows(dev, which, columns, typ):
    """matrices whose rows are whole 16-byte pieces apart and hold no whole number of them: their last row's last element ends the memory that a product
    reads, and counts for much here"""
    M, D, F, O, dtype = 70, 72, 80, 40, TYPES[typ]
    if which == "w_down":
        F = columns
    else:
        D = columns
    x, wg, wu, wd, dy = _inputs(dev, M, D, F, O, dtype, 21)
    for t in (x, wg, wu, wd):
        t[-1, -1] = 12.0
    wide = lambda t: torch.cat((t, torch.full((t.shape[0], -t.shape[1] % 8 + 8), float("nan"), dtype=dtype, device=dev)), 1)[:, :t.shape[1]]
    args = [wide(x) if which == "x" else x] + [wide(t) if which == "w_gate and w_up" else t for t in (wg, wu)] + [wide(wd) if which == "w_down" else wd]
    want = ref.gated_ffn(x, wg, wu, wd, "silu", dtype, dy)
    for g, w, what in zip(_run(*args, dy, "silu"), want, ("y", "dx", "dw_gate", "dw_up", "dw_down")):
        if dtype == torch.float16:  # 12^5 = 248832 is past its range: values of 65520 and more round to infinity
            over = w.val.abs() - w.err >= 65520
            assert (g[over].double() == w.val[over].sign() * float("inf")).all()
            g, w = g.masked_fill(over, 0), ref.V(w.val.masked_fill(over, 0), w.err)
        _check(g, w, what)


def test_few_rows_against_very_many(dev):
    """2^26 rows of the weights: as workgroups of 16 rows each they would be 2^32 threads, more than a launch holds"""
    from gddim_amd import ops
    M, D, F, O, dtype = 2, 8, 1 << 26, 8, torch.bfloat16
    x, wg, wu, _, _ = _inputs(dev, M, D, F, 1, dtype, 22)
    at = torch.tensor([0, 1, 15, 16, 12345678, F // 2, F - 17, F - 2, F - 1], device=dev)
    wd = torch.zeros(O, F, dtype=dtype, device=dev)
    wd[:, at] = torch.randn(O, len(at), generator=torch.Generator(dev).manual_seed(23), device=dev).to(dtype)
    y, saved = ops.gated_ffn(x, wg, wu, wd, save=True)
    gate, up = ref.product(ref.V(x.double()), ref.V(wg.double())), ref.product(ref.V(x.double()), ref.V(wu.double()))
    _check(saved[0], gate, "gate")
    _check(saved[1], up, "up")
    hidden = (ref.act(gate, "silu")[0] * up).rounded(dtype)
    _check(saved[2], hidden, "hidden")
    # all other products are zeros, which round nothing
    _check(y, ref.product(ref.V(hidden.val[:, at], hidden.err[:, at]), ref.V(wd[:, at].double())).rounded(dtype), "y")


@pytest.mark.parametrize("size", [(70, 64, 72, 40), (3, 64, 72, 40), (33, 65, 71, 39), (300, 256, 688, 256)], ids=str)
@pytest.mark.parametrize("scale", [-18, -14, -8, 9])
def test_gradients_of_small_and_large_scale_in_fp16(dev, scale, size):
    """dgate and dup are rounded to fp16 before they are summed: down to its subnormal step, 2^-24, and within 65504 as long as they stay so themselves"""
    x, wg, wu, wd, dy = _inputs(dev, *size, torch.float16, 24)
    dy = dy * 2.0 ** scale
    want = ref.gated_ffn(x, wg, wu, wd, "silu", torch.float16, dy)
    for g, w, what in zip(_run(x, wg, wu, wd, dy, "silu"), want, ("y", "dx", "dw_gate", "dw_up", "dw_down")):
        _check(g, w, what)


def test_hidden_gradients_past_the_range_of_fp16(dev):
    """dgate = 65536 is an infinity before it is summed; bf16 and float32 hold it"""
    for typ, dtype in TYPES.items():
        x, w, dy = (torch.full((1, 1), v, dtype=dtype, device=dev) for v in (32.0, 1.0, 2048.0))
        dx, dwg, _, dwd = _run(x, w, w, w, dy, "silu")[1:]
        assert dwd.item() == (float("inf") if typ == "f16" else 2048.0 * 1024.0)  # the result itself
        if typ == "f16":
            assert dwg.item() == float("inf") and dx.item() == float("inf")
        else:
            assert dwg.item() == 65536.0 * 32.0 and dx.item() == 65536.0 * 2


@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("exponent", [10, 40, 62, 65, 90, 120])
def test_activations_of_very_large_projections(dev, exponent, typ, kind):
    """z = +-2^n: the activation is z or 0, its derivative 1 or 0, also where z^2 and z^3 overflow; powers of two, so nothing rounds"""
    dtype = TYPES[typ]
    for sign in (1.0, -1.0):
        z, small, one = sign * 2.0 ** exponent, 2.0 ** -100, torch.ones(1, 1, dtype=dtype, device=dev)
        x, wu = one * z, one * small
        y, dx, dwg, _, dwd = _run(x, one, wu, one, one, kind)  # gate = z, up = z 2^-100
        want = (z * z * small, 2 * z * small, z * small * z, z * z * small) if sign > 0 else (0.0,) * 4
        for g, w, what in zip((y, dx, dwg, dwd), want, ("y", "dx", "dw_gate", "dw_down")):
            assert g.item() == (w if abs(w) < 2.0 ** 128 else float("inf")), (what, g.item(), w)  # (past the range of both types)


@pytest.mark.parametrize("which", [0, 1, 2, 3, 4])
def test_lazily_negated_tensors(dev, which):
    """matrices of one column are taken with any stride, the imaginary part of a conjugate among them"""
    args = list(_inputs(dev, 5, 1, 1, 1, torch.float32, 25))
    want = _run(*[-t if i == which else t for i, t in enumerate(args)], "gelu")
    args[which] = torch.complex(args[which], args[which]).conj().imag
    assert args[which].is_neg()
    for g, w in zip(_run(*args, "gelu"), want):
        assert torch.equal(g, w)
