"""GPU tests of the rotary operators (positions with several axes; norms of queries and keys with the rotation in the same pass, and their
gradients) against plain float64 forms on the CPU.  Bounds: tests/token_reference.py."""
import pytest
import torch

import token_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.fixture(scope="module")
def dev(native_lib):
    assert torch.cuda.is_available(), "GPU tests need a visible MI355X"
    return torch.device("cuda", 0)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _pos(g, kind, shape, far):
    p = torch.randint(-far, far, shape, generator=g)
    return p.float() * 0.37 if kind == "f32" else p.to(torch.int32 if kind == "i32" else torch.int64)


def _layout(t, how, dev):
    """t on the device in another memory layout (same values, shape (B, N, H, D))"""
    if how == "dense":
        return t.to(dev)
    if how == "bhnd":  # (B, H, N, D) in memory
        return t.to(dev).transpose(1, 2).contiguous().transpose(1, 2)
    B, N, H, D = t.shape
    if how == "packed":  # heads in the middle of a wider projection
        big = torch.full((B, N, H + 3, D), 7.0, dtype=t.dtype, device=dev)
        big[:, :, 1:1 + H] = t.to(dev)
        return big[:, :, 1:1 + H]
    if how == "offset":  # one element off any alignment, odd row stride
        big = torch.full((B * N * H * (D + 1) + 1,), 7.0, dtype=t.dtype, device=dev)
        v = big[1:].view(B, N, H, D + 1)[..., :D]
        v.copy_(t)
        return v
    assert how == "channels"  # channels not adjacent
    return t.to(dev).transpose(2, 3).contiguous().transpose(2, 3)


SHAPES = [
    # B, N, H, Hk, D, sections, layout
    (1, 1, 1, 1, 2, (2,), "dense"),
    (2, 3, 2, 1, 64, (64,), "dense"),
    (1, 5, 4, 2, 128, (16, 56, 56), "bhnd"),
    (2, 7, 3, 3, 72, (24, 24), "packed"),
    (3, 4, 5, 1, 80, (16, 32, 32), "dense"),
    (1, 6, 2, 2, 7, (4, 2), "dense"),          # an odd head: one channel without a partner
    (2, 5, 3, 1, 128, (32, 32), "offset"),
    (1, 3, 2, 2, 33, (2, 2, 2, 2), "offset"),
    (1, 2, 2, 1, 512, (512,), "dense"),
    (1, 2, 3, 1, 512, (100, 200), "offset"),   # a head over more than one wave's lanes
    (2, 3, 4, 4, 20, (8, 12), "dense"),
    (1, 9, 33, 3, 96, (32, 32, 32), "packed"),
    (1, 4, 2, 2, 64, (32, 32), "channels"),
    (2, 4301, 2, 1, 16, (4, 6, 6), "dense"),   # tokens enough to fill the chip: whole tokens per wave
    (3, 8191, 1, 1, 64, (24, 16, 24), "bhnd"),  # ... and several small ones
    (2, 20011, 3, 1, 16, (16,), "dense"),
    (1, 33001, 2, 2, 7, (4, 2), "packed"),
    (2, 3, 2, 1, 260, (100, 60), "dense"),      # wide heads in whole vectors of 8 bytes, not of 16
    (1, 5, 3, 2, 508, (508,), "packed"),
    (1, 4, 2, 3, 300, (4, 200), "bhnd"),
]


@pytest.mark.parametrize("paired", ["interleaved", "halves"])
@pytest.mark.parametrize("typ", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rotary(dev, shape, typ, paired):
    from gddim_amd import ops
    B, N, H, _, D, sections, how = shape
    dtype = TYPES[typ]
    g = _gen(SHAPES.index(shape))
    x = torch.randn(B, N, H, D, generator=g).to(dtype)
    kind = {"f32": "f32", "bf16": "i64", "f16": "i32"}[typ]
    pos = _pos(g, kind, (N, len(sections)) if paired == "halves" else (B, N, len(sections)), 1000)
    axes = ops.RotaryAxes(sections, theta=500.0, paired=paired, device=dev)
    phi = ref.angles(pos, sections, 500.0, B, N)
    xd = _layout(x, how, dev)
    for inverse in (False, True):
        got = ops.rotary(xd, pos.to(dev), axes, inverse=inverse)
        want, mag = ref.rotate(x.double(), phi, sections, paired, inverse)
        assert got.dtype == dtype
        ref.assert_within(got, want, ref.bound(want, mag, ref.ROTATION, dtype), "inverse=%s" % inverse)
        if how == "bhnd":
            assert got.transpose(1, 2).is_contiguous()
    assert torch.equal(xd.cpu(), x)


@pytest.mark.parametrize("far", [1 << 20, (1 << 31) - 1])
def test_far_positions(dev, far):
    """Angles of positions up to 2^31: 64 bits hold them to 2^31 * 2^-53 * 2 (the product and the table) = 4.8e-7 turns of a radian."""
    from gddim_amd import ops
    B, N, H, D, sections = 1, 64, 2, 32, (20, 12)
    g = _gen(5)
    x = torch.randn(B, N, H, D, generator=g)
    pos = torch.randint(-far, far, (N, 2), generator=g)
    axes = ops.RotaryAxes(sections, device=dev)
    got = ops.rotary(x.to(dev), pos.to(dev), axes)
    want, mag = ref.rotate(x.double(), ref.angles(pos, sections, 10000.0, B, N), sections, "interleaved")
    ref.assert_within(got, want, ref.bound(want, mag, ref.ROTATION, torch.float32) + mag * (4 * far * 2.0 ** -53))


def test_given_frequencies_and_shared_positions(dev):
    from gddim_amd import ops
    freq = torch.linspace(3.0, 0.01, 12, dtype=torch.float64)
    axes = ops.RotaryAxes((8, 16), frequencies=freq, paired="halves", device=dev)
    g = _gen(6)
    x = torch.randn(3, 5, 2, 24, generator=g)
    pos = torch.randint(0, 50, (1, 5, 2), generator=g)
    want, mag = ref.rotate(x.double(), ref.angles(pos, (8, 16), 0, 3, 5, freq), (8, 16), "halves")
    limit = ref.bound(want, mag, ref.ROTATION, torch.float32)
    ref.assert_within(ops.rotary(x.to(dev), pos.to(dev), axes), want, limit)
    ref.assert_within(ops.rotary(x.to(dev), pos[0].to(dev), axes), want, limit)
    strided = torch.zeros(5, 4, dtype=torch.int64, device=dev)
    strided[:, ::2] = pos[0].to(dev)
    ref.assert_within(ops.rotary(x.to(dev), strided[:, ::2], axes), want, limit)
    one = x[:1, :, :1].to(dev).expand(3, 5, 2, 24)  # one head seen as many
    want, mag = ref.rotate(x[:1, :, :1].double().expand(3, 5, 2, 24), ref.angles(pos, (8, 16), 0, 3, 5, freq), (8, 16), "halves")
    ref.assert_within(ops.rotary(one, pos.to(dev), axes), want, ref.bound(want, mag, ref.ROTATION, torch.float32))


def test_offsets_past_32_bits(dev):
    from gddim_amd import ops
    D, far_row = 64, (1 << 31) + 128
    big = torch.empty(far_row + D, dtype=torch.bfloat16, device=dev)
    x = torch.randn(2, 1, 1, D, generator=_gen(8)).to(torch.bfloat16)
    xd = big.as_strided((2, 1, 1, D), (far_row, D, D, 1))
    xd.copy_(x)
    pos = torch.tensor([[[3, 4]], [[5, 6]]])
    axes = ops.RotaryAxes((32, 32), device=dev)
    want, mag = ref.rotate(x.double(), ref.angles(pos, (32, 32), 10000.0, 2, 1), (32, 32), "interleaved")
    ref.assert_within(ops.rotary(xd, pos.to(dev), axes), want, ref.bound(want, mag, ref.ROTATION, torch.bfloat16))


def _qk_case(dev, shape, typ, paired, weights, seed):
    from gddim_amd import ops
    B, N, H, Hk, D, sections, how = shape
    dtype = TYPES[typ]
    g = _gen(seed)
    q, k = torch.randn(B, N, H, D, generator=g).to(dtype), (3 * torch.randn(B, N, Hk, D, generator=g)).to(dtype)
    gq, gk = torch.randn(B, N, H, D, generator=g).to(dtype), torch.randn(B, N, Hk, D, generator=g).to(dtype)
    w = [None, None]
    if weights != "none":
        wt = torch.float32 if weights == "f32" else dtype
        w = [(1 + 0.3 * torch.randn(D, generator=g)).to(wt) for _ in range(2)]
    if weights == "q":
        w[1] = None
    pos = _pos(g, "i64", (B, N, len(sections)), 300)
    axes = ops.RotaryAxes(sections, paired=paired, device=dev)
    return q, k, gq, gk, w, pos, axes


def _f64(t):
    return None if t is None else t.double()


@pytest.mark.parametrize("paired", ["interleaved", "halves"])
@pytest.mark.parametrize("typ,weights", [("f32", "own"), ("bf16", "own"), ("bf16", "f32"), ("f16", "q"), ("f32", "none")])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_qk_norm_rotary_and_gradients(dev, shape, typ, weights, paired):
    from gddim_amd import ops
    B, N, H, Hk, D, sections, how = shape
    dtype, eps = TYPES[typ], 1e-5
    q, k, gq, gk, w, pos, axes = _qk_case(dev, shape, typ, paired, weights, 11)
    phi = ref.angles(pos, sections, 10000.0, B, N)
    qd, kd = _layout(q, how, dev), _layout(k, how, dev)
    wd = [None if t is None else t.to(dev) for t in w]
    out = ops.qk_norm_rotary(qd, kd, wd[0], wd[1], pos.to(dev), axes, eps=eps)
    for got, x, wt in ((out[0], q, w[0]), (out[1], k, w[1])):
        want, mag, n = ref.norm_rotary(x.double(), _f64(wt), phi, sections, paired, eps)
        ref.assert_within(got, want, ref.bound(want, mag, n, dtype), "forward")
    args = (_layout(gq, how, dev), _layout(gk, how, dev), qd, kd, wd[0], wd[1], pos.to(dev), axes)
    grads = ops.qk_norm_rotary_backward(*args, eps=eps)
    for dx, dw, x, gy, wt in ((grads[0], grads[2], q, gq, w[0]), (grads[1], grads[3], k, gk, w[1])):
        want, mag, dww, dwm, n = ref.norm_rotary_backward(gy.double(), x.double(), _f64(wt), phi, sections, paired, eps)
        ref.assert_within(dx, want, ref.bound(want, mag, n, dtype), "dx")
        if wt is None:
            assert dw is None
        else:
            # dw: the terms' own roundings, then additions on a term's way: its wave's heads, shuffles, waves, workgroups (< 64 in sequence here)
            assert dw.dtype == wt.dtype
            ref.assert_within(dw, dww, ref.bound(dww, dwm, n + 128, wt.dtype), "dw")
    again = ops.qk_norm_rotary_backward(*args, eps=eps)
    for a, b in zip(grads, again):
        assert (a is None and b is None) or torch.equal(a, b)


def test_gradients_against_differences(dev):
    """dx and dw against central differences of the float64 form, h = 1e-5: h^2 times a third derivative of order 10 plus 1e-16/h, under 1e-8."""
    from gddim_amd import ops
    shape, eps = (1, 3, 2, 1, 12, (4, 6), "dense"), 1e-2
    q, k, gq, gk, w, pos, axes = _qk_case(dev, shape, "f32", "halves", "own", 3)
    phi = ref.angles(pos, shape[5], 10000.0, 1, 3)
    grads = ops.qk_norm_rotary_backward(gq.to(dev), gk.to(dev), q.to(dev), k.to(dev), w[0].to(dev), w[1].to(dev), pos.to(dev), axes, eps=eps)

    def loss(x, wt, gy):
        return float((ref.norm_rotary(x, wt, phi, shape[5], "halves", eps)[0] * gy.double()).sum())

    h = 1e-5
    for dx, dw, x, gy, wt in ((grads[0], grads[2], q, gq, w[0]), (grads[1], grads[3], k, gk, w[1])):
        x, wt = x.double(), wt.double()
        for t, got in ((x, dx), (wt, dw)):
            flat, num = t.view(-1), torch.empty(t.numel(), dtype=torch.float64)
            for i in range(t.numel()):
                keep = flat[i].item()
                flat[i] = keep + h
                up = loss(x, wt, gy)
                flat[i] = keep - h
                num[i] = (up - loss(x, wt, gy)) / (2 * h)
                flat[i] = keep
            assert (got.cpu().double().view(-1) - num).abs().max() < 1e-4 * max(1.0, num.abs().max())


def test_rows_of_zeros_infinities_and_nan_stay_their_own(dev):
    from gddim_amd import ops
    axes = ops.RotaryAxes((16, 16), device=dev)
    g = _gen(2)
    q = torch.randn(1, 4, 8, 32, generator=g)
    q[0, 0, 3] = 0.0
    q[0, 1, 2] = float("inf")
    q[0, 2, 1, 5] = float("nan")
    k, pos, w = torch.randn(1, 4, 2, 32, generator=g), torch.randint(0, 9, (4, 2), generator=g), torch.ones(32)
    phi = ref.angles(pos, (16, 16), 10000.0, 1, 4)
    got = ops.qk_norm_rotary(q.to(dev), k.to(dev), w.to(dev), None, pos.to(dev), axes)[0].cpu()
    assert (got[0, 0, 3] == 0).all() and torch.isnan(got[0, 1, 2]).all() and torch.isnan(got[0, 2, 1]).all()
    clean = torch.ones(1, 4, 8, dtype=torch.bool)
    clean[0, 1, 2] = clean[0, 2, 1] = False
    want, mag, n = ref.norm_rotary(q.double(), None, phi, (16, 16), "interleaved", 1e-6)
    ref.assert_within(got[clean], want[clean], ref.bound(want, mag, n, torch.float32)[clean])


def test_no_tokens(dev):
    from gddim_amd import ops
    axes = ops.RotaryAxes((8, 8), device=dev)
    w = torch.ones(16, device=dev)
    for shape in ((0, 5, 2, 16), (3, 0, 2, 16)):
        x = torch.empty(shape, device=dev)
        pos = torch.empty(shape[1], 2, dtype=torch.int64, device=dev)
        assert ops.rotary(x, pos, axes).shape == shape
        assert ops.qk_norm_rotary(x, x, w, w, pos, axes)[1].shape == shape
        dq, dk, dwq, dwk = ops.qk_norm_rotary_backward(x, x, x, x, w, w, pos, axes)
        assert dq.shape == shape and (dwq == 0).all() and (dwk == 0).all()


def test_other_streams_and_graph_replays(dev):
    """Calls follow the current stream; a captured forward and backward gives the eager bits on every replay, with new inputs too."""
    from gddim_amd import ops
    shape = (2, 37, 4, 2, 64, (32, 32), "dense")
    q, k, gq, gk, w, pos, axes = _qk_case(dev, shape, "bf16", "interleaved", "own", 4)
    st = [t.to(dev) for t in (q, k, gq, gk, w[0], w[1], pos)]

    def step(s):
        return ops.qk_norm_rotary(s[0], s[1], s[4], s[5], s[6], axes) + ops.qk_norm_rotary_backward(s[2], s[3], s[0], s[1], s[4], s[5], s[6], axes)

    eager = step(st)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(st)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(st)
    for trial in range(4):
        st[0].copy_(torch.randn(q.shape, generator=_gen(trial)).to(q.dtype))
        st[2].copy_(torch.randn(q.shape, generator=_gen(90 + trial)).to(q.dtype))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(step(st), captured):
            assert torch.equal(a, b)


def test_refusals_on_the_gpu(dev):
    from gddim_amd import ops
    from gddim_amd._abi import GddimError
    axes = ops.RotaryAxes((8, 8), device=dev)
    x, pos, w = torch.randn(2, 3, 4, 16, device=dev), torch.zeros(3, 2, dtype=torch.int64, device=dev), torch.ones(16, device=dev)
    bad = [
        lambda: ops.rotary(x[0], pos, axes),
        lambda: ops.rotary(x.double(), pos, axes),
        lambda: ops.rotary(x, pos.double(), axes),
        lambda: ops.rotary(x, pos.cpu(), axes),
        lambda: ops.rotary(x, pos[:2], axes),
        lambda: ops.rotary(x, pos[:, :1], axes),
        lambda: ops.rotary(x[..., :12], pos, axes),
        lambda: ops.rotary(x, pos, (8, 8)),
        lambda: ops.rotary(x, pos, ops.RotaryAxes((8, 8), device="cpu")),
        lambda: ops.rotary(x.requires_grad_(), pos, axes),
        lambda: ops.qk_norm_rotary(x.detach(), x.detach().half(), None, None, pos, axes),
        lambda: ops.qk_norm_rotary(x.detach(), x.detach()[:, :2], None, None, pos, axes),
        lambda: ops.qk_norm_rotary(x.detach(), x.detach(), w[:8], None, pos, axes),
        lambda: ops.qk_norm_rotary(x.detach(), x.detach(), w.double(), None, pos, axes),
        lambda: ops.qk_norm_rotary(x.detach().half(), x.detach().half(), w, w.half(), pos, axes),
        lambda: ops.qk_norm_rotary(x.detach(), x.detach(), w, w, pos, axes, eps=-1.0),
        lambda: ops.qk_norm_rotary_backward(x.detach()[:, :, :2], x.detach(), x.detach(), x.detach(), w, w, pos, axes),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(GddimError):
            call()
            pytest.fail("call %d was not refused" % i)
    with torch.no_grad():
        ops.rotary(x, pos, axes)


def test_axes_are_ready_for_any_stream(dev):
    """a table made while its stream is busy, used on another one at once"""
    from gddim_amd import ops
    g = _gen(77)
    x, pos = torch.randn(1, 65, 2, 16, generator=g).to(dev), torch.randint(-99, 99, (65, 1), generator=g).to(dev)
    freq = torch.rand(8, dtype=torch.float64, generator=g)
    want = ops.rotary(x, pos, ops.RotaryAxes((16,), frequencies=freq, device=dev))
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    busy = torch.randn(4096, 4096, device=dev)
    for _ in range(20):
        busy = torch.mm(busy, busy) * 1e-3
    axes = ops.RotaryAxes((16,), frequencies=freq.to(dev), device=dev)
    with torch.cuda.stream(other):
        got = ops.rotary(x, pos, axes)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


PARTIAL = [
    # D, sections, head stride: vectors of 16 and 8 bytes and single pairs; lanes whose pairs turn in part, heads over more than 64 lanes
    (64, (16, 16), 64), (64, (20, 16), 64), (72, (24, 24), 80), (40, (8, 4), 44), (24, (8, 2), 25), (33, (4, 6), 33), (260, (100, 60), 260), (512, (128, 66), 513), (16, (2,), 16),
]


def _strided(t, apart, dev):
    """t (B, N, heads, D) on the device with heads `apart` elements from each other"""
    big = torch.zeros(t.shape[:3] + (apart,), dtype=t.dtype, device=dev)
    big[..., :t.shape[3]] = t.to(dev)
    return big[..., :t.shape[3]]


@pytest.mark.parametrize("paired", ["interleaved", "halves"])
@pytest.mark.parametrize("typ", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("form", PARTIAL, ids=str)
def test_channels_behind_the_sections_pass_through(dev, form, typ, paired):
    """as they are, whatever lies beside them: infinities, NaN and the sign of zeros"""
    from gddim_amd import ops
    D, sections, apart = form
    R, dtype = sum(sections), TYPES[typ]
    g = _gen(31)
    x = torch.randn(2, 5, 3, D, generator=g).to(dtype)
    special = torch.tensor([float("inf"), float("-inf"), float("nan"), -0.0, 0.0])
    rest = x[..., R:]
    at = torch.rand(rest.shape, generator=g) < 0.4
    rest[at] = special[torch.randint(0, 5, (int(at.sum()),), generator=g)].to(dtype)
    pos = torch.randint(-40, 40, (5, len(sections)), generator=g)
    phi = ref.angles(pos, sections, 10000.0, 2, 5)
    axes = ops.RotaryAxes(sections, paired=paired, device=dev)
    for inverse in (False, True):
        got = ops.rotary(_strided(x, apart, dev), pos.to(dev), axes, inverse=inverse).cpu()
        want, mag = ref.rotate(x.double(), phi, sections, paired, inverse)
        ref.assert_within(got[..., :R], want[..., :R], ref.bound(want, mag, ref.ROTATION, dtype)[..., :R])
        out, nan = got[..., R:], torch.isnan(rest)
        assert torch.equal(torch.isnan(out), nan)
        assert torch.equal(out[~nan], rest[~nan]) and torch.equal(torch.signbit(out[~nan]), torch.signbit(rest[~nan]))


@pytest.mark.parametrize("paired", ["interleaved", "halves"])
@pytest.mark.parametrize("typ", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("form", PARTIAL, ids=str)
def test_gradients_behind_the_sections_stay_their_own(dev, form, typ, paired):
    """an infinite gradient of a channel that passes through is its weight's alone; an infinite input leaves zeros of its head's other channels"""
    from gddim_amd import ops
    D, sections, apart = form
    R, dtype, eps = sum(sections), TYPES[typ], 1e-5
    g = _gen(32)
    q, gy = (torch.randn(1, 4, 2, D, generator=g).to(dtype) for _ in range(2))
    q[0, 1, 0, R] = q[0, 1, 0, R].abs() + 0.5  # (a product of an infinity with zero would be NaN by the formula)
    w, pos = (1 + 0.3 * torch.randn(D, generator=g)).to(dtype), torch.randint(-40, 40, (4, len(sections)), generator=g)
    phi = ref.angles(pos, sections, 10000.0, 1, 4)
    axes = ops.RotaryAxes(sections, paired=paired, device=dev)
    gy[0, 1, 0, R] = float("inf")
    qd, gd = _strided(q, apart, dev), _strided(gy, apart, dev)
    dq, dk, dwq, dwk = ops.qk_norm_rotary_backward(gd, gd, qd, qd, w.to(dev), w.to(dev), pos.to(dev), axes, eps=eps)
    want, mag, dww, dwm, n = ref.norm_rotary_backward(gy.double(), q.double(), w.double(), phi, sections, paired, eps)
    others = torch.arange(D) != R
    limit = ref.bound(dww, dwm, n + 128, dtype)
    for dw in (dwq, dwk):
        assert dw[R] == float("inf")
        ref.assert_within(dw[others.to(dev)], dww[others], limit[others], "dw")
    heads = torch.ones(1, 4, 2, dtype=torch.bool)
    heads[0, 1, 0] = False
    ref.assert_within(dq.cpu()[heads], want[heads], ref.bound(want, mag, n, dtype)[heads], "dx")

    q[0, 2, 1, R] = float("inf")
    out = ops.qk_norm_rotary(_strided(q, apart, dev), qd, w.to(dev), w.to(dev), pos.to(dev), axes, eps=eps)[0].cpu()
    assert torch.isnan(out[0, 2, 1, R]) and (out[0, 2, 1][others] == 0).all()


def test_lazily_negated_positions_are_refused(dev):
    """the imaginary part of a conjugate is a view with a sign to come: its memory holds the other one"""
    from gddim_amd import ops
    from gddim_amd._abi import GddimError
    x, axes = torch.randn(1, 5, 2, 16, generator=_gen(40)).to(dev), ops.RotaryAxes((8, 8), device=dev)
    z = torch.complex(torch.zeros(5, 2), torch.randint(-9, 9, (5, 2), generator=_gen(41)).float()).to(dev)
    pos = z.conj().imag
    assert pos.is_neg()
    for call in (lambda: ops.rotary(x, pos, axes), lambda: ops.qk_norm_rotary(x, x, None, None, pos, axes), lambda: ops.qk_norm_rotary_backward(x, x, x, x, None, None, pos, axes)):
        with pytest.raises(GddimError, match="resolve_neg"):
            call()
    assert torch.equal(ops.rotary(x, pos.resolve_neg(), axes), ops.rotary(x, -z.imag.contiguous(), axes))
    zx = torch.complex(x, x)
    assert torch.equal(ops.rotary(zx.conj().imag, z.imag, axes), ops.rotary(-x, z.imag, axes))  # channels two apart: copied, and the sign with them
