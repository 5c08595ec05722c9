"""CPU tests of the token operators' boundary: argument checks of the Python wrappers and of the C entry points (which refuse before anything
is launched), and the float64 forms that the GPU tests compare with, against autograd."""
import ctypes

import pytest
import torch

import token_reference as ref


def test_rotary_axes_checks(native_lib):
    from gddim_amd import ops
    from gddim_amd._abi import GddimError
    for kw in (dict(sections=()), dict(sections=(2,) * 5), dict(sections=(3,)), dict(sections=(0,)), dict(sections=(4,), paired="quarters"),
               dict(sections=(4,), theta=0.0), dict(sections=(4,), theta=float("nan")), dict(sections=(4, 4), frequencies=[1.0])):
        with pytest.raises(GddimError):
            ops.RotaryAxes(device="cpu", **kw)
    axes = ops.RotaryAxes((4, 6), theta=100.0, device="cpu")
    want = [100.0 ** (-2 * j / s) for s in (4, 6) for j in range(s // 2)]
    assert axes.frequencies.tolist() == want and axes.frequencies.dtype == torch.float64


def test_no_cpu_fallback(native_lib):
    from gddim_amd import ops
    from gddim_amd._abi import GddimError
    axes, x, pos = ops.RotaryAxes((4,), device="cpu"), torch.zeros(1, 2, 1, 4), torch.zeros(2, 1, dtype=torch.int64)
    for call in (lambda: ops.rotary(x, pos, axes), lambda: ops.qk_norm_rotary(x, x, None, None, pos, axes),
                 lambda: ops.qk_norm_rotary_backward(x, x, x, x, None, None, pos, axes), lambda: ops.rotary([1.0], pos, axes)):
        with pytest.raises(GddimError):
            call()


def _desc(**kw):
    from gddim_amd._abi import RotaryDesc
    d = dict(dtype=0, batch=1, tokens=4, head_dim=16, n_axes=2, section=(8, 8), paired_halves=0, pos_type=0, pos=64, pos_stride_b=0, pos_stride_n=2,
             pos_stride_axis=1, freq=64)
    d.update(kw)
    d["section"] = (ctypes.c_int * 4)(*d["section"])
    return ctypes.byref(RotaryDesc(**d))


@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(dtype=-1), dict(pos_type=9), dict(batch=-1), dict(batch=1 << 16, tokens=1 << 15), dict(head_dim=1), dict(head_dim=513),
    dict(n_axes=0), dict(n_axes=5), dict(section=(8, 10)), dict(section=(8, 7)), dict(section=(8, 0)), dict(section=(8, -8)), dict(section=(2 ** 31 - 2, 8)),
    dict(pos=None), dict(freq=None)], ids=str)
def test_c_entry_points_refuse_descriptions(native_lib, bad):
    """None of these reaches a launch: the fake addresses are never read."""
    from gddim_amd._abi import Heads
    h = ctypes.byref(Heads(64, 64, 16, 16))
    assert native_lib.gd_rotary(_desc(**bad), h, h, 1, 0, None) != 0
    assert native_lib.gd_last_error()
    assert native_lib.gd_qk_norm_rotary(_desc(**bad), h, h, h, h, 1, 1, None, None, 0, 1e-6, None) != 0
    assert native_lib.gd_qk_norm_rotary_backward(_desc(**bad), h, h, h, h, h, h, 1, 1, None, None, 0, 1e-6, 64, None, None, None) != 0


def test_c_entry_points_refuse_arguments(native_lib):
    from gddim_amd._abi import Heads
    h, null, d = ctypes.byref(Heads(64, 64, 16, 16)), ctypes.byref(Heads(None, 64, 16, 16)), _desc()
    assert native_lib.gd_rotary(None, h, h, 1, 0, None) != 0
    assert native_lib.gd_rotary(d, h, null, 1, 0, None) != 0
    assert native_lib.gd_rotary(d, None, h, 1, 0, None) != 0
    for heads in (0, -1, 1 << 16):
        assert native_lib.gd_rotary(d, h, h, heads, 0, None) != 0
        assert native_lib.gd_qk_norm_rotary(d, h, h, h, h, 1, heads, None, None, 0, 1e-6, None) != 0
    for eps in (-1.0, float("nan")):
        assert native_lib.gd_qk_norm_rotary(d, h, h, h, h, 1, 1, None, None, 0, eps, None) != 0
    assert native_lib.gd_qk_norm_rotary_backward(d, h, h, h, h, h, h, 1, 1, None, None, 0, 1e-6, None, None, None, None) != 0
    assert native_lib.gd_qk_norm_rotary_backward_workspace(128) > 0


@pytest.mark.parametrize("paired", ["interleaved", "halves"])
def test_float64_forms_against_autograd(paired):
    """The formulas that the GPU tests hold the kernels to, against differentiation of the forward form."""
    g = torch.Generator().manual_seed(0)
    x, dy = torch.randn(2, 3, 2, 14, generator=g, dtype=torch.float64), torch.randn(2, 3, 2, 14, generator=g, dtype=torch.float64)
    w = torch.randn(14, generator=g, dtype=torch.float64)
    phi = ref.angles(torch.randint(0, 50, (3, 2), generator=g), (4, 8), 100.0, 2, 3)
    xa, wa = x.clone().requires_grad_(), w.clone().requires_grad_()
    rho = 1.0 / torch.sqrt((xa * xa).mean(-1, keepdim=True) + 1e-3)
    ia, ib = ref.pair_index((4, 8), paired)
    y = xa * rho * wa
    z = torch.complex(y[..., ia], y[..., ib]) * torch.polar(torch.ones_like(phi), phi)[:, :, None]
    loss = (z.real * dy[..., ia] + z.imag * dy[..., ib]).sum() + (y[..., 12:] * dy[..., 12:]).sum()
    dx, dw = torch.autograd.grad(loss, (xa, wa))
    got = ref.norm_rotary_backward(dy, x, w, phi, (4, 8), paired, 1e-3)
    assert (got[0] - dx).abs().max() < 1e-12 and (got[2] - dw).abs().max() < 1e-12
    out = ref.norm_rotary(x, w, phi, (4, 8), paired, 1e-3)[0]
    assert (out[..., ia] - z.real).abs().max() < 1e-12 and (out[..., ib] - z.imag).abs().max() < 1e-12


def _ffn(**kw):
    from gddim_amd._abi import FfnDesc
    d = dict(dtype=1, act=0, rows=4, in_=8, hidden=16, out=8, unaligned=0, ld_x=8, ld_w_in=8, ld_w_down=16)
    d.update(kw)
    return ctypes.byref(FfnDesc(**d))


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(act=3), dict(act=-1), dict(rows=-1), dict(in_=0), dict(hidden=0), dict(out=0), dict(ld_x=7), dict(ld_w_in=7),
                                 dict(ld_w_down=15), dict(rows=(1 << 30) + 1)], ids=str)
def test_c_gated_ffn_refuses_descriptions(native_lib, bad):
    d = _ffn(**bad)
    assert native_lib.gd_gated_ffn_workspace(d, 0) == -1 and native_lib.gd_gated_ffn_workspace(d, 1) == -1
    assert native_lib.gd_gated_ffn(d, 64, 64, 64, 64, None, None, 64, 64, 64, None) != 0
    assert native_lib.gd_gated_ffn_backward(d, 64, 8, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, None) != 0


def test_c_gated_ffn_refuses_arguments(native_lib):
    d = _ffn()
    for null in range(4):
        args = [64] * 4
        args[null] = None
        assert native_lib.gd_gated_ffn(d, *args, None, None, 64, 64, 64, None) != 0
    assert native_lib.gd_gated_ffn(None, 64, 64, 64, 64, None, None, 64, 64, 64, None) != 0
    assert native_lib.gd_gated_ffn(d, 64, 64, 64, 64, 64, None, 64, 64, 64, None) != 0   # gate without up
    assert native_lib.gd_gated_ffn(d, 64, 64, 64, 64, None, None, None, 64, 64, None) != 0
    assert native_lib.gd_gated_ffn(d, 64, 64, 64, 64, None, None, 64, 64, 72, None) != 0  # workspace off its alignment
    assert native_lib.gd_gated_ffn_backward(d, 64, 7, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, None) != 0
    assert native_lib.gd_gated_ffn_backward(d, 64, 8, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, None, None) != 0
    assert native_lib.gd_gated_ffn(d, 72, 64, 64, 64, None, None, 64, 64, 64, None) != 0  # a tensor off its alignment and not said so
    assert b"unaligned" in native_lib.gd_last_error()
    assert native_lib.gd_gated_ffn_backward(d, 64, 9, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, None) != 0  # ... rows of dy
    assert b"unaligned" in native_lib.gd_last_error()
    assert native_lib.gd_gated_ffn(_ffn(rows=0), None, 64, 64, 64, None, None, None, None, None, None) == 0  # no rows: nothing is launched
    assert native_lib.gd_gated_ffn_workspace(d, 1) >= 2 * 4 * 16 * 2


def test_c_gated_ffn_workspace_over_all_sizes(native_lib):
    """planning (on the host, for 256 compute units without a GPU) gives a size for every shape, none among them"""
    for dtype in (0, 1, 2):
        for rows in (0, 1, 2, 15, 16, 17, 33, 48, 64, 65, 128, 255, 256, 257, 1000, 4096, 70000, 1 << 30):
            for in_, hidden, out in ((1, 1, 1), (8, 8, 8), (7, 13, 5), (64, 2056, 64), (1024, 4096, 1024), (264, 24, 2048)):
                for unaligned in (0, 1):
                    d = _ffn(dtype=dtype, rows=rows, in_=in_, hidden=hidden, out=out, unaligned=unaligned, ld_x=in_, ld_w_in=in_, ld_w_down=hidden)
                    assert native_lib.gd_gated_ffn_workspace(d, 0) >= 0
                    assert native_lib.gd_gated_ffn_workspace(d, 1) >= 2 * rows * hidden * (4 if dtype == 0 else 2)


def test_gated_ffn_needs_a_gpu(native_lib):
    from gddim_amd import ops
    from gddim_amd._abi import GddimError
    x, w = torch.zeros(2, 4), torch.zeros(6, 4)
    with pytest.raises(GddimError):
        ops.gated_ffn(x, w, w, w.t())
    with pytest.raises(GddimError):
        ops.gated_ffn_backward(x, x, w, w, w.t(), (x, x, x))


@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
def test_float64_block_against_autograd(kind):
    g = torch.Generator().manual_seed(1)
    n = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)
    x, wg, wu, wd, dy = n(5, 6), n(7, 6), n(7, 6), n(4, 7), n(5, 4)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    f = torch.nn.functional
    a = f.linear(leaves[0], leaves[1])
    a = f.silu(a) if kind == "silu" else f.gelu(a, approximate="tanh" if kind == "gelu_tanh" else "none")
    y = f.linear(a * f.linear(leaves[0], leaves[2]), leaves[3])
    grads = torch.autograd.grad(y, leaves, dy)
    got = ref.gated_ffn(x, wg, wu, wd, kind, torch.float64, dy)
    for a, b in zip(got, (y,) + grads):
        assert (a.val - b).abs().max() < 1e-12


def test_packed_structures_are_the_header_s(native_lib):
    """token_ops hands the C structures over as packed bytes: the same bytes as the ctypes mirrors of the header"""
    from gddim_amd import _abi, token_ops
    r = _abi.RotaryDesc(1, 2, 3, 4, 2, (ctypes.c_int * 4)(8, 6, 0, 0), 1, 2, 1 << 40, 5, 6, 7, 1 << 41)
    assert bytes(r) == token_ops._ROTARY.pack(1, 2, 3, 4, 2, 8, 6, 0, 0, 1, 2, 1 << 40, 5, 6, 7, 1 << 41)
    assert bytes(_abi.Heads(1 << 40, 2, 3, 4)) == token_ops._HEADS.pack(1 << 40, 2, 3, 4)
    assert bytes(_abi.FfnDesc(1, 2, 3, 4, 5, 6, 1, 8, 9, 10)) == token_ops._FFN.pack(1, 2, 3, 4, 5, 6, 1, 8, 9, 10)


def test_rotary_axes_copies(native_lib):
    """a copy has a table of its own; a given table is taken over by value"""
    import copy
    from gddim_amd import ops
    f = torch.ones(2, dtype=torch.float64)
    axes = ops.RotaryAxes((4,), frequencies=f, device="cpu")
    f.zero_()
    assert axes.frequencies.tolist() == [1.0, 1.0]
    other = copy.deepcopy(axes)
    assert other.frequencies.data_ptr() != axes.frequencies.data_ptr() and other.sections == axes.sections
    with pytest.raises(AttributeError):  # a kernel reads as many of them as the sections say
        axes.frequencies = torch.ones(1)


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    """The entry points' host code over launchers that only write down what they are asked for (tests/token_launches.cpp)."""
    import os
    import subprocess
    from gddim_amd import build
    here = os.path.dirname(os.path.abspath(__file__))
    lib = str(tmp_path_factory.mktemp("launches") / "token_launches.so")
    subprocess.check_call([build._hipcc(), "-x", "hip", "--cuda-host-only", "-O1", "-std=c++17", "-fPIC", "-shared", os.path.join(here, "token_launches.cpp"), "-o", lib])
    lib = ctypes.CDLL(lib)
    lib.gd_gated_ffn_workspace.restype = ctypes.c_longlong
    ll, p = ctypes.c_longlong, ctypes.c_void_p
    lib.gd_gated_ffn.argtypes, lib.gd_gated_ffn_backward.argtypes = [p] * 11, [p, p, ll] + [p] * 13

    def ask(d, out):
        lib.forget_launches()
        at = 1 << 20  # an address that nothing reads
        assert lib.gd_gated_ffn(d, at, at, at, at, None, None, at, at, at, None) == 0
        assert lib.gd_gated_ffn_backward(d, at, out, at, at, at, at, at, at, at, at, at, at, at, at, None) == 0
        rows = []
        for i in range(lib.launches()):
            row = (ctypes.c_longlong * 6)()
            lib.launch(i, row)
            rows.append(list(row))
        assert [r[0] for r in rows] == [0, 1, 2, 3, 4]
        return rows, [at + lib.gd_gated_ffn_workspace(d, b) for b in (0, 1)]

    return ask


def test_c_gated_ffn_launches_are_within_a_grid_s_limits(launches):
    """no launch of 2^32 threads or more, and none whose partial sums leave the workspace"""
    for dtype in (0, 1, 2):
        for rows in (1, 2, 16, 17, 33, 100, 256, 1000, 70001):
            for in_, hidden, out in ((8, 8, 8), (1024, 4096, 1024), (8, 1 << 22, 8), (8, 1 << 26, 8), (16, (1 << 28) + 16, 8), (8, 64, 1 << 26), (8, 1 << 30, 8), (64, 72, 1 << 30)):
                for unaligned in (0, 1):
                    if rows * hidden >= 1 << 38 or rows * out >= 1 << 38:  # (half a terabyte: no card holds it)
                        continue
                    d = _ffn(dtype=dtype, rows=rows, in_=in_, hidden=hidden, out=out, unaligned=unaligned, ld_x=in_, ld_w_in=in_, ld_w_down=hidden)
                    shapes, ends = launches(d, out)
                    for kind, tile, grid, threads, join, partial in shapes:
                        what = (dtype, rows, in_, hidden, out, unaligned, kind, tile)
                        assert 0 < grid * threads < 1 << 32 and 0 <= join * 256 < 1 << 32, what
                        assert partial <= ends[kind > 1], what


def test_forward_mode_tangents_are_refused(native_lib):
    """a dual tensor does not require grad; its tangent would be lost without a word"""
    from torch.autograd import forward_ad
    from gddim_amd import ops
    from gddim_amd._abi import GddimError
    axes, x, w, pos = ops.RotaryAxes((4,), device="cpu"), torch.zeros(1, 2, 1, 4), torch.zeros(4), torch.zeros(2, 1)
    m, a, b = torch.zeros(2, 4), torch.zeros(6, 4), torch.zeros(4, 6)
    with forward_ad.dual_level(), torch.no_grad():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: ops.rotary(dual(x), pos, axes), lambda: ops.qk_norm_rotary(dual(x), x, w, w, pos, axes),
                     lambda: ops.qk_norm_rotary_backward(x, x, dual(x), x, w, w, pos, axes), lambda: ops.gated_ffn(dual(m), a, a, b),
                     lambda: ops.gated_ffn_backward(m, dual(m), a, a, b, (m, m, m))):
            with pytest.raises(GddimError, match="tangent"):
                call()
        with pytest.raises(GddimError, match="GPU only"):
            ops.rotary(x, pos, axes)


def test_c_entry_points_refuse_an_eps_past_float32(native_lib):
    """1e39 reaches the C interface as an infinity, and every head would come out as zeros"""
    from gddim_amd._abi import Heads
    h, d = ctypes.byref(Heads(64, 64, 16, 16)), _desc()
    for eps in (1e39, float("inf"), -1.0, float("nan")):
        assert native_lib.gd_qk_norm_rotary(d, h, h, h, h, 1, 1, None, None, 0, eps, None) != 0
        assert b"eps" in native_lib.gd_last_error()
        assert native_lib.gd_qk_norm_rotary_backward(d, h, h, h, h, h, h, 1, 1, None, None, 0, eps, 64, None, None, None) != 0
        assert b"eps" in native_lib.gd_last_error()
