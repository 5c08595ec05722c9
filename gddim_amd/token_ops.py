"""Token operators of the C ABI on torch device tensors: positions with several axes, norms of queries and keys with the rotation in the same
pass, the gated feed-forward block (include/gddim_amd.h, "token operators").

Tensors are float32, bfloat16 or float16 and stay in their type; work is queued on the current stream of the tensors' device, nothing
synchronises, and every call can be captured into a graph.  The operators record no autograd graph: gradients come from the *_backward calls, and a
tensor that requires grad is refused while grad mode is on.  No reference counterpart."""
import functools
import math
import struct

from . import _abi
from ._abi import GddimError, check

# gd_rotary_desc, gd_heads and gd_ffn_desc as bytes: packed in a third of the time that filling a ctypes structure takes
_ROTARY, _HEADS, _FFN = struct.Struct("@11iP3qP"), struct.Struct("@P3q"), struct.Struct("@7i3q")
_TORCH = None


def _torch():
    """(torch, element type codes, position type codes), imported once"""
    global _TORCH
    if _TORCH is None:
        import torch
        _TORCH = (torch, {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}, {torch.int32: 0, torch.int64: 1, torch.float32: 2})
    return _TORCH


def _raw_stream(index):
    """hipStream_t of a device's current stream (torch's own short way where it has one: the public one builds two objects for a small call's 1.9 us)"""
    torch = _torch()[0]
    short = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return short(index) if short is not None else torch.cuda.current_stream(index).cuda_stream


def _call(t, fn, *args):
    """fn(*args, stream) on t's device and its current stream, whatever device is current"""
    torch = _torch()[0]
    index = t.get_device()
    if torch.cuda.current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        check(rc)


def _on_gpu(t, name):
    torch = _torch()[0]
    if not isinstance(t, torch.Tensor):
        raise GddimError("%s: expected a torch tensor, got %s" % (name, type(t).__name__))
    forward = torch.autograd.forward_ad
    if getattr(forward, "_current_level", 0) >= 0 and forward.unpack_dual(t).tangent is not None:  # (no level, no tangents: asked first, in a quarter of the time)
        raise GddimError("%s carries a forward-mode tangent: the token operators have no forward-mode derivative" % name)
    if not t.is_cuda:
        raise GddimError("gddim_amd operators run on the GPU only (%s is a %s tensor); there is no CPU fallback" % (name, t.device))
    if t.requires_grad and torch.is_grad_enabled():
        raise GddimError("%s requires grad: the token operators record no autograd graph; call them under torch.no_grad() and take gradients "
                         "from the *_backward calls" % name)


def _like(t, name, ref, ref_name):
    _on_gpu(t, name)
    if t.dtype is not ref.dtype or t.get_device() != ref.get_device():
        raise GddimError("%s is %s on %s, %s is %s on %s: types and devices must agree" % (name, t.dtype, t.device, ref_name, ref.dtype, ref.device))


class RotaryAxes:
    """How the channels of a head turn with positions of one to four axes (time, height, width, ...).

    sections[a] channels (even) turn with axis a, in this order; channels behind the last section pass through.  Pair j of a section turns
    by pos * theta^(-2 j / sections[a]); `frequencies` (sum(sections) / 2 radians per unit of position) replaces these.  paired:
    'interleaved' -- channels (2 p, 2 p + 1) -- or 'halves' -- channels (p, p + sum(sections) / 2).  Keeps one float64 table on `device`, whose memory is
    like any tensor's: it has to be kept as long as a captured graph that used it is replayed, and until work queued on a stream other than the one it was
    made on has ended."""

    def __init__(self, sections, theta=10000.0, paired="interleaved", device=None, frequencies=None):
        torch = _torch()[0]
        self.sections = tuple(int(s) for s in sections)
        if not 1 <= len(self.sections) <= _abi.GD_MAX_AXES:
            raise GddimError("RotaryAxes: %d axes, 1 to %d are supported" % (len(self.sections), _abi.GD_MAX_AXES))
        if any(s < 2 or s % 2 for s in self.sections):
            raise GddimError("RotaryAxes: sections %r must be even and at least 2" % (self.sections,))
        if paired not in ("interleaved", "halves"):
            raise GddimError("RotaryAxes: paired=%r, expected 'interleaved' or 'halves'" % (paired,))
        if not (theta > 0.0 and math.isfinite(theta)):
            raise GddimError("RotaryAxes: theta=%r must be positive" % (theta,))
        self.theta, self.paired = float(theta), paired
        if frequencies is None:
            frequencies = [self.theta ** (-2.0 * j / s) for s in self.sections for j in range(s // 2)]
        device = torch.device("cuda") if device is None else torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        # from a table of its own in host memory: the copy has ended when this returns, so that any stream may use it
        self._frequencies = torch.as_tensor(frequencies, dtype=torch.float64).detach().cpu().clone(memory_format=torch.contiguous_format).to(device)
        if tuple(self._frequencies.shape) != (sum(self.sections) // 2,):
            raise GddimError("RotaryAxes: frequencies of shape %s, expected (%d,)" % (tuple(self._frequencies.shape), sum(self.sections) // 2))
        self.device = device
        self._rotated = sum(self.sections)
        self._index = device.index if device.type == "cuda" else -1
        self._halves = int(paired == "halves")
        self._section = self.sections + (0,) * (_abi.GD_MAX_AXES - len(self.sections))

    @property
    def frequencies(self):
        """radians per unit of position, (sum(sections) / 2,) float64"""
        return self._frequencies


def _heads(t):
    """(tensor, its view): channels adjacent, (B, N, heads, D)"""
    s = t.stride()
    if s[3] != 1 and t.shape[3] > 1:
        t = t.contiguous()
        s = t.stride()
    return t, _HEADS.pack(t.data_ptr(), s[0], s[1], s[2])


def _dense_heads(t):
    """the view of an output of _new"""
    s = t.stride()
    return _HEADS.pack(t.data_ptr(), s[0], s[1], s[2])


def _check_heads(t, name, like=None, like_name=None):
    _on_gpu(t, name) if like is None else _like(t, name, like, like_name)
    if t.dim() != 4:
        raise GddimError("%s has shape %s, expected (B, N, heads, D)" % (name, tuple(t.shape)))
    if t.dtype not in _torch()[1]:
        raise GddimError("%s is %s; float32, bfloat16 and float16 are supported" % (name, t.dtype))


def _new(t):
    """An output like t: its order of dimensions where t is dense with adjacent channels ((B, heads, N, D) seen as (B, N, heads, D)), else contiguous."""
    torch = _torch()[0]
    if t.is_contiguous():
        return torch.empty_like(t)
    if 0 not in t.stride():
        out = torch.empty_like(t)
        if out.stride(3) == 1:
            return out
    return t.new_empty(t.shape)


def _rotary_desc(x, pos, axes):
    _, types, pos_types = _torch()
    if not isinstance(axes, RotaryAxes):
        raise GddimError("axes: expected a RotaryAxes, got %s" % type(axes).__name__)
    B, N, _, D = x.shape
    _on_gpu(pos, "pos")
    kind = pos_types.get(pos.dtype)
    if kind == 2 and pos.is_neg():
        raise GddimError("pos is a lazily negated view (of a conjugate): its memory holds the other sign; give pos.resolve_neg()")
    if kind is None:
        raise GddimError("pos is %s; int32, int64 and float32 positions are supported" % pos.dtype)
    index = x.get_device()
    if pos.get_device() != index or axes._index != index:
        raise GddimError("tensors on %s, positions on %s, axes on %s: devices must agree" % (x.device, pos.device, axes.device))
    A = len(axes.sections)
    ps, st = tuple(pos.shape), pos.stride()
    if ps == (N, A):
        sb, sn, sa = 0, st[0], st[1]
    elif ps == (B, N, A):
        sb, sn, sa = st
    elif ps == (1, N, A):
        sb, sn, sa = 0, st[1], st[2]
    else:
        raise GddimError("pos has shape %s, expected (%d, %d) or (%d, %d, %d)" % (ps, N, A, B, N, A))
    if axes._rotated > D:
        raise GddimError("sections %r of %d channels exceed the head's %d" % (axes.sections, axes._rotated, D))
    if B * N >= 1 << 31:
        raise GddimError("%d x %d tokens do not fit 31 bits" % (B, N))
    return _ROTARY.pack(types[x.dtype], B, N, D, A, *axes._section, axes._halves, kind, pos.data_ptr(), sb, sn, sa, axes._frequencies.data_ptr())


def rotary(x, pos, axes, inverse=False):
    """Rotary positions with several axes: x (B, N, heads, D) turned by pos (N, axes) or (B, N, axes) as `axes` (RotaryAxes) says.

    inverse=True turns back, which is also the gradient of the forward call.  Any strides with adjacent channels; the result keeps x's
    order of dimensions where x is dense."""
    _check_heads(x, "x")
    desc = _rotary_desc(x, pos, axes)
    out = _new(x)
    x, view = _heads(x)
    _call(x, _abi.lib().gd_rotary, desc, view, _dense_heads(out), x.shape[2], int(bool(inverse)))
    return out


def _norm_weight(w, name, q):
    if w is None:
        return None
    _on_gpu(w, name)
    if tuple(w.shape) != (q.shape[3],):
        raise GddimError("%s has shape %s, expected (%d,)" % (name, tuple(w.shape), q.shape[3]))
    if w.get_device() != q.get_device() or w.dtype is not q.dtype and w.dtype is not _torch()[0].float32:
        raise GddimError("%s is %s on %s; the tensors' type %s or float32, on %s, is supported" % (name, w.dtype, w.device, q.dtype, q.device))
    return w.contiguous()


def _check_qk(q, k, w_q, w_k, eps):
    """(weight_q, weight_k, their addresses, are they float32 beside another type)"""
    _check_heads(q, "q")
    _check_heads(k, "k", q, "q")
    qs, ks = q.shape, k.shape
    if qs[0] != ks[0] or qs[1] != ks[1] or qs[3] != ks[3]:
        raise GddimError("q %s and k %s must agree in all but their heads" % (tuple(qs), tuple(ks)))
    if not (0.0 <= eps < math.inf):
        raise GddimError("eps=%r must be finite and not negative" % (eps,))
    w_q, w_k = _norm_weight(w_q, "weight_q", q), _norm_weight(w_k, "weight_k", q)
    if w_q is not None and w_k is not None and w_q.dtype is not w_k.dtype:
        raise GddimError("weight_q is %s, weight_k %s: their types must agree" % (w_q.dtype, w_k.dtype))
    w = w_q if w_q is not None else w_k
    return (w_q, w_k, w_q.data_ptr() if w_q is not None else None, w_k.data_ptr() if w_k is not None else None,
            int(w is not None and w.dtype is not q.dtype))


def qk_norm_rotary(q, k, weight_q, weight_k, pos, axes, eps=1e-6):
    """RMS norms of queries and keys for each head, then the rotation, in one pass: q (B, N, heads, D) and k (B, N, key heads, D), views of a
    packed projection among them, weights (D,) of their type or float32 (None: ones).  Returns (q', k')."""
    w_q, w_k, p_q, p_k, w_f32 = _check_qk(q, k, weight_q, weight_k, eps)
    desc = _rotary_desc(q, pos, axes)
    qo, ko = _new(q), _new(k)
    (q, qv), (k, kv) = _heads(q), _heads(k)
    _call(q, _abi.lib().gd_qk_norm_rotary, desc, qv, kv, _dense_heads(qo), _dense_heads(ko), q.shape[2], k.shape[2], p_q, p_k, w_f32, eps)
    return qo, ko


def qk_norm_rotary_backward(dq_out, dk_out, q, k, weight_q, weight_k, pos, axes, eps=1e-6):
    """Gradients of qk_norm_rotary: (dq, dk, dweight_q, dweight_k) from those of its outputs (None for a weight that is None).  The same bits
    every time."""
    torch = _torch()[0]
    w_q, w_k, p_q, p_k, w_f32 = _check_qk(q, k, weight_q, weight_k, eps)
    for g, name, t in ((dq_out, "dq_out", q), (dk_out, "dk_out", k)):
        _check_heads(g, name, q, "q")
        if g.shape != t.shape:
            raise GddimError("%s has shape %s, expected %s" % (name, tuple(g.shape), tuple(t.shape)))
    desc = _rotary_desc(q, pos, axes)
    dq, dk = _new(q), _new(k)
    dwq, dwk = (torch.empty_like(w) if w is not None else None for w in (w_q, w_k))
    (q, qv), (k, kv), (dq_out, gqv), (dk_out, gkv) = _heads(q), _heads(k), _heads(dq_out), _heads(dk_out)
    lib = _abi.lib()
    ws = q.new_empty(lib.gd_qk_norm_rotary_backward_workspace(q.shape[3]), dtype=torch.uint8)
    _call(q, lib.gd_qk_norm_rotary_backward, desc, gqv, gkv, qv, kv, _dense_heads(dq), _dense_heads(dk), q.shape[2], k.shape[2], p_q, p_k, w_f32, eps, ws.data_ptr(),
          dwq.data_ptr() if dwq is not None else None, dwk.data_ptr() if dwk is not None else None)
    return dq, dk, dwq, dwk


# ---- gated feed-forward block ------------------------------------------------------------------------------------------------
_ACTS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}


def _rows(t, columns):
    """t (..., columns) as a matrix with adjacent columns and rows at least a row apart: a view where there is one"""
    if columns == 1:
        t = t.resolve_neg()  # (a lazily negated view has strides of two or more, the imaginary part of a conjugate; with more columns it is copied below)
    if t.dim() == 2 and t.is_contiguous():
        return t
    if t.dim() != 2:
        t = t.reshape(-1, columns)
    if (columns > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < columns):
        t = t.contiguous()
    return t


def _check_ffn(x, w_gate, w_up, w_down, act):
    """(x as a matrix, the weights with adjacent columns, the fields of gd_ffn_desc)"""
    _on_gpu(x, "x")
    code, kind = _torch()[1].get(x.dtype), _ACTS.get(act)
    if kind is None:
        raise GddimError("act=%r, expected one of %s" % (act, sorted(_ACTS)))
    if code is None:
        raise GddimError("x is %s; float32, bfloat16 and float16 are supported" % x.dtype)
    _like(w_gate, "w_gate", x, "x")
    _like(w_up, "w_up", x, "x")
    _like(w_down, "w_down", x, "x")
    xs, gs, us, ds = tuple(x.shape), tuple(w_gate.shape), tuple(w_up.shape), tuple(w_down.shape)
    if not xs or len(gs) != 2 or len(ds) != 2 or gs != us or gs[1] != xs[-1] or ds[1] != gs[0] or 0 in gs or ds[0] == 0:
        raise GddimError("x %s, w_gate %s, w_up %s, w_down %s do not fit (..., in), (hidden, in), (hidden, in), (out, hidden)" % (xs, gs, us, ds))
    x, w_gate, w_up, w_down = _rows(x, gs[1]), _rows(w_gate, gs[1]), _rows(w_up, gs[1]), _rows(w_down, gs[0])
    ld = w_gate.stride(0)
    if ld != w_up.stride(0):  # (of a single row: never used)
        if gs[0] > 1:
            w_gate, w_up = w_gate.contiguous(), w_up.contiguous()
        ld = gs[1]
    rows = x.shape[0]
    if rows > 1 << 30 or gs[0] > 1 << 30 or gs[1] > 1 << 30 or ds[0] > 1 << 30:
        raise GddimError("sizes past 2^30: %d rows, %d -> %d -> %d" % (rows, gs[1], gs[0], ds[0]))
    unaligned = int((x.data_ptr() | w_gate.data_ptr() | w_up.data_ptr() | w_down.data_ptr()) & 15 != 0)
    return x, w_gate, w_up, w_down, (code, kind, rows, gs[1], gs[0], ds[0], unaligned, x.stride(0), ld, w_down.stride(0))


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(fields, backward, device):
    """gd_gated_ffn_workspace of these sizes on this device (its compute units count)"""
    with _torch()[0].cuda.device(device):
        n = _abi.lib().gd_gated_ffn_workspace(_FFN.pack(*fields), backward)
    if n < 0:
        check(1)
    return n


def _workspace(x, fields, backward):
    """(tensor or None, its address or None)"""
    n = _workspace_bytes(fields, backward, x.get_device())
    if not n:
        return None, None
    t = x.new_empty(n, dtype=_torch()[0].uint8)
    return t, t.data_ptr()


def gated_ffn(x, w_gate, w_up, w_down, act="silu", save=False):
    """Gated feed-forward block (act(x w_gate^T) * (x w_up^T)) w_down^T: x (..., in), weights as torch.nn.Linear keeps them -- w_gate and w_up
    (hidden, in), w_down (out, hidden) -- act 'silu', 'gelu' or 'gelu_tanh'.  Returns y (..., out); with save=True (y, saved), saved for
    gated_ffn_backward (the two projections in float32 and their product).  Both projections, the activation and the product are one kernel where the
    sums are not split; where they are (little to fill the chip with), a second one joins them and applies activation and product."""
    x_in = x
    x, w_gate, w_up, w_down, fields = _check_ffn(x, w_gate, w_up, w_down, act)
    rows, F, O = fields[2], fields[4], fields[5]
    y, hidden = x.new_empty((rows, O)), x.new_empty((rows, F))
    ws, ws_at = _workspace(x, fields, 0)
    if save:
        gate, up = (x.new_empty((rows, F), dtype=_torch()[0].float32) for _ in range(2))
    _call(x, _abi.lib().gd_gated_ffn, _FFN.pack(*fields), x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(), gate.data_ptr() if save else None,
          up.data_ptr() if save else None, hidden.data_ptr(), y.data_ptr(), ws_at)
    if x_in.dim() != 2:
        y = y.view(*x_in.shape[:-1], O)
    return (y, (gate, up, hidden)) if save else y


def gated_ffn_backward(dy, x, w_gate, w_up, w_down, saved, act="silu"):
    """Gradients (dx, dw_gate, dw_up, dw_down) of gated_ffn from that of its result and what the call with save=True kept (left as it was).  The
    same bits every time.  The gradients of both projections are rounded to x's type before they are summed: in float16 past 65504 infinite, under
    2^-25 zero."""
    x_in = x
    x, w_gate, w_up, w_down, fields = _check_ffn(x, w_gate, w_up, w_down, act)
    M, D, F, O = fields[2:6]
    _like(dy, "dy", x, "x")
    if dy.shape != x_in.shape[:-1] + (O,):
        raise GddimError("dy has shape %s, expected %s" % (tuple(dy.shape), tuple(x_in.shape[:-1]) + (O,)))
    if not isinstance(saved, tuple) or len(saved) != 3:
        raise GddimError("saved: expected the second result of gated_ffn(..., save=True)")
    for t, name in zip(saved, ("gate", "up", "hidden")):
        _on_gpu(t, "saved " + name)
        if t.dtype is not (x.dtype if name == "hidden" else _torch()[0].float32) or t.get_device() != x.get_device():
            raise GddimError("saved %s is %s on %s: not what gated_ffn(..., save=True) gave for x" % (name, t.dtype, t.device))
        if tuple(t.shape) != (M, F) or not t.is_contiguous():
            raise GddimError("saved %s has shape %s, expected (%d, %d), dense" % (name, tuple(t.shape), M, F))
    dy = _rows(dy, O)
    gate, up, hidden = saved
    apart = dy.stride(0) * dy.element_size() if M > 1 else 0  # rows of dy: within what the aligned path takes, where dense ones would be
    if (dy.data_ptr() | gate.data_ptr() | up.data_ptr() | hidden.data_ptr()) & 15 or (dy.stride(0) != O and (apart % 16 or apart > 1 << 22)):
        fields = fields[:6] + (1,) + fields[7:]
    dx, dwg, dwu, dwd = x.new_empty((M, D)), x.new_empty((F, D)), x.new_empty((F, D)), x.new_empty((O, F))
    ws, ws_at = _workspace(x, fields, 1)
    _call(x, _abi.lib().gd_gated_ffn_backward, _FFN.pack(*fields), dy.data_ptr(), dy.stride(0), x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(),
          w_down.data_ptr(), gate.data_ptr(), up.data_ptr(), hidden.data_ptr(), dx.data_ptr(), dwg.data_ptr(), dwu.data_ptr(), dwd.data_ptr(), ws_at)
    return dx.view(x_in.shape), dwg, dwu, dwd
