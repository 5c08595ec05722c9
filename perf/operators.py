"""Measured cases of the token operators: positions with several axes, norms of queries and keys for each head with the rotation in the
same pass, and the gated feed-forward block -- what a score network made of attention blocks runs beside the two products of its attention.

`run` computes one pass of a case: in plain torch operations while `own` is false, through gddim_amd.ops where it is true.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_POS = {"i32": torch.int32, "i64": torch.int64, "f32": torch.float32}


def _rotary_case(name, **kw):
    case = dict(op="rotary", name=name, B=1, N=1, H=1, D=64, sections="32,32", paired="interleaved", pos="i64", shared_pos=True, far=0,
                inverse=False, type="bf16")
    case.update(kw)
    return case


def _qk_case(name, **kw):
    case = dict(op="qk_norm_rotary", name=name, B=1, N=1, H=1, Hk=1, D=64, sections="32,32", paired="interleaved", pos="i64",
                shared_pos=True, far=0, train=False, type="bf16")
    case.update(kw)
    return case


def _ffn_case(name, **kw):
    case = dict(op="gated_ffn", name=name, M=1, D=256, F=684, act="silu", train=False, type="bf16")
    case.update(kw)
    return case


def listed():
    return [
        # one new token for each of 8 running sequences, far along their single axis: all latency
        _rotary_case("rotary_step", B=8, N=1, H=8, D=64, sections="64", paired="halves", shared_pos=False, far=1 << 20),
        # a batch of 32x32 images and one class token in float32, the type of the framework's own networks
        _rotary_case("rotary_image", B=16, N=1025, H=8, D=64, sections="32,32", pos="i32", type="f32"),
        # one clip of 13 x 45 x 80 latent tokens: time, height and width
        _rotary_case("rotary_video", B=1, N=46800, H=16, D=128, sections="16,56,56"),
        # one new token for each of 4 sequences, four queries to a key
        _qk_case("qk_step", B=4, N=1, H=16, Hk=4, D=128, sections="128", paired="halves", shared_pos=False, far=1 << 17),
        # the 16x16 attention level of the CIFAR-10 networks (256 channels) at the benchmark's batch, float32
        _qk_case("qk_image", B=256, N=256, H=4, Hk=4, D=64, sections="32,32", pos="i32", type="f32"),
        # a training step over a clip: shared key heads, an odd number of tokens
        _qk_case("qk_video_train", B=2, N=8191, H=16, Hk=4, D=128, sections="32,48,48", train=True),
        # a training step where nothing is a power of two: part of each head rotates, positions lie between the pixels
        _qk_case("qk_odd_train", B=3, N=777, H=6, Hk=6, D=72, sections="24,24", pos="f32", shared_pos=False, train=True, type="f16"),
        # one conditioning vector: the weights' bytes
        _ffn_case("ffn_single", M=1, D=1024, F=2736),
        # a few rows, one more than a tile holds
        _ffn_case("ffn_rows", M=33, D=1024, F=4096, act="gelu", type="f16"),
        # a training step over 16 images of 16x16 tokens at 256 channels in float32
        _ffn_case("ffn_image_train", M=4096, D=256, F=684, train=True, type="f32"),
        # the forward pass of 8 images of 32x32 tokens and a class token
        _ffn_case("ffn_image", M=8200, D=512, F=1368, act="gelu_tanh"),
        # a training step over a long clip
        _ffn_case("ffn_video_train", M=16384, D=1024, F=4096, train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _sections(rng, D):
    pairs = D // 2 if rng.random() < 0.7 else max(1, D // 3)
    axes = min(rng.choice([1, 2, 3]), pairs)
    cuts = sorted(rng.sample(range(1, pairs), axes - 1)) if axes > 1 else []
    return ",".join(str(2 * (b - a)) for a, b in zip([0] + cuts, cuts + [pairs]))


def draw(rng):
    op = rng.choice(["rotary", "qk_norm_rotary", "gated_ffn"])
    typ = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "gated_ffn":
        M, D, F = _log_int(rng, 1, 16384), _log_int(rng, 64, 1024), _log_int(rng, 128, 4096)
        if rng.random() < 0.7:  # most networks keep whole vectors
            D, F = -(-D // 8) * 8, -(-F // 8) * 8
        if typ == "f32":
            M = min(M, 8192)
        return dict(op=op, M=M, D=D, F=F, act=rng.choice(["silu", "gelu", "gelu_tanh"]), train=rng.random() < 0.5, type=typ)
    D = rng.choice([16, 32, 40, 64, 64, 72, 80, 96, 128, 128, 192, 256])
    H = rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 24])
    B = _log_int(rng, 1, 64)
    N = _log_int(rng, 1, 16384)
    N = max(1, min(N, 90_000_000 // (B * H * D)))
    case = dict(op=op, B=B, N=N, H=H, D=D, sections=_sections(rng, D), paired=rng.choice(["interleaved", "halves"]),
                pos=rng.choice(["i32", "i64", "f32"]), shared_pos=rng.random() < 0.5, far=rng.choice([0, 0, 1 << 16, 1 << 22]), type=typ)
    if op == "rotary":
        case["inverse"] = rng.random() < 0.3
    else:
        case["N"] = max(1, min(N, 22_000_000 // (B * H * D)))
        case["Hk"] = rng.choice([h for h in (1, 2, 3, 4, 6, 8, 12, 16, 24) if H % h == 0])
        case["train"] = rng.random() < 0.5
    return case


def _axis_of_pairs(sections):
    return [a for a, s in enumerate(sections) for _ in range(s // 2)]


def _frequencies(sections):
    return [10000.0 ** (-2.0 * j / s) for s in sections for j in range(s // 2)]


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    typ = _TYPES[case["type"]]

    def normal(*shape, scale=1.0, dtype=typ):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    state = dict(case)
    if case["op"] == "gated_ffn":
        M, D, F = case["M"], case["D"], case["F"]
        state.update(x=normal(M, D), w_gate=normal(F, D, scale=D ** -0.5), w_up=normal(F, D, scale=D ** -0.5),
                     w_down=normal(D, F, scale=F ** -0.5))
        if case["train"]:
            state["dy"] = normal(M, D)
        return state
    B, N, H, D = case["B"], case["N"], case["H"], case["D"]
    sections = tuple(int(s) for s in case["sections"].split(","))
    A = len(sections)
    # token positions: rows of a grid, or anywhere up to `far`; fractional ones where a grid of another resolution is mapped in
    shape = (N, A) if case["shared_pos"] else (B, N, A)
    if case["far"]:
        pos = torch.randint(0, case["far"], shape, generator=g, device="cuda")
    else:
        side = max(1, round(N ** (1.0 / A)))
        n = torch.arange(N, device="cuda")
        pos = torch.stack([torch.div(n, side ** (A - 1 - a), rounding_mode="floor") % (side if a else 1 << 30) for a in range(A)], -1)
        if not case["shared_pos"]:
            pos = pos + torch.randint(0, 8, (B, 1, A), generator=g, device="cuda")
    if case["pos"] == "f32":
        pos = pos.float() * 0.75
    state.update(pos=pos.to(_POS[case["pos"]]), sections=sections,
                 freq=torch.tensor(_frequencies(sections), dtype=torch.float64, device="cuda"),
                 pair_axis=torch.tensor(_axis_of_pairs(sections), device="cuda"))
    if case["op"] == "rotary":
        state["x"] = normal(B, N, H, D)
    else:
        Hk = case["Hk"]
        qkv = normal(B, N, H + 2 * Hk, D)  # the packed projection that a block has in hand; values are not touched here
        state.update(q=qkv[:, :, :H], k=qkv[:, :, H:H + Hk], eps=1e-6)
        state.update(w_q=(1.0 + normal(D, scale=0.2, dtype=torch.float32)).to(typ), w_k=(1.0 + normal(D, scale=0.2, dtype=torch.float32)).to(typ))
        if case["train"]:
            state.update(dq_out=normal(B, N, H, D), dk_out=normal(B, N, Hk, D))
    if own:
        from gddim_amd import ops
        state["axes"] = ops.RotaryAxes(sections, theta=10000.0, paired=case["paired"], device="cuda")
    return state


# ---- plain forms -------------------------------------------------------------------------------------------
def _cos_sin(s):
    # far positions times a frequency: the angle in 64 bits, its cosine and sine rounded to 32
    angle = s["pos"].double()[..., s["pair_axis"]] * s["freq"]
    if s["shared_pos"]:
        angle = angle.unsqueeze(0)
    angle = angle.unsqueeze(2)
    return torch.cos(angle).float(), torch.sin(angle).float()


def _rotate(x, cos, sin, s, inverse=False):
    R = sum(s["sections"])
    rot, rest = x[..., :R], x[..., R:]
    if inverse:
        sin = -sin
    if s["paired"] == "interleaved":
        a, b = rot[..., 0::2], rot[..., 1::2]
        out = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = rot[..., :R // 2], rot[..., R // 2:]
        out = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((out, rest), -1) if rest.shape[-1] else out


def _norm_rotate(x, w, cos, sin, s):
    x = x.float()
    return _rotate(x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * w.float(), cos, sin, s)


def _norm_rotate_backward(dy, x, w, cos, sin, s):
    x, w = x.float(), w.float()
    g = _rotate(dy.float(), cos, sin, s, inverse=True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"])
    xh = x * r
    gw = g * w
    dx = r * (gw - xh * (gw * xh).mean(-1, keepdim=True))
    return dx, (g * xh).sum((0, 1, 2))


def _act(z, act):
    """activation and its derivative"""
    if act == "silu":
        t = 1.0 / (1.0 + torch.exp(-z))
        return z * t, t * (1.0 + z * (1.0 - t))
    if act == "gelu":
        c = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * c, c + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    k, c = math.sqrt(2.0 / math.pi), 0.044715
    t = torch.tanh(k * (z + c * z * z * z))
    return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * k * (1.0 + 3.0 * c * z * z)


def _ffn(s):
    typ = s["x"].dtype
    x, wg, wu, wd = s["x"].float(), s["w_gate"].float(), s["w_up"].float(), s["w_down"].float()
    gate, up = x @ wg.t(), x @ wu.t()
    a, da = _act(gate, s["act"])
    h = a * up
    y = h @ wd.t()
    if not s["train"]:
        return y.to(typ)
    dy = s["dy"].float()
    dh = dy @ wd
    dgate, dup = dh * up * da, dh * a
    grads = (dgate @ wg + dup @ wu, dgate.t() @ x, dup.t() @ x, dy.t() @ h)
    return (y.to(typ),) + tuple(t.to(typ) for t in grads)


def _run_plain(s):
    if s["op"] == "gated_ffn":
        return _ffn(s)
    cos, sin = _cos_sin(s)
    if s["op"] == "rotary":
        return _rotate(s["x"].float(), cos, sin, s, s["inverse"]).to(s["x"].dtype)
    typ = s["q"].dtype
    out = tuple(_norm_rotate(x, w, cos, sin, s).to(typ) for x, w in ((s["q"], s["w_q"]), (s["k"], s["w_k"])))
    if not s["train"]:
        return out
    dq, dwq = _norm_rotate_backward(s["dq_out"], s["q"], s["w_q"], cos, sin, s)
    dk, dwk = _norm_rotate_backward(s["dk_out"], s["k"], s["w_k"], cos, sin, s)
    return out + (dq.to(typ), dk.to(typ), dwq.to(typ), dwk.to(typ))


def _run_own(s):
    from gddim_amd import ops
    if s["op"] == "rotary":
        return ops.rotary(s["x"], s["pos"], s["axes"], inverse=s["inverse"])
    if s["op"] == "qk_norm_rotary":
        out = ops.qk_norm_rotary(s["q"], s["k"], s["w_q"], s["w_k"], s["pos"], s["axes"], eps=s["eps"])
        if not s["train"]:
            return out
        return out + ops.qk_norm_rotary_backward(s["dq_out"], s["dk_out"], s["q"], s["k"], s["w_q"], s["w_k"], s["pos"], s["axes"],
                                                 eps=s["eps"])
    if not s["train"]:
        return ops.gated_ffn(s["x"], s["w_gate"], s["w_up"], s["w_down"], act=s["act"])
    y, saved = ops.gated_ffn(s["x"], s["w_gate"], s["w_up"], s["w_down"], act=s["act"], save=True)
    return (y,) + ops.gated_ffn_backward(s["dy"], s["x"], s["w_gate"], s["w_up"], s["w_down"], saved, act=s["act"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}[case["type"]]
    if case["op"] == "gated_ffn":
        M, D, F = case["M"], case["D"], case["F"]
        weights, rows = 3 * D * F, M * D
        if case["train"]:  # x, dy, the weights in; y, dx and the weights' gradients out
            return {"bytes": size * (2 * weights + 4 * rows), "flops": 18.0 * M * D * F}
        return {"bytes": size * (weights + 2 * rows), "flops": 6.0 * M * D * F}
    B, N, D = case["B"], case["N"], case["D"]
    A = len(case["sections"].split(","))
    pos = (N if case["shared_pos"] else B * N) * A * {"i32": 4, "i64": 8, "f32": 4}[case["pos"]]
    if case["op"] == "rotary":
        elements = B * N * case["H"] * D
        return {"bytes": 2 * size * elements + pos, "flops": 3.0 * elements}
    elements = B * N * (case["H"] + case["Hk"]) * D
    if case["train"]:
        return {"bytes": size * (4 * elements + 4 * D) + pos, "flops": 24.0 * elements}
    return {"bytes": size * (2 * elements + 2 * D) + pos, "flops": 8.0 * elements}


# ---- the definition in 64 bits: rotations as products of complex numbers, gradients by differentiation -------------------------------
def _exact_rotate(x, s, sign=1.0):
    angle = torch.stack([s["pos"][..., a].double() * f for a, f in zip(_axis_of_pairs(s["sections"]), _frequencies(s["sections"]))], -1)
    if s["shared_pos"]:
        angle = angle[None]
    turn = torch.polar(torch.ones_like(angle), sign * angle)[:, :, None]
    R = sum(s["sections"])
    rot = x[..., :R]
    if s["paired"] == "interleaved":
        z = torch.view_as_complex(rot.reshape(*rot.shape[:-1], R // 2, 2)) * turn
        out = torch.view_as_real(z).reshape(rot.shape)
    else:
        z = torch.complex(rot[..., :R // 2].contiguous(), rot[..., R // 2:].contiguous()) * turn
        out = torch.cat((z.real, z.imag), -1)
    return torch.cat((out, x[..., R:]), -1)


def _exact_act(z, act):
    if act == "silu":
        return torch.nn.functional.silu(z)
    return torch.nn.functional.gelu(z, approximate="tanh" if act == "gelu_tanh" else "none")


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "rotary":
        return _exact_rotate(s["x"].double(), s, -1.0 if s["inverse"] else 1.0)
    if s["op"] == "qk_norm_rotary":
        leaves = [s[n].double().requires_grad_(s["train"]) for n in ("q", "k", "w_q", "w_k")]
        out = []
        for x, w in ((leaves[0], leaves[2]), (leaves[1], leaves[3])):
            rms = torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + s["eps"])
            out.append(_exact_rotate(x / rms * w, s))
        if not s["train"]:
            return tuple(out)
        grads = torch.autograd.grad(out, leaves, [s["dq_out"].double(), s["dk_out"].double()])
        return tuple(t.detach() for t in out) + tuple(grads)
    leaves = [s[n].double().requires_grad_(s["train"]) for n in ("x", "w_gate", "w_up", "w_down")]
    x, wg, wu, wd = leaves
    F = torch.nn.functional
    y = F.linear(_exact_act(F.linear(x, wg), s["act"]) * F.linear(x, wu), wd)
    if not s["train"]:
        return y
    return (y.detach(),) + tuple(torch.autograd.grad(y, leaves, s["dy"].double()))
