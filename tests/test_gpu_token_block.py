"""The token operators together, as an attention block over 16x16 image tokens runs them beside the framework's own projections and attention core: projection,
query / key norms with row and column positions, attention, residual, gated feed-forward block, residual -- eagerly and from a captured graph."""
import pytest
import torch

import token_reference as ref

pytestmark = pytest.mark.gpu


def _weights(C, F, dev):
    g = torch.Generator(dev).manual_seed(0)
    n = lambda *s, scale=1.0: torch.randn(s, generator=g, device=dev) * scale
    return dict(qkv=n(3 * C, C, scale=C ** -0.5), nq=1 + n(64, scale=0.1), nk=1 + n(64, scale=0.1), gate=n(F, C, scale=C ** -0.5), up=n(F, C, scale=C ** -0.5),
                down=n(C, F, scale=F ** -0.5))


def _block(x, w, pos, axes):
    from gddim_amd import ops
    B, N, C = x.shape
    H = C // 64
    qkv = ops.conv2d(x.view(B, 16, 16, C), w["qkv"], KH=1, KW=1, pad=0).view(B, N, 3 * H, 64)
    q, k = ops.qk_norm_rotary(qkv[:, :, :H], qkv[:, :, H:2 * H], w["nq"], w["nk"], pos, axes)
    packed = torch.cat([t.transpose(1, 2).reshape(B * H, N, 64) for t in (q, k, qkv[:, :, 2 * H:])], -1)
    a = ops.attention(packed).view(B, H, N, 64).transpose(1, 2).reshape(B, N, C)
    h = x + a
    return h + ops.gated_ffn(h, w["gate"], w["up"], w["down"])


def _block64(x, w, pos):
    x, w = x.double().cpu(), {k: v.double().cpu() for k, v in w.items()}
    B, N, C = x.shape
    H = C // 64
    qkv = (x @ w["qkv"].t()).view(B, N, 3 * H, 64)
    phi = ref.angles(pos, (32, 32), 100.0, B, N)
    q = ref.norm_rotary(qkv[:, :, :H], w["nq"], phi, (32, 32), "interleaved", 1e-6)[0].transpose(1, 2)
    k = ref.norm_rotary(qkv[:, :, H:2 * H], w["nk"], phi, (32, 32), "interleaved", 1e-6)[0].transpose(1, 2)
    a = torch.softmax(q @ k.transpose(-1, -2) / 8.0, -1) @ qkv[:, :, 2 * H:].transpose(1, 2)
    h = x + a.transpose(1, 2).reshape(B, N, C)
    return h + ref.gated_ffn(h, w["gate"], w["up"], w["down"], "silu", torch.float64).val


def test_attention_block_over_image_tokens(native_lib):
    from gddim_amd import ops
    dev = torch.device("cuda", 0)
    B, N, C, F = 3, 256, 256, 684
    w = _weights(C, F, dev)
    side = torch.arange(16)
    pos = torch.stack(torch.meshgrid(side, side, indexing="ij"), -1).reshape(N, 2)
    axes = ops.RotaryAxes((32, 32), theta=100.0, device=dev)
    x = torch.randn(B, N, C, generator=torch.Generator(dev).manual_seed(1), device=dev)
    pos_dev = pos.to(dev)
    y = _block(x, w, pos_dev, axes)
    want = _block64(x, w, pos)
    # sums of up to 684 float32 terms, five in a row, a softmax of scores up to ~64 between them: 5 * 684 * 2^-24 = 2e-4 of the values, if all roundings
    # went one way
    assert float((y.cpu().double() - want).abs().max()) < 2e-4 * float(want.abs().max())

    # the block's token operators in a graph (the attention core keeps a scratch of its own shape per call; all memory comes from the graph's pool)
    graph = torch.cuda.CUDAGraph()
    side_stream = torch.cuda.Stream()
    side_stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side_stream):
        _block(x, w, pos_dev, axes)
    torch.cuda.current_stream().wait_stream(side_stream)
    with torch.cuda.graph(graph):
        captured = _block(x, w, pos_dev, axes)
    for trial in range(4):
        x.copy_(torch.randn(B, N, C, generator=torch.Generator(dev).manual_seed(trial + 2), device=dev))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, _block(x, w, pos_dev, axes))


def test_gradients_through_norms_and_feed_forward(native_lib):
    """Forward and backward of the feed-forward block and of the norms chained by hand: the gradient of a loss through both is the product of theirs."""
    from gddim_amd import ops
    dev = torch.device("cuda", 0)
    B, N, H, D, F = 2, 33, 4, 64, 344
    C = H * D
    g = torch.Generator(dev).manual_seed(3)
    n = lambda *s, scale=1.0: torch.randn(s, generator=g, device=dev) * scale
    x, wq, wk, wg, wu, wd = n(B, N, 2 * C), 1 + n(D, scale=0.1), 1 + n(D, scale=0.1), n(F, C, scale=C ** -0.5), n(F, C, scale=C ** -0.5), n(C, F, scale=F ** -0.5)
    pos = torch.randint(0, 40, (N, 2), generator=g, device=dev)
    axes = ops.RotaryAxes((32, 32), device=dev)
    q, k = x.view(B, N, 2 * H, D)[:, :, :H], x.view(B, N, 2 * H, D)[:, :, H:]
    dy, dk_out = n(B, N, C), n(B, N, H, D)
    q2, k2 = ops.qk_norm_rotary(q, k, wq, wk, pos, axes)
    y, saved = ops.gated_ffn(q2.view(B, N, C), wg, wu, wd, save=True)
    dq2, *dw = ops.gated_ffn_backward(dy, q2.view(B, N, C), wg, wu, wd, saved)
    dq, dk, dwq, dwk = ops.qk_norm_rotary_backward(dq2.view(B, N, H, D), dk_out, q, k, wq, wk, pos, axes)
    leaves = [t.double().cpu().requires_grad_() for t in (x, wq, wk, wg, wu, wd)]
    phi = ref.angles(pos, (32, 32), 10000.0, B, N)
    xa = leaves[0].view(B, N, 2 * H, D)

    def turned(t, w):
        z = t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * w
        c = torch.view_as_complex(z.reshape(*z.shape[:-1], D // 2, 2)) * torch.polar(torch.ones_like(phi), phi)[:, :, None]
        return torch.view_as_real(c).reshape(z.shape)

    f = torch.nn.functional
    h = turned(xa[:, :, :H], leaves[1]).reshape(B, N, C)
    out = f.linear(f.silu(f.linear(h, leaves[3])) * f.linear(h, leaves[4]), leaves[5])
    loss = (out * dy.double().cpu()).sum() + (turned(xa[:, :, H:], leaves[2]) * dk_out.double().cpu()).sum()
    want = torch.autograd.grad(loss, leaves)
    got = [torch.cat((dq, dk), 2).view(B, N, 2 * C), dwq, dwk] + dw
    for i, (a, b) in enumerate(zip(got, want)):
        # float32 sums of up to 344 terms, three in a row: 3 * 344 * 2^-24 = 6e-5, and the norms' 64
        assert float((a.cpu().double() - b).abs().max()) < 1e-4 * float(b.abs().max()), i


def test_forward_mode_tangents_are_refused(native_lib):
    from torch.autograd import forward_ad
    from gddim_amd import ops
    from gddim_amd._abi import GddimError
    dev = torch.device("cuda", 0)
    x, w, pos = torch.randn(1, 2, 1, 4, device=dev), torch.randn(4, device=dev), torch.zeros(2, 1, device=dev)
    axes, m, a = ops.RotaryAxes((4,), device=dev), torch.randn(2, 4, device=dev), torch.randn(4, 4, device=dev)
    y, saved = ops.gated_ffn(m, a, a, a, save=True)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: ops.rotary(x, dual(pos), axes), lambda: ops.qk_norm_rotary(x, dual(x), w, w, pos, axes), lambda: ops.qk_norm_rotary(x, x, dual(w), w, pos, axes),
                     lambda: ops.qk_norm_rotary_backward(x, dual(x), x, x, w, w, pos, axes), lambda: ops.gated_ffn(m, a, dual(a), a), lambda: ops.gated_ffn(m, a, a, dual(a)),
                     lambda: ops.gated_ffn_backward(dual(m), m, a, a, a, saved), lambda: ops.gated_ffn_backward(m, m, a, a, a, (dual(saved[0]),) + saved[1:])):
            with pytest.raises(GddimError, match="tangent"):
                call()
        assert torch.equal(ops.gated_ffn(m, a, a, a), y)  # tensors without one are taken inside a level, too
