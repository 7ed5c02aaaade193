"""The training pass as a user runs it: projections, Q/K norm + rotation and attention in one differentiable chain, its
gradients against the explicit operators' (which have their own tests against the formulas) and against 64-bit
autograd, and the attention backend's switch to it."""

import math

import pytest
import torch

from gpu_util import status_clean

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.fixture(scope="module")
def lib(ogx_lib):
    from opengenie_b200 import attention_backend, ltx_ops, training

    return ltx_ops, training, attention_backend


def _inputs(B, L, heads, kv_heads, seed=0, norm="head"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    x = (r(B, L, 256)).to(BF)
    w = (r((heads + 2 * kv_heads) * 128, 256) / 16).to(BF).requires_grad_()
    wide = (128, 128) if norm == "head" else (heads * 128, kv_heads * 128)
    qw, kw = ((1 + 0.1 * r(n)).to(BF).requires_grad_() for n in wide)
    freq = 100.0 ** (-torch.arange(64, device="cuda") / 64)
    angle = torch.arange(L, device="cuda")[:, None] * freq
    return x, w, qw, kw, angle.cos()[None], angle.sin()[None]


@pytest.mark.parametrize("norm,heads,kv_heads,inter", [("head", 4, 2, True), ("row", 2, 2, False)])
def test_chain_matches_the_explicit_operators_and_64_bit_autograd(lib, norm, heads, kv_heads, inter):
    ops, training, _ = lib
    B, L, block = 2, 250, 50
    x, w, qw, kw, cos, sin = _inputs(B, L, heads, kv_heads, norm=norm)
    lengths = torch.tensor([250, 130], device="cuda", dtype=torch.int32)
    split = [heads * 128, kv_heads * 128, kv_heads * 128]
    masks = dict(kv_heads=kv_heads, causal_block=block, q_lengths=lengths, kv_lengths=lengths)
    layout = dict(kv_heads=kv_heads, norm=norm, interleaved=inter)

    qkv = torch.nn.functional.linear(x, w)
    q, k, v = qkv.split(split, -1)
    qr, kr = training.qk_norm_rope(q, k, qw, kw, 1e-6, cos, sin, heads, **layout)
    out = training.attention(qr, kr, v, heads, **masks)
    target = torch.randn(out.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9)).to(BF)
    loss = (out.float() * target.float()).sum()
    got = torch.autograd.grad(loss, (w, qw, kw))
    assert status_clean()

    # the same pass with the explicit operators: bit for bit
    with torch.no_grad():
        q2, k2 = ops.fused_qk_norm_rope(q, k, qw, kw, 1e-6, cos, sin, heads, **layout)
        out2, lse = ops.attention_with_lse(q2, k2, v, heads, **masks)
        assert torch.equal(out, out2)
        dqr, dkr, dv = ops.attention_backward(target, q2, k2, v, out2, lse, heads, **masks)
        dq, dk, dqw, dkw = ops.fused_qk_norm_rope_backward(dqr, dkr, q, k, qw, kw, 1e-6, cos, sin, heads, **layout)
        dw = torch.cat((dq, dk, dv), -1).flatten(0, 1).t() @ x.flatten(0, 1)
    assert torch.equal(got[1], dqw.to(BF)) and torch.equal(got[2], dkw.to(BF))
    assert torch.equal(got[0], dw)

    # 64-bit autograd of the whole chain.  Each stage rounds its bf16 results by at most 2^-8 of their size; five stages
    # of independent roundings lie between the weights and their gradients, each summed over hundreds of rows, so the
    # gradients' difference is a few 2^-8 of their norm at most: 5 * 2^-8 = 0.02.
    w64, qw64, kw64 = (t.detach().double().requires_grad_() for t in (w, qw, kw))
    q, k, v = (x.double() @ w64.t()).split(split, -1)

    def rotate(t, weight, n):
        t = t.unflatten(-1, (n, 128))
        over = (-1,) if norm == "head" else (-2, -1)
        t = t * torch.rsqrt(t.square().mean(over, keepdim=True) + 1e-6) * weight.view(-1, 128)
        c, s = cos.double().unsqueeze(2), sin.double().unsqueeze(2)
        a, b = (t[..., 0::2], t[..., 1::2]) if inter else t.chunk(2, -1)
        pair = a * c - b * s, b * c + a * s
        return (torch.stack(pair, -1).flatten(-2) if inter else torch.cat(pair, -1)).transpose(1, 2)

    q, k = rotate(q, qw64, heads), rotate(k, kw64, kv_heads).repeat_interleave(heads // kv_heads, 1)
    v = v.unflatten(-1, (kv_heads, 128)).transpose(1, 2).repeat_interleave(heads // kv_heads, 1)
    i = torch.arange(L, device="cuda")
    see = (i[None] // block <= i[:, None] // block) & (i < lengths[:, None, None, None])
    rows = (i[None, :, None] < lengths[:, None, None])[:, None]
    p = torch.softmax((q @ k.transpose(-1, -2) * 128 ** -0.5).masked_fill(~see, -math.inf), -1)
    ref = (torch.where(rows, p @ v, 0.0)).transpose(1, 2).flatten(2)
    for a, b in zip(got, torch.autograd.grad((ref * target.double()).sum(), (w64, qw64, kw64))):
        assert (a.double() - b).norm() <= 5 * 2.0 ** -8 * b.norm()


def test_expanded_and_transposed_gradients(lib):
    ops, training, _ = lib
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn((2, 60, 256), device="cuda", generator=g).to(BF).requires_grad_() for _ in range(3))
    out = training.attention(q, k, v, 2, causal_block=1)
    a = torch.autograd.grad(out.sum(), (q, k, v), retain_graph=True)  # an expanded scalar
    b = torch.autograd.grad(out, (q, k, v), torch.ones_like(out), retain_graph=True)
    c = torch.autograd.grad(out.transpose(0, 2).contiguous().sum(), (q, k, v))
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(a, b, c))
    with pytest.raises(RuntimeError):  # the gradient itself is not differentiable
        out = training.attention(q, k, v, 2)
        torch.autograd.grad(torch.autograd.grad(out.sum(), q, create_graph=True)[0].sum(), q)


def test_one_unused_output_and_the_rotation_alone(lib):
    ops, training, _ = lib
    x, w, qw, kw, cos, sin = _inputs(1, 33, 2, 2)
    q, k = (torch.randn((1, 33, 256), device="cuda").to(BF).requires_grad_() for _ in range(2))
    qr, _ = training.qk_norm_rope(q, k, qw, kw, 1e-6, cos, sin, 2)
    dq, dk = torch.autograd.grad(qr.float().square().sum(), (q, k))
    assert dq.any() and not dk.any()
    qr, kr = training.qk_norm_rope(q, k, None, None, 0.0, cos, sin, 2, norm="none")
    dq, dk = torch.autograd.grad((qr.float() + kr.float()).sum(), (q, k))
    assert torch.equal(dq, dk)


def test_backend_is_differentiable_only_where_asked(lib):
    ops, training, backend = lib
    g = torch.Generator(device="cuda").manual_seed(4)
    q, k, v = (torch.randn((1, n, 512), device="cuda", generator=g).to(BF) for n in (90, 40, 40))
    fn = backend.attention_function("b200-native")
    plain = fn(q, k, v, 4)
    assert torch.equal(plain, ops.attention(q, k, v, 4)) and not plain.requires_grad
    v.requires_grad_()
    out = fn(q, k, v, 4)
    assert out.requires_grad and torch.equal(out, ops.attention_with_lse(q, k, v, 4)[0])
    lse = ops.attention_with_lse(q, k, v.detach(), 4)[1]
    (dv,) = torch.autograd.grad(out.float().sum(), v)
    assert torch.equal(dv, ops.attention_backward(torch.ones_like(out), q, k, v.detach(), out.detach(), lse, 4)[2])
    with torch.no_grad():
        assert torch.equal(fn(q, k, v, 4), plain)


def test_explicit_operators_captured_while_an_eager_graph_lives(lib):
    ops, training, _ = lib
    x, w, qw, kw, cos, sin = _inputs(1, 100, 2, 2)
    q, k, v = (torch.randn((1, 100, 256), device="cuda").to(BF).requires_grad_() for _ in range(3))
    qr, kr = training.qk_norm_rope(q, k, qw, kw, 1e-6, cos, sin, 2)
    eager = training.attention(qr, kr, v, 2)  # its graph stays alive
    dout = torch.randn_like(eager)

    def step():
        a, b = ops.fused_qk_norm_rope(q, k, qw, kw, 1e-6, cos, sin, 2)
        out, lse = ops.attention_with_lse(a, b, v, 2)
        da, db, dv = ops.attention_backward(dout, a, b, v, out, lse, 2)
        return *ops.fused_qk_norm_rope_backward(da, db, q, k, qw, kw, 1e-6, cos, sin, 2), dv

    with torch.no_grad():
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step()
    graph.replay()
    torch.cuda.synchronize()
    want = torch.autograd.grad(eager, (q, k, qw, kw, v), dout)
    for a, b in zip(captured, want):
        assert torch.equal(a.to(b.dtype), b)


def test_another_current_device_or_stream_is_respected(lib):
    """The call runs on the current stream of the tensors' device (this machine has one)."""
    ops, training, _ = lib
    q, k, v = (torch.randn((1, 70, 256), device="cuda:0").to(BF) for _ in range(3))
    want = ops.attention_with_lse(q, k, v, 2)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.attention_with_lse(q, k, v, 2)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
