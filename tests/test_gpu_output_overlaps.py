"""Outputs that share buffers with inputs: what is apart gives the results of separate tensors, updates in place too, and
the rest is refused before anything runs."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
D = 128


@pytest.fixture(scope="module")
def ops(ogx_lib):
    from opengenie_b200 import ltx_ops

    return ltx_ops


def _randn(seed, *shape):
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(BF)


def _same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


def _buffer(layout, B, L, W):
    """[B, L, W] of NaN in a larger buffer: contiguous, batches interleaved, or rows and batches with padding."""
    if layout == "interleaved":
        return torch.full((L, B, W + 8), float("nan"), device="cuda", dtype=BF).transpose(0, 1)[..., :W]
    if layout == "padded":
        return torch.full((B * (L * (W + 8) + 24),), float("nan"), device="cuda", dtype=BF).as_strided(
            (B, L, W), (L * (W + 8) + 24, W + 8, 1))
    return torch.full((B, L, W), float("nan"), device="cuda", dtype=BF)


@pytest.mark.parametrize("layout", ["contiguous", "interleaved", "padded"])
def test_attention_and_its_gradients_within_one_buffer(ops, layout):
    B, L, heads = 2, 150, 2
    C = heads * D
    x = _randn(1, B, L, 4 * C)
    plain = [t.contiguous() for t in x.split(C, -1)]
    q, k, v, dout = plain
    out, lse = ops.attention_with_lse(q, k, v, heads, causal_block=1)
    grads = ops.attention_backward(dout, q, k, v, out, lse, heads, causal_block=1)
    # columns: inputs, output and gradients side by side
    buf = _buffer(layout, B, L, 8 * C)
    parts = buf.split(C, -1)
    buf[..., :4 * C] = x
    a, b = ops.attention_with_lse(*parts[:3], heads, causal_block=1, out=parts[4])
    assert torch.equal(a, out) and torch.equal(b, lse)
    got = ops.attention_backward(parts[3], *parts[:3], parts[4], b, heads, causal_block=1, grads=parts[5:])
    assert _same(got, grads) and torch.equal(buf[..., :4 * C], x) and torch.equal(parts[4], out)
    # in place over q's columns
    a, _ = ops.attention_with_lse(*parts[:3], heads, causal_block=1, out=parts[0])
    assert torch.equal(a, out) and torch.equal(buf[..., C:4 * C], x[..., C:])


@pytest.mark.parametrize("layout", ["contiguous", "padded"])
def test_attention_over_other_tokens_of_one_buffer(ops, layout):
    B, L, heads = 2, 150, 2
    q, k, v = (_randn(s, B, L, heads * D) for s in (1, 2, 3))
    out, lse = ops.attention_with_lse(q, k, v, heads)
    buf = _buffer(layout, B, 2 * L, heads * D)
    buf[:, L:] = k
    got, got_lse = ops.attention_with_lse(q, buf[:, L:], v, heads, out=buf[:, :L])
    assert torch.equal(got, out) and torch.equal(got_lse, lse) and torch.equal(buf[:, L:], k)


def test_attention_refuses_outputs_over_inputs(ops):
    B, L, heads = 1, 200, 2
    C = heads * D
    rows = _randn(4, B, L, 3 * C + 64)
    keep = rows.clone()
    q, k, v = rows[..., :C], rows[..., C:2 * C], rows[..., 2 * C:3 * C]
    dout = _randn(5, B, L, C)
    out, lse = ops.attention_with_lse(q, k, v, heads)
    packed = rows.flatten()[:L * C].view(B, L, C)  # q's address, other strides
    tokens = _randn(6, B, 2 * L, C)
    for bad in (rows[..., 8:8 + C], rows[..., C + 8:2 * C + 8], rows[..., D:D + C], packed):
        with pytest.raises(ValueError, match="out_alias"):
            ops.attention_with_lse(q, k, v, heads, out=bad)
    with pytest.raises(ValueError, match="out_alias"):
        ops.attention_with_lse(tokens[:, :L], k, v, heads, out=tokens[:, 1:L + 1])
    fine = [torch.empty_like(out) for _ in range(3)]
    for i in range(3):
        for bad in (rows[..., 8:8 + C], rows[..., C + D:2 * C + D], packed, dout, out):
            with pytest.raises(ValueError, match="grads_alias"):
                ops.attention_backward(dout, q, k, v, out, lse, heads, grads=[*fine[:i], bad, *fine[i + 1:]])
    with pytest.raises(ValueError, match="grads_alias"):
        ops.attention_backward(dout, q, k, v, out, lse, heads, grads=(tokens[:, :L], tokens[:, L - 1:2 * L - 1], fine[2]))
    torch.cuda.synchronize()
    assert torch.equal(rows, keep)


@pytest.mark.parametrize("norm", ["head", "row", "none"])
@pytest.mark.parametrize("layout", ["contiguous", "interleaved", "padded"])
def test_norm_rotation_within_one_buffer(ops, norm, layout):
    B, L, heads, kv = 2, 150, 4, 2
    C, K = heads * D, kv * D
    x = _randn(1, B, L, 2 * (C + K))
    q, k, dq, dk = (t.contiguous() for t in x.split([C, K, C, K], -1))
    wide = {"head": (D, D), "row": (C, K), "none": None}[norm]
    w = [1 + 0.1 * _randn(2, n).float() for n in wide] if wide else [None, None]
    angle = torch.rand((1, L, 64), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) * 6.0
    rest = (*w, 1e-6, angle.cos(), angle.sin(), heads)
    args = dict(kv_heads=kv, norm=norm, interleaved=True)
    want = ops.fused_qk_norm_rope(q, k, *rest, **args)
    grads = ops.fused_qk_norm_rope_backward(dq, dk, q, k, *rest, **args)

    def fill():
        buf = _buffer(layout, B, L, 3 * (C + K))
        buf[..., :2 * (C + K)] = x
        return buf, buf.split([C, K, C, K, C, K], -1)

    buf, p = fill()
    assert _same(ops.fused_qk_norm_rope(p[0], p[1], *rest, out=(p[4], p[5]), **args), want)
    got = ops.fused_qk_norm_rope_backward(p[2], p[3], p[0], p[1], *rest, out=(p[4], p[5]), **args)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(got, grads))
    assert torch.equal(buf[..., :2 * (C + K)], x)
    # in place: over the inputs, and over the inputs' gradients or the inputs in the gradient
    for into in ((0, 1), (2, 3), (0, 3)):
        buf, p = fill()
        got = ops.fused_qk_norm_rope_backward(p[2], p[3], p[0], p[1], *rest, out=(p[into[0]], p[into[1]]), **args)
        assert all(a is b is None or torch.equal(a, b) for a, b in zip(got, grads))
    buf, p = fill()
    assert _same(ops.fused_qk_norm_rope(p[0], p[1], *rest, out=(p[0], p[1]), **args), want)
    assert torch.equal(buf[..., C + K:2 * (C + K)], x[..., C + K:])


def test_norm_rotation_refuses_outputs_over_other_tensors(ops):
    B, L, heads = 1, 100, 2
    q, k, dq, dk = (_randn(s, B, L, heads * D) for s in range(4))
    keep = [t.clone() for t in (q, k, dq, dk)]
    angle = torch.rand((1, L, 64), device="cuda")
    rest = (torch.ones(D, device="cuda"), torch.ones(D, device="cuda"), 1e-6, angle.cos(), angle.sin(), heads)
    new = torch.empty_like(q)
    two = _randn(5, B, 2 * L, heads * D)
    for bad in ((k, q), (new, new), (new, q), (k, new), (two[:, :L], two[:, 1:L + 1])):
        with pytest.raises(ValueError, match="out_alias"):
            ops.fused_qk_norm_rope(q, k, *rest, out=bad)
    with pytest.raises(ValueError, match="out_alias"):
        ops.fused_qk_norm_rope(two[:, :L], k, *rest, out=(two[:, 1:L + 1], new))
    for bad in ((dk, dq), (k, q), (new, new), (dk, new), (new, q), (new, dq)):
        with pytest.raises(ValueError, match="out_alias"):
            ops.fused_qk_norm_rope_backward(dq, dk, q, k, *rest, out=bad)
    torch.cuda.synchronize()
    assert _same((q, k, dq, dk), keep)
