"""GPU parity of the Q/K norm + rotation and its gradients against their formulas in 64 bits.

Tolerances, per element.  y and dx are rounded to bf16 once: at most H = 2^-8 of the value.  Before that everything is
32-bit: the products and the norm's sum are off by less than 2^-20 of the terms that are added, which matters where
they cancel.  The weights' gradients are 32-bit sums; a chain of n additions is off by at most n 2^-24 of the sum of
magnitudes, and no chain here is longer than 512."""

import pytest
import torch

pytestmark = pytest.mark.gpu

H = 2.0 ** -8


@pytest.fixture(scope="module")
def ops(ogx_lib):
    from opengenie_b200 import ltx_ops

    return ltx_ops


def _case(B, L, heads, kv_heads, hd, norm, half, per_head, batched, wdtype, cdtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    q, k = (r(B, L, heads * hd) * 2).to(torch.bfloat16), (r(B, L, kv_heads * hd) * 0.3).to(torch.bfloat16)
    wide = {"head": (hd, hd), "row": (heads * hd, kv_heads * hd), "none": None}[norm]
    w = [(1 + 0.2 * r(n)).to(wdtype) for n in wide] if wide else [None, None]
    lead = (B if batched else 1,) + ((heads,) if per_head else ())
    angle = 6.3 * torch.rand(lead + (L, half), device="cuda", generator=g)
    dq, dk = r(B, L, heads * hd).to(torch.bfloat16), r(B, L, kv_heads * hd).to(torch.bfloat16)
    return q, k, *w, angle.cos().to(cdtype), angle.sin().to(cdtype), dq, dk


def _formula(x, w, cos, sin, heads, norm, interleaved, eps, dy=None):
    """(y, tolerance) or ((dx, tolerance), (dw, tolerance))."""
    hd = x.shape[-1] // heads
    x = x.double().unflatten(-1, (heads, hd))
    cos, sin = (t.double().transpose(1, 2) if t.ndim == 4 else t.double().unsqueeze(2) for t in (cos, sin))
    half = cos.shape[-1]

    def turn(z, sign):
        r, rest = z[..., :2 * half], z[..., 2 * half:]
        a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :half], r[..., half:])
        new = a * cos - sign * b * sin, b * cos + sign * a * sin
        size = a.abs() * cos.abs() + b.abs() * sin.abs(), b.abs() * cos.abs() + a.abs() * sin.abs()
        join = lambda p: torch.stack(p, -1).flatten(-2) if interleaved else torch.cat(p, -1)  # noqa: E731
        return torch.cat((join(new), rest), -1), torch.cat((join(size), rest.abs()), -1)

    r = torch.ones((), device="cuda", dtype=torch.float64)
    over = (-1,) if norm == "head" else (-2, -1)
    wd = torch.ones((), device="cuda", dtype=torch.float64)
    if norm != "none":
        r = torch.rsqrt(x.square().mean(over, keepdim=True) + eps)
        wd = w.double().view(-1, hd)
    if dy is None:
        y, size = turn(x * r * wd, 1)
        return y.flatten(2), (H * y.abs() + 2.0 ** -20 * size).flatten(2)
    g, size = turn(dy.double().unflatten(-1, (heads, hd)), -1)
    if norm == "none":
        return (g.flatten(2), (H * g.abs() + 2.0 ** -20 * size).flatten(2)), None
    dot, dots = (g * wd * x).mean(over, keepdim=True), (size * wd.abs() * x.abs()).mean(over, keepdim=True)
    dx = r * g * wd - x * r ** 3 * dot
    tol = H * dx.abs() + 2.0 ** -20 * (r * size * wd.abs() + x.abs() * r ** 3 * dots)
    at = (0, 1, 2) if norm == "head" else (0, 1)
    dw, tw = (g * x * r).sum(at), 512 * 2.0 ** -24 * (size * x.abs() * r).sum(at)
    return (dx.flatten(2), tol.flatten(2)), (dw.flatten(), tw.flatten())


BF, F32 = torch.bfloat16, torch.float32
CASES = [
    # B, L, heads, kv_heads, hd, norm, half, per_head, batched tables, weights, tables, interleaved
    (1, 1, 1, 1, 128, "head", 64, False, False, BF, F32, False),
    (4, 1, 32, 8, 128, "head", 64, False, True, F32, F32, True),
    (2, 77, 5, 5, 128, "head", 8, True, False, BF, BF, False),
    (1, 300, 16, 1, 64, "head", 32, False, False, F32, BF, False),
    (3, 41, 7, 3, 128, "head", 48, False, True, BF, BF, True),
    (2, 65, 40, 8, 64, "head", 16, False, False, BF, F32, True),
    (1, 513, 32, 32, 128, "row", 64, True, False, BF, BF, False),
    (2, 33, 12, 4, 128, "row", 64, False, True, F32, F32, False),
    (1, 100, 2, 1, 64, "row", 8, False, False, F32, F32, True),
    (1, 19, 64, 64, 128, "row", 32, True, False, BF, F32, True),
    (1, 70, 100, 28, 64, "row", 24, False, False, BF, F32, False),
    (2, 50, 64, 64, 128, "head", 64, True, True, F32, BF, False),
    (2, 130, 6, 2, 128, "none", 40, False, False, BF, F32, False),
    (1, 3, 3, 3, 64, "none", 32, True, False, BF, BF, True),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_forward_and_gradients_against_the_formulas(ops, case):
    B, L, heads, kv_heads, hd, norm, half, per_head, batched, wd, cd, inter = case
    q, k, qw, kw, cos, sin, dq, dk = _case(B, L, heads, kv_heads, hd, norm, half, per_head, batched, wd, cd, seed=L + heads)
    args = dict(kv_heads=kv_heads, norm=norm, interleaved=inter)
    got = ops.fused_qk_norm_rope(q, k, qw, kw, 1e-6, cos, sin, heads, **args)
    for y, x, w, h in zip(got, (q, k), (qw, kw), (heads, kv_heads)):
        ref, tol = _formula(x, w, cos, sin, h, norm, inter, 1e-6)
        assert ((y.double() - ref).abs() <= tol).all()
    grads = ops.fused_qk_norm_rope_backward(dq, dk, q, k, qw, kw, 1e-6, cos, sin, heads, **args)
    for i, (x, dy, w, h) in enumerate(((q, dq, qw, heads), (k, dk, kw, kv_heads))):
        (ref, tol), weight = _formula(x, w, cos, sin, h, norm, inter, 1e-6, dy)
        assert ((grads[i].double() - ref).abs() <= tol).all()
        if weight is None:
            assert grads[2 + i] is None
        else:
            assert grads[2 + i].dtype == torch.float32
            assert ((grads[2 + i].double() - weight[0]).abs() <= weight[1]).all()
    again = ops.fused_qk_norm_rope_backward(dq, dk, q, k, qw, kw, 1e-6, cos, sin, heads, **args)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(grads, again))
    # in place: the outputs over the inputs, the gradients over those of the outputs
    q2, k2, dq2, dk2 = (t.clone() for t in (q, k, dq, dk))
    ops.fused_qk_norm_rope_backward(dq2, dk2, q, k, qw, kw, 1e-6, cos, sin, heads, out=(dq2, dk2), **args)
    ops.fused_qk_norm_rope(q2, k2, qw, kw, 1e-6, cos, sin, heads, out=(q2, k2), **args)
    assert all(torch.equal(a, b) for a, b in zip((q2, k2, dq2, dk2), (*got, *grads[:2])))


def test_row_norm_is_the_video_blocks_norm(ops):
    """norm='row' at the block's width against the block's own op: the same formula, so at most one bf16 step apart."""
    q, k, qw, kw, cos, sin, _, _ = _case(1, 300, 32, 32, 128, "row", 64, True, False, BF, BF, seed=8)
    a = ops.fused_qk_norm_rope(q, k, qw, kw, 1e-6, cos, sin, 32, norm="row")
    b = ops.fused_video_qk_rmsnorm_rope(q, k, qw, kw, 1e-6, cos, sin)
    for x, y in zip(a, b):
        # half a step each around values that differ by 32-bit rounding
        assert ((x.double() - y.double()).abs() <= 2 * H * y.double().abs() + 2.0 ** -18).all()
        assert (x != y).double().mean() < 1e-2


def test_strided_rows_zero_rows_and_guard_columns(ops):
    B, L, heads, kv = 2, 45, 8, 2
    q, k, qw, kw, cos, sin, dq, dk = _case(B, L, heads, kv, 128, "head", 64, False, False, F32, F32, seed=2)
    rows = torch.zeros((B, L, (heads + kv) * 128 + 8), device="cuda", dtype=BF)
    rows[..., 8:8 + heads * 128], rows[..., 8 + heads * 128:] = q, k
    rows[0, 3] = 0  # a row of zeros: eps keeps its inverse norm finite
    qs, ks = rows[..., 8:8 + heads * 128], rows[..., 8 + heads * 128:]
    wide = torch.randn((1, L, 3 * 64 + 8), device="cuda")
    c, s = wide[..., 64:128], wide[..., 128:192]
    got = ops.fused_qk_norm_rope(qs, ks, qw, kw, 1e-6, c, s, heads, kv_heads=kv)
    ref = ops.fused_qk_norm_rope(qs.contiguous(), ks.contiguous(), qw, kw, 1e-6, c.contiguous(), s.contiguous(), heads,
                                 kv_heads=kv)
    assert all(torch.equal(a, b) for a, b in zip(got, ref)) and not got[0][0, 3].any()
    gbuf = torch.full((L, B, (heads + kv) * 128 + 16), 3.0, device="cuda", dtype=BF).transpose(0, 1)
    into = gbuf[..., 8:8 + heads * 128], gbuf[..., 8 + heads * 128:-8]
    grads = ops.fused_qk_norm_rope_backward(dq, dk, qs, ks, qw, kw, 1e-6, c, s, heads, kv_heads=kv, out=into)
    plain = ops.fused_qk_norm_rope_backward(dq, dk, qs.contiguous(), ks.contiguous(), qw, kw, 1e-6, c.contiguous(),
                                            s.contiguous(), heads, kv_heads=kv)
    assert all(torch.equal(a, b) for a, b in zip(grads, plain))
    assert (gbuf[..., :8] == 3).all() and (gbuf[..., -8:] == 3).all()


def test_zero_eps_does_not_leak_from_idle_lanes(ops):
    """Head counts that leave groups of the last token's team without work, and eps = 0."""
    q, k, qw, kw, cos, sin, dq, dk = _case(1, 5, 3, 2, 128, "head", 64, False, False, F32, F32, seed=6)
    for norm, w in (("head", (qw, kw)), ("row", (qw.repeat(3), kw.repeat(2)))):
        grads = ops.fused_qk_norm_rope_backward(dq, dk, q, k, *w, 0.0, cos, sin, 3, kv_heads=2, norm=norm)
        assert all(torch.isfinite(g).all() for g in grads)


def test_captured_in_a_graph_and_on_two_streams(ops):
    sets = [_case(2, 200, 8, 8, 128, "head", 64, False, False, BF, F32, seed=s) for s in (1, 2)]
    step = lambda t: ops.fused_qk_norm_rope_backward(t[6], t[7], t[0], t[1], t[2], t[3], 1e-6, t[4], t[5], 8)  # noqa: E731
    want = [step(t) for t in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], []
    for t in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(t))
        graphs.append(graph)
    for _ in range(3):
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for w, x in zip(want, outs) for a, b in zip(w, x))
