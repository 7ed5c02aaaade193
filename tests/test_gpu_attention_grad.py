"""GPU parity of attention with statistics and of attention's gradients against their formulas in 64 bits, at the
lengths, masks and layouts where they can go wrong.

Tolerances, per element.  A bf16 rounding is off by at most H = 2^-8 of the value.  Forward: P is rounded once before
the product with V and out once after it, so |err| <= H |out| + H sum_j P |v|; the exponential (a quarter of them a
polynomial, 7.5e-5 < 2^-13) and the 32-bit sums add less than H / 8 of the same terms.  Backward, from the given out
and lse: dV as out; dS = P (dP - delta) is rounded once, and its 32-bit sums of 128 products are off by less than
2^-17 of sum |dO| |v|, so |err dq| <= H |dq| + c sum_j (9/8 H |dS| + 2^-15 P sum_d |dO v|) |k|, dk likewise."""

import math

import pytest
import torch

from gpu_util import status_clean

pytestmark = pytest.mark.gpu

H = 2.0 ** -8
D = 128


@pytest.fixture(scope="module")
def ops(ogx_lib):
    from opengenie_b200 import ltx_ops

    return ltx_ops


def _case(B, L, M, heads, kv_heads, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda n, h: (torch.randn((B, n, h * D), device="cuda", generator=g) * scale).to(torch.bfloat16)  # noqa: E731
    return r(L, heads), r(M, kv_heads), r(M, kv_heads), r(L, heads)


def _heads(x, heads, group=1):
    x = x.double().unflatten(-1, (heads, D)).transpose(1, 2)
    return x.repeat_interleave(group, 1) if group > 1 else x


def _see(B, L, M, block, ql, kl):
    i, j = torch.arange(L)[:, None], torch.arange(M)[None]
    see = torch.ones((B, 1, L, M), dtype=torch.bool)
    if block:
        see &= j // block <= torch.div(i + M - L, block, rounding_mode="floor")
    if ql is not None:
        see &= i < torch.tensor(ql).view(B, 1, 1, 1)
    if kl is not None:
        see &= j < torch.tensor(kl).view(B, 1, 1, 1)
    return see.cuda()


def _fold(x):
    return x.transpose(1, 2).flatten(2)


def _formulas(q, k, v, dout, heads, kv_heads, see, out=None, lse=None, c=D ** -0.5):
    """Results and tolerances in 64 bits; masked entries of the inputs are never used."""
    group = heads // kv_heads
    row_ok = see.any(-1, keepdim=True).transpose(1, 2).squeeze(-1)  # [B, L, 1]
    key_ok = see.any(-2).transpose(1, 2)
    clean = lambda x, ok: torch.where(ok, x.double(), torch.zeros((), dtype=torch.float64, device="cuda"))  # noqa: E731
    q, dout = (_heads(clean(x, row_ok), heads) for x in (q, dout))
    k, v = (_heads(clean(x, key_ok), kv_heads, group) for x in (k, v))
    s = (q @ k.transpose(-1, -2) * c).masked_fill(~see, -math.inf)
    ref_lse = torch.logsumexp(s, -1)
    if out is None:
        p = torch.softmax(s, -1).masked_fill(~see, 0.0)
        p = torch.where(torch.isnan(p), 0.0, p)
        o = p @ v
        return _fold(o), H * 9 / 8 * (_fold(o).abs() + _fold(p @ v.abs())), ref_lse
    l64 = lse.double().masked_fill(torch.isinf(lse), 0.0)[..., None]
    p = torch.exp(s - l64)
    delta = (dout * _heads(clean(out, row_ok), heads)).sum(-1, keepdim=True)
    ds = p * (dout @ v.transpose(-1, -2) - delta)
    eds = 9 / 8 * H * ds.abs() + 2.0 ** -15 * p * (dout.abs() @ v.abs().transpose(-1, -2))
    fold = lambda x: _fold(x.unflatten(1, (kv_heads, group)).sum(2))  # noqa: E731
    dq, tq = _fold(c * ds @ k), _fold(c * eds @ k.abs())
    dk, tk = fold(c * ds.transpose(-1, -2) @ q), fold(c * eds.transpose(-1, -2) @ q.abs())
    dv, tv = fold(p.transpose(-1, -2) @ dout), fold(9 / 8 * H * p.transpose(-1, -2) @ dout.abs())
    return [(g, t + 9 / 8 * H * g.abs() + 1e-30) for g, t in ((dq, tq), (dk, tk), (dv, tv))]


def _int32(x):
    return None if x is None else torch.tensor(x, device="cuda", dtype=torch.int32)


CASES = [
    # B, L, L_kv, heads, kv_heads, causal_block, q_lengths, kv_lengths
    (1, 1, 1, 1, 1, 0, None, None),
    (1, 1, 300, 2, 1, 0, None, None),
    (2, 77, 77, 4, 2, 1, None, None),
    (1, 128, 128, 2, 2, 0, None, None),
    (1, 129, 257, 2, 1, 1, None, None),
    (1, 257, 129, 2, 2, 1, None, None),  # the first 128 rows see no key
    (2, 256, 640, 2, 2, 0, None, (640, 65)),
    (3, 300, 200, 2, 1, 7, None, (200, 0, 150)),
    (2, 513, 513, 4, 1, 64, (513, 300), (513, 300)),
    (3, 200, 330, 2, 2, 0, (200, 0, 1), (1, 330, 129)),
    (2, 385, 1100, 2, 1, 100, (128, 385), (1100, 1024)),
    (1, 900, 900, 2, 2, 576, None, None),
    (1, 1300, 64, 2, 2, 0, (1290,), (63,)),
    (1, 64, 1300, 8, 1, 0, None, (1281,)),
    # few tiles on one side: the sums over the other are shared by several CTAs and joined
    (1, 1, 5000, 4, 2, 0, None, None),
    (2, 3, 4000, 2, 1, 1, None, (3900, 70)),
    (2, 130, 3333, 2, 2, 100, (130, 1), (3333, 1000)),
    (1, 4000, 20, 4, 1, 0, (3950,), None),
    (2, 5001, 130, 2, 2, 7, (5001, 3000), (130, 64)),
    (1, 3000, 3000, 1, 1, 1, (2900,), (2950,)),
    # two, four, eight and 128 query heads of a key/value head in a Q tile, and groups that are no power of two
    (3, 1, 700, 8, 2, 1, (1, 0, 1), (700, 64, 0)),
    (2, 65, 190, 8, 1, 3, (64, 65), (190, 129)),
    (1, 130, 130, 4, 2, 1, None, (97,)),
    (2, 3, 300, 128, 1, 0, (3, 2), (300, 1)),
    (1, 129, 140, 12, 2, 5, (127,), None),
    # more query blocks than CTAs at a time, with empty ones among them
    (2, 700, 70, 64, 64, 0, (700, 300), (70, 33)),
    (2, 700, 130, 64, 32, 7, (650, 0), (130, 100)),
    (8, 100, 70, 64, 64, 0, (100, 0, 1, 100, 99, 100, 64, 100), (70, 70, 70, 0, 1, 64, 65, 70)),
    (3, 1025, 1025, 20, 4, 100, (1025, 257, 1000), (1025, 300, 1000)),
]


@pytest.mark.parametrize("poison", [False, True])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_and_gradients_against_the_formulas(ops, case, poison):
    B, L, M, heads, kv_heads, block, ql, kl = case
    q, k, v, dout = _case(B, L, M, heads, kv_heads, seed=L * 7 + M)
    if poison:  # what lies past the lengths may be anything
        for b in range(B):
            for lengths, tensors in ((ql, (q, dout)), (kl, (k, v))):
                for n, t in enumerate(tensors if lengths is not None else ()):
                    t[b, lengths[b]:] = math.nan if n else math.inf
    see = _see(B, L, M, block, ql, kl)
    args = dict(kv_heads=kv_heads, causal_block=block, q_lengths=_int32(ql), kv_lengths=_int32(kl))
    out, lse = ops.attention_with_lse(q, k, v, heads, **args)
    ref, tol, ref_lse = _formulas(q, k, v, dout, heads, kv_heads, see)
    assert status_clean()
    assert torch.equal(torch.isinf(lse), torch.isinf(ref_lse))
    fine = ~torch.isinf(ref_lse)
    assert ((lse.double() - ref_lse)[fine].abs() <= 2.0 ** -12 + 2.0 ** -20 * ref_lse[fine].abs()).all()
    assert ((out.double() - ref).abs() <= tol).all()
    assert not out[~see.any(-1)[:, 0]].any()  # rows that see no key: exactly zero
    if poison and ql is not None:
        out = out.clone()
        for b in range(B):
            out[b, ql[b]:] = math.nan
    grads = ops.attention_backward(dout, q, k, v, out, lse, heads, **args)
    assert status_clean()
    for name, got, (ref, tol) in zip(("dq", "dk", "dv"), grads,
                                     _formulas(q, k, v, dout, heads, kv_heads, see, out, lse)):
        worst = ((got.double() - ref).abs() / tol).max().item()
        assert worst <= 1.0, (name, worst)
    dq, dk, dv = grads
    assert not dq[~see.any(-1)[:, 0]].any()
    hidden = ~see.any(-2)[:, 0]
    assert not dk[hidden].any() and not dv[hidden].any()
    again = ops.attention_backward(dout, q, k, v, out, lse, heads, **args)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))  # one order of summation


def test_single_visible_key_gives_its_value_and_no_score_gradient(ops):
    """A softmax over one key is constant: out is v bit for bit, and dS = P (dO . v - dO . out) cancels up to the
    32-bit sums."""
    q, k, v, dout = _case(2, 40, 1, 2, 2, seed=3)
    out, lse = ops.attention_with_lse(q, k, v, 2)
    assert torch.equal(out, v.expand_as(out))
    dq, dk, dv = ops.attention_backward(dout, q, k, v, out, lse, 2)
    bound = 2.0 ** -15 * (dout.double() * out.double()).abs().unflatten(-1, (2, D)).sum(-1).max() * k.abs().max()
    assert dq.double().abs().max() <= bound and dk.double().abs().max() <= bound * 40


@pytest.mark.parametrize("L,M", [(300, 300), (77, 1024), (1, 1)])
def test_without_masks_the_output_is_the_dense_attention(ops, L, M):
    """The dense kernel's exponentials differ by its polynomial alone (within H / 8 of the same terms), so each is
    within the forward tolerance of the formula and they are within both of each other; most elements are equal."""
    q, k, v, dout = _case(2, L, M, 4, 4, seed=L)
    out, _ = ops.attention_with_lse(q, k, v, 4)
    dense = ops.attention(q, k, v, 4)
    _, tol, _ = _formulas(q, k, v, dout, 4, 4, _see(2, L, M, 0, None, None))
    assert ((out.double() - dense.double()).abs() <= 2 * tol).all()


@pytest.mark.parametrize("scale", [0.05, 4.0])
def test_flat_and_sharp_scores_and_another_softmax_scale(ops, scale):
    q, k, v, dout = _case(1, 200, 200, 2, 2, seed=9, scale=scale)
    see = _see(1, 200, 200, 1, None, None)
    c = 0.1
    out, lse = ops.attention_with_lse(q, k, v, 2, softmax_scale=c, causal_block=1)
    ref, tol, _ = _formulas(q, k, v, dout, 2, 2, see, c=c)
    # the scores' 32-bit sums: 128 products, off by 2^-17 of sum |q k| each, move P by as much
    slack = 2.0 ** -17 * c * (q.double().abs().max() * k.double().abs().max() * D)
    assert ((out.double() - ref).abs() <= tol * (1 + slack / H)).all()
    grads = ops.attention_backward(dout, q, k, v, out, lse, 2, softmax_scale=c, causal_block=1)
    for got, (ref, tol) in zip(grads, _formulas(q, k, v, dout, 2, 2, see, out, lse, c=c)):
        assert ((got.double() - ref).abs() <= tol * (1 + slack / H)).all()


def test_strided_rows_given_outputs_and_expanded_batches(ops):
    """Packed projections in, packed gradients out, keys and values broadcast over the batch."""
    B, L, heads = 2, 333, 4
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = torch.randn((B, L, 3 * heads * D + 8), device="cuda", generator=g).to(torch.bfloat16)
    q, k, v = (rows[..., 8 + i * heads * D:8 + (i + 1) * heads * D] for i in range(3))
    dout = torch.randn((L, B, heads * D), device="cuda", generator=g).to(torch.bfloat16).transpose(0, 1)
    buf = torch.full((L, B, heads * D + 16), 7.0, device="cuda", dtype=torch.bfloat16).transpose(0, 1)
    out, lse = ops.attention_with_lse(q, k, v, heads, causal_block=1, out=buf[..., 8:-8])
    plain = ops.attention_with_lse(q.contiguous(), k.contiguous(), v.contiguous(), heads, causal_block=1)
    assert torch.equal(out, plain[0]) and torch.equal(lse, plain[1])
    assert (buf[..., :8] == 7).all() and (buf[..., -8:] == 7).all()
    packed = torch.full((B, L, 3 * heads * D + 8), 5.0, device="cuda", dtype=torch.bfloat16)
    into = tuple(packed[..., i * heads * D:(i + 1) * heads * D] for i in range(3))
    got = ops.attention_backward(dout, q, k, v, out, lse, heads, causal_block=1, grads=into)
    ref = ops.attention_backward(dout.contiguous(), q.contiguous(), k.contiguous(), v.contiguous(), plain[0], plain[1],
                                 heads, causal_block=1)
    assert all(torch.equal(a, b) for a, b in zip(got, ref)) and (packed[..., -8:] == 5).all()
    k1, v1 = (t[:1].contiguous().expand(B, -1, -1) for t in (k, v))
    a = ops.attention_with_lse(q, k1, v1, heads)
    b = ops.attention_with_lse(q, k1.contiguous(), v1.contiguous(), heads)
    assert torch.equal(a[0], b[0])
    ga = ops.attention_backward(dout, q, k1, v1, a[0], a[1], heads)
    gb = ops.attention_backward(dout, q, k1.contiguous(), v1.contiguous(), b[0], b[1], heads)
    assert all(torch.equal(x, y) for x, y in zip(ga, gb))


def test_outputs_over_inputs(ops):
    q, k, v, dout = _case(1, 300, 300, 2, 2, seed=5)
    want, lse = ops.attention_with_lse(q, k, v, 2)
    grads = [torch.empty_like(q) for _ in range(3)]
    for bad in (k, v):
        with pytest.raises(ValueError, match="out_alias"):
            ops.attention_with_lse(q, k, v, 2, out=bad)
    for i, bad in ((0, q), (1, k), (2, v), (0, dout), (0, want), (1, grads[0])):
        with pytest.raises(ValueError, match="grads_alias"):
            ops.attention_backward(dout, q, k, v, want, lse, 2, grads=[*grads[:i], bad, *grads[i + 1:]])
    over, _ = ops.attention_with_lse(q, k, v, 2, out=q)  # every block reads its own rows before it writes them
    assert over is q and torch.equal(over, want)


def test_two_streams_and_captured_graphs_share_nothing(ops):
    sets = [_case(1, 400, 400, 4, 2, seed=s) for s in (1, 2)]
    step = lambda t: ops.attention_backward(  # noqa: E731
        t[3], t[0], t[1], t[2], *ops.attention_with_lse(t[0], t[1], t[2], 4, kv_heads=2, causal_block=1), 4,
        kv_heads=2, causal_block=1)
    want = [step(t) for t in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for st, t in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(step(t))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for w, x in zip(want, got) for a, b in zip(w, x))
    graphs, outs = [], []
    for t in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(t))
        graphs.append(graph)
    for t in sets:
        t[3].mul_(2)  # dout doubles exactly, and so do the gradients
    for _ in range(3):
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(2 * a, b) for w, x in zip(want, outs) for a, b in zip(w, x))


def test_gradients_against_differences(ops):
    """Directional derivatives of sum(out * dout) by central differences of the 64-bit forward formula."""
    q, k, v, dout = _case(1, 150, 190, 2, 1, seed=5, scale=0.5)
    see = _see(1, 150, 190, 3, None, None)
    out, lse = ops.attention_with_lse(q, k, v, 2, kv_heads=1, causal_block=3)
    grads = ops.attention_backward(dout, q, k, v, out, lse, 2, kv_heads=1, causal_block=3)
    g = torch.Generator(device="cuda").manual_seed(2)
    value = lambda *t: (_formulas(*t, dout, 2, 1, see)[0] * dout.double()).sum()  # noqa: E731
    inputs = [t.double() for t in (q, k, v)]
    exact = _formulas(q, k, v, dout, 2, 1, see, out, lse)
    for n in range(3):
        d = torch.randn(inputs[n].shape, device="cuda", generator=g, dtype=torch.float64)
        e = 1e-4
        moved = [[t + s * e * d if i == n else t for i, t in enumerate(inputs)] for s in (1, -1)]
        slope = (value(*moved[0]) - value(*moved[1])) / (2 * e)
        got = (grads[n].double() * d).sum()
        # each element's tolerance, and delta's error from the rounded out: H |out| |dO| per row through P k or P q
        bound = (exact[n][1] * d.abs()).sum() + H * (out.double() * dout.double()).abs().sum() * d.abs().max()
        assert (got - slope).abs() <= bound
        assert (got - slope).abs() <= 0.02 * slope.abs() + 0.02 * (exact[n][0] * d).square().sum().sqrt()


def test_rows_beyond_32_bit_offsets(ops):
    """Element offsets past 2^31: a token stride of 2^23 elements over 300 rows (a 5 GB buffer read and written in
    place)."""
    L, stride = 300, 1 << 23
    need = ((L - 1) * stride + 3 * D) * 2
    if torch.cuda.mem_get_info()[0] < need + (1 << 30):
        pytest.skip("not enough free memory")
    g = torch.Generator(device="cuda").manual_seed(4)
    flat = torch.empty((need // 2,), device="cuda", dtype=torch.bfloat16)
    rows = flat.as_strided((1, L, 3 * D), (0, stride, 1))
    rows.copy_(torch.randn((1, L, 3 * D), device="cuda", generator=g).to(torch.bfloat16))
    q, k, v = rows.split([D] * 3, -1)
    dout = torch.randn((1, L, D), device="cuda", generator=g).to(torch.bfloat16)
    qc, kc, vc = (t.contiguous() for t in (q, k, v))
    out, lse = ops.attention_with_lse(q, k, v, 1)
    ref, ref_lse = ops.attention_with_lse(qc, kc, vc, 1)
    assert torch.equal(out, ref) and torch.equal(lse, ref_lse)
    want = ops.attention_backward(dout, qc, kc, vc, out, lse, 1)
    got = ops.attention_backward(dout, q, k, v, out, lse, 1)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    grads = rows.split([D] * 3, -1)  # the inputs are copied out: their rows take the gradients
    got = ops.attention_backward(dout, qc, kc, vc, out, lse, 1, grads=grads)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
