"""Attention with statistics and its gradients on the GPU where inputs hold what a formula in exact numbers never meets:
rows that no mask lets in, values that are not finite, and the longest rows."""

import math

import pytest
import torch

from gpu_util import status_clean

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
D = 128


@pytest.fixture(scope="module")
def ops(ogx_lib):
    from opengenie_b200 import ltx_ops

    return ltx_ops


def _randn(seed, *shapes):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(s, device="cuda", generator=g).to(BF) for s in shapes]


def _int32(x):
    return None if x is None else torch.tensor(x, device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("B,L,M,heads,kv_heads,block,ql,kl", [
    (1, 300, 200, 2, 1, 7, None, None),
    (1, 257, 129, 2, 2, 1, None, None),  # a whole tile of them
    (2, 200, 70, 4, 2, 3, (200, 150), (70, 66)),  # rows without keys and rows past the length in one tile
    (2, 100, 40, 2, 2, 1, (55, 100), None),  # a clip that ends before its first row with a key
    (3, 700, 333, 4, 1, 100, (700, 650, 3), (333, 1, 0)),
    (1, 4000, 20, 4, 1, 1, (3990,), None),  # sums shared by several CTAs
    (2, 5001, 130, 2, 2, 7, None, (130, 64)),
], ids=str)
def test_rows_that_causality_leaves_without_keys_may_hold_anything(ops, B, L, M, heads, kv_heads, block, ql, kl):
    """The sequences end together, so with more queries than keys the first L - L_kv rows see no key.  They give nothing
    to dk and dv, whatever they hold: the results equal those of rows of zeros bit for bit."""
    q, dout, k, v = _randn(L + M, (B, L, heads * D), (B, L, heads * D), (B, M, kv_heads * D), (B, M, kv_heads * D))
    args = dict(kv_heads=kv_heads, causal_block=block, q_lengths=_int32(ql), kv_lengths=_int32(kl))
    blind = L - M
    results = []
    for a, b in ((0.0, 0.0), (math.nan, math.inf), (math.inf, math.nan)):
        q[:, :blind], dout[:, :blind] = a, b
        out, lse = ops.attention_with_lse(q, k, v, heads, **args)
        assert not out[:, :blind].any() and (lse[..., :blind] == -math.inf).all()
        results.append((out, lse, *ops.attention_backward(dout, q, k, v, out, lse, heads, **args)))
        assert status_clean() and not results[-1][2][:, :blind].any()
    for got in results[1:]:
        for x, y in zip(got, results[0]):
            assert torch.equal(x, y)


FORMS = [
    # B, L, L_kv, heads, kv_heads, causal_block: one and two Q tiles per CTA, packed heads, shared key sums
    (1, 90, 200, 2, 2, 0),
    (2, 300, 300, 2, 1, 1),
    (1, 1, 5000, 8, 2, 0),
    (1, 1300, 700, 32, 32, 0),
    (1, 1100, 1100, 32, 8, 100),
]


def _sees(L, M, block, key):
    """The rows that see `key`."""
    i = torch.arange(L, device="cuda")
    return key // block <= torch.div(i + M - L, block, rounding_mode="floor") if block else i >= 0


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("key", [5, 50, 63, 64 + 49, -1])
def test_a_score_that_is_nan_or_infinite_reaches_every_row_that_sees_it(ops, form, bad, key):
    """softmax of a row with a NaN or +inf score is NaN in every column (inf - inf), and the log of its sum NaN or +inf,
    wherever the key lies in its tile; rows that do not see the key are as they were, bit for bit."""
    B, L, M, heads, kv_heads, block = form
    q, k, v = _randn(M + key, (B, L, heads * D), (B, M, kv_heads * D), (B, M, kv_heads * D))
    q[..., ::D] = q[..., ::D].abs() + 0.5  # column 0 of each head: a positive times +inf
    args = dict(kv_heads=kv_heads, causal_block=block)
    out, lse = ops.attention_with_lse(q, k, v, heads, **args)
    assert torch.isfinite(lse).logical_or(lse == -math.inf).all() and torch.isfinite(out).all()
    k[0, key, ::D] = bad
    got, got_lse = ops.attention_with_lse(q, k, v, heads, **args)
    assert status_clean()
    hit = torch.zeros((B, L), dtype=torch.bool, device="cuda")
    hit[0] = _sees(L, M, block, key % M)
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], out[~hit])
    rows = hit[:, None].expand_as(lse)
    assert (torch.isnan(got_lse[rows]) if math.isnan(bad) else got_lse[rows] == math.inf).all()
    assert torch.equal(got_lse[~rows], lse[~rows])


@pytest.mark.parametrize("form", FORMS, ids=str)
def test_scores_of_minus_infinity_weigh_nothing(ops, form):
    """A first tile and more of scores of -inf: the other keys are what counts.  A row of nothing else is 0 / 0."""
    B, L, M, heads, kv_heads, block = form
    q, k, v = _randn(M, (B, L, heads * D), (B, M, kv_heads * D), (B, M, kv_heads * D))
    q[..., ::D] = q[..., ::D].abs() + 0.5
    k[:, :130, ::D] = -math.inf
    out, lse = ops.attention_with_lse(q, k, v, heads, kv_heads=kv_heads, causal_block=block)
    assert status_clean()
    sees = torch.stack([_sees(L, M, block, j) for j in range(M)], -1)
    one = lambda x, h: x.double().unflatten(-1, (-1, D))[..., h, :]  # noqa: E731
    for h in range(heads):
        s = one(q, h) @ one(k, h * kv_heads // heads).transpose(-1, -2) * D ** -0.5
        s = s.masked_fill(~sees, -math.inf)
        p, values = torch.softmax(s, -1), one(v, h * kv_heads // heads)
        none = ~(s > -math.inf).any(-1)
        blind = ~sees.any(-1).expand_as(none)
        assert torch.isnan(one(out, h)[none & ~blind]).all() and not one(out, h)[blind].any()
        # P and the output are rounded to bf16 once each (2^-8 at most), and an eighth of it for the rest
        tol = 2.0 ** -8 * 9 / 8 * ((p @ values).abs() + p @ values.abs())
        assert ((one(out, h) - p @ values).abs() <= tol)[~none].all()
        want = torch.logsumexp(s, -1)
        assert torch.equal(lse[:, h] == -math.inf, none)
        assert ((lse[:, h].double() - want).abs() <= 2.0 ** -12)[~none].all()


@pytest.mark.parametrize("L,M", [(200, 200), (40, 700), (4000, 40), (1000, 300)])
@pytest.mark.parametrize("at", [3, 27, 31])
def test_values_that_are_not_finite_reach_the_gradients(ops, L, M, at):
    """What one row or key that is NaN makes of the gradients, by their formulas: a query's NaN reaches its dq and every dk
    and dv, a key's every gradient, a value's dq and dk (dv = P^T dout does not read it), an infinite score all but the dv
    of keys whose P = exp(s - inf) is 0.  The other batch and head keep their bits."""
    heads = 2
    clean = _randn(L + M, (2, L, heads * D), (2, M, heads * D), (2, M, heads * D), (2, L, heads * D))
    clean[0][..., ::D] = clean[0][..., ::D].abs() + 0.5

    def gradients(q, k, v, dout):
        out, lse = ops.attention_with_lse(q, k, v, heads)
        grads = ops.attention_backward(dout, q, k, v, out, lse, heads)
        assert status_clean()
        return grads

    want = gradients(*clean)
    for n, column, value, finite in ((0, slice(D), math.nan, (True, False, False)),
                                     (1, slice(D), math.nan, (False, False, False)),
                                     (2, slice(D), math.nan, (False, False, True)),
                                     (1, slice(1), math.inf, (False, False, None)),
                                     (3, slice(D), math.nan, (True, False, False))):
        given = [t.clone() for t in clean]
        given[n][1, at, column] = value
        for i, (got, ref) in enumerate(zip(gradients(*given), want)):
            assert torch.equal(got[0], ref[0]) and torch.equal(got[1, :, D:], ref[1, :, D:])
            here = got[1, :, :D]
            if finite[i]:  # dq but for the query's own row, or all of dv
                rest = torch.arange(here.shape[0], device="cuda") != at if i == 0 else slice(None)
                assert torch.equal(here[rest], ref[1, :, :D][rest])
                assert i == 2 or torch.isnan(here[at]).all()
            elif finite[i] is None:
                rest = torch.arange(M, device="cuda") != at
                assert torch.isnan(here[at]).all() and here[rest].abs().max() < 1e-30
            else:
                assert torch.isnan(here).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("key", [5, 50, 120, 199])
def test_dense_attention_with_a_score_that_is_nan_or_infinite(ops, bad, key):
    """The dense attention, too: NaN in every row of that head and batch, the others as they were."""
    q, k, v = _randn(key, (2, 300, 2 * D), (2, 200, 2 * D), (2, 200, 2 * D))
    q[..., ::D] = q[..., ::D].abs() + 0.5
    want = ops.attention(q, k, v, 2)
    k[1, key, D] = bad
    got = ops.attention(q, k, v, 2)
    assert status_clean()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1, :, :D], want[1, :, :D])
    assert torch.isnan(got[1, :, D:]).all()


def test_rows_of_the_largest_length(ops):
    """2^25 keys, the most that is taken, with enough queries that no row's sum is shared out: some warps wait for the
    whole of it.  Equal scores: P = 1, the sum 2^25 and the mean of the values, which are 1 or -1 by turns of 64 keys and
    3 at one key in 1024."""
    n, rows = 1 << 25, 148 * 256
    if torch.cuda.mem_get_info()[0] < 3 * n * D * 2:
        pytest.skip("not enough free memory")
    q = torch.zeros((1, rows, D), device="cuda", dtype=BF)
    k = torch.zeros((1, n, D), device="cuda", dtype=BF)
    v = torch.ones((1, n, D), device="cuda", dtype=BF)
    v.view(1, n // 128, 2, 64, D)[:, :, 1] = -1
    v.view(1, n // 1024, 1024, D)[:, :, 5] = 3  # 1 before
    from opengenie_b200 import _lib

    assert ops._workspace_bytes("ogx_attention_fwd_lse_workspace", 0, 1, rows, n, 1, 1) == 0
    lengths = torch.tensor([n - 3], device="cuda", dtype=torch.int32)  # and a last tile with rows to zero
    out, lse = ops.attention_with_lse(q, k, v, 1, kv_lengths=lengths)
    assert _lib.device_status() == 0
    # the products' sums are whole numbers below 2^24; the sum of P, 2^19 tiles in 32 bits, is off by 2^19 2^-24 at most
    assert (lse - math.log(n - 3)).abs().max() <= 2.0 ** -5
    mean = (2 * (n / 1024) + 3) / (n - 3)
    assert ((out.double() - mean).abs() <= mean * (2.0 ** -8 + 2.0 ** -5)).all()


@pytest.mark.parametrize("chunk", range(4))
@pytest.mark.parametrize("L,M", [(40, 64), (1300, 64), (40, 5000)])
def test_statistics_of_short_rows_are_as_exact_as_32_bits(ops, chunk, L, M):
    """Rows whose weight lies in one chunk of 16 keys, one of which has its exponentials from a polynomial (off by 2.7e-6 at
    most; hardware's by 2^-22).  The scores are exact: small whole numbers and a scale of 1/8.  Scaling, the maximum and
    the logarithm round values of up to (1 + |lse|) log2(e) four times, by 2^-24 each."""
    g = torch.Generator(device="cuda").manual_seed(chunk)
    q = torch.zeros((1, L, D), device="cuda", dtype=BF)
    k, v = torch.zeros((1, M, D), device="cuda", dtype=BF), torch.ones((1, M, D), device="cuda", dtype=BF)
    q[..., 1:9] = torch.randint(-2, 3, (1, L, 8), device="cuda", generator=g).to(BF)
    k[..., 1:9] = torch.randint(-2, 3, (1, M, 8), device="cuda", generator=g).to(BF)
    q[..., 0], k[..., 0] = 1, -2000  # the other keys' weight is e^-250
    k[:, 16 * chunk:16 * chunk + 16, 0] = 0
    _, lse = ops.attention_with_lse(q, k, v, 1, softmax_scale=0.125)
    want = torch.logsumexp(q.double() @ k.double().transpose(-1, -2) * 0.125, -1)
    assert ((lse[:, 0].double() - want).abs() <= 2.7e-6 + 4 * 1.45 * 2.0 ** -24 * (1 + want.abs())).all()
