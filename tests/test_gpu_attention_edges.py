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
