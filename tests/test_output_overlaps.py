"""Outputs over memory that is still read: the check of address ranges against sets of addresses, and the refusals of the
training-pass entry points (no GPU: every call here is turned down before the device is touched)."""

import os
import random
import shutil
import subprocess

import pytest

from opengenie_b200 import _lib
from test_attention_grad_guards import BWD, FWD, NORM, NORM_OUT, NORM_REFUSALS

CSRC = os.path.join(os.path.dirname(_lib.__file__), "csrc")

HARNESS = r"""
#include <cstdio>
#include "regions.h"
static bool read(ogx::Region* r) {
  long long base, v[7];
  if (scanf("%lld", &base) != 1) return false;
  for (long long& x : v)
    if (scanf("%lld", &x) != 1) return false;
  *r = ogx::Region{reinterpret_cast<const char*>(base), v[0], {v[1], v[2], v[3]}, {v[4], v[5], v[6]}};
  return true;
}
int main() {
  ogx::Region a, b;
  while (read(&a) && read(&b)) printf("%d %d %d\n", ogx::meet(a, b), ogx::same_region(a, b), ogx::runs_apart(a));
}
"""


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    """pairs of (base, width, counts, strides) -> (meet, same, runs of the first apart)"""
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    at = tmp_path_factory.mktemp("regions")
    (at / "h.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-I", CSRC, "-o", str(at / "h"), str(at / "h.cpp")], check=True)

    def run(pairs):
        text = "\n".join(" ".join(map(str, (base, width, *n, *s))) for pair in pairs for base, width, n, s in pair)
        out = subprocess.run([str(at / "h")], input=text, capture_output=True, text=True, check=True).stdout
        return [tuple(bool(int(x)) for x in line.split()) for line in out.splitlines()]

    return run


def _runs(region):
    base, width, n, s = region
    starts = [base + i * s[0] + j * s[1] + k * s[2] for i in range(n[0]) for j in range(n[1]) for k in range(n[2])]
    return [set(range(x, x + width)) for x in starts]


def _bytes(region):
    return set().union(*_runs(region))


def test_regions_that_are_called_apart_share_no_byte(check):
    rng = random.Random(1)
    pick = lambda: (rng.randint(1000, 1150), rng.randint(1, 12), [rng.choice([1, 1, 2]), rng.randint(1, 4), rng.randint(1, 5)],  # noqa: E731
                    [rng.choice([0, 4, 60, 150]), rng.choice([-20, 0, 6, 8, 24, 48, 100]), rng.choice([-8, 0, 4, 8, 12, 16, 24])])
    pairs = []
    for _ in range(4000):
        a, b = pick(), pick()
        if rng.random() < 0.5:
            b = (b[0], b[1], b[2], a[3])  # the same strides
        pairs.append((a, b))
    apart = 0
    for (a, b), (meets, same, runs) in zip(pairs, check(pairs)):
        shared = bool(_bytes(a) & _bytes(b))
        assert meets or not shared, (a, b)
        apart += not meets
        assert not same or (a[:3] == b[:3] and _bytes(a) == _bytes(b))
        if runs and a[2][0] == 1:  # outputs have two axes
            assert sum(map(len, _runs(a))) == len(_bytes(a)), a
    assert apart > 500


def test_slices_of_one_buffer_are_told_apart_exactly(check):
    """Columns, tokens and batches of one [B, L, W] or [L, B, W] buffer, with padding behind its rows and batches."""
    rng = random.Random(2)
    pairs = []
    for _ in range(3000):
        B, L, W = rng.randint(1, 3), rng.randint(1, 5), rng.choice([8, 12])
        st = W + rng.choice([0, 4])
        sb = L * st + rng.choice([0, 4, 8])
        if rng.random() < 0.4:
            st, sb = B * W + rng.choice([0, 4]), W
        sides = []
        for _ in range(2):
            c0, t0, b0 = rng.randrange(W), rng.randrange(L), rng.randrange(B)
            sides.append((1000 + b0 * sb + t0 * st + c0, rng.randint(1, W - c0), [1, rng.randint(1, B - b0), rng.randint(1, L - t0)],
                          [0, sb, st]))
        pairs.append(tuple(sides))
    for (a, b), (meets, same, runs) in zip(pairs, check(pairs)):
        assert runs
        # slices of other batches and tokens of an interleaved buffer lie in one another: refused, though apart
        interleaved = a[3][1] < a[3][2]
        shared = bool(_bytes(a) & _bytes(b))
        assert meets == shared or (interleaved and meets), (a, b)
        assert same == (a[0] == b[0] and a[1] == b[1] and a[2] == b[2])


def test_strides_past_64_bits_of_reach(check):
    far = (1 << 40, 256, [1, 60000, 1 << 25], [0, 1 << 39, 1 << 39])
    assert check([(far, (1 << 41, 256, [1, 1, 1], [0, 0, 0]))])[0][0]  # one of its runs starts there
    assert not check([(far, ((1 << 40) - 256, 256, [1, 1, 1], [0, 0, 0]))])[0][0]


# the entries' arguments with memory of its own for each: 1 MiB apart
def _own(base, *names):
    return {**base, **{name: (i + 1) << 20 for i, name in enumerate(names)}}


FWD_OWN = _own(FWD, "q", "k", "v", "out", "lse", "q_lengths", "kv_lengths")
BWD_OWN = _own(BWD, "dout", "q", "k", "v", "out", "lse", "q_lengths", "kv_lengths", "dq", "dk", "dv")
BWD_OWN["workspace"] = 1 << 30
QK = {**NORM, **NORM_OUT}
QK_OWN = _own(QK, "q", "k", "q_weight", "k_weight", "cos", "sin", "q_out", "k_out")
GRADS = dict(dq_out=0, dq_out_stride_b=1536, dq_out_stride_t=512, dk_out=0, dk_out_stride_b=768, dk_out_stride_t=256)
TAIL = dict(dq_weight=0, dk_weight=0, workspace=1 << 30, workspace_bytes=1 << 40, stream=None)
QKB_OWN = _own({**GRADS, **QK, **TAIL}, "dq_out", "dk_out", "q", "k", "q_weight", "k_weight", "cos", "sin", "q_out",
               "k_out", "dq_weight", "dk_weight")
MIB = 1 << 20


def _refused(ogx_lib, entry, call, reason):
    """Both forms of the entry turn the call down."""
    assert getattr(ogx_lib, entry)(*call.values()) == -1
    assert ogx_lib.ogx_last_error().decode().split(":")[0] == reason
    with pytest.raises(_lib.OgxArgumentError, match=reason) as raised:
        _lib.call_packed(entry, *(0 if x is None else x for x in call.values()))
    assert isinstance(raised.value, ValueError) and isinstance(raised.value, _lib.OgxError)


@pytest.mark.parametrize("change", [
    dict(out=2 * MIB), dict(out=3 * MIB),  # k, v
    dict(out=2 * MIB + 16), dict(out=2 * MIB - 16), dict(out=3 * MIB + 256),  # eight columns or a head into or before them
    dict(out=1 * MIB, out_stride_t=520), dict(out=1 * MIB + 16), dict(out=1 * MIB + 1024),  # q otherwise than q itself
    dict(out=5 * MIB), dict(lse=2 * MIB + 64), dict(out=6 * MIB), dict(out=7 * MIB - 16),  # lse, lengths
    dict(batch=2, out_stride_b=512), dict(batch=2, out_stride_b=0),  # batches over one another
    dict(batch=2, q_stride_b=8192, out=1 * MIB),  # q with another batch stride
], ids=str)
def test_attention_refuses_overlaps(ogx_lib, change):
    _refused(ogx_lib, "ogx_attention_fwd_lse", {**FWD_OWN, **change}, "out_alias")


@pytest.mark.parametrize("change", [
    *(dict([(g, i * MIB)]) for g in ("dq", "dk", "dv") for i in range(1, 6)),  # dout, q, k, v, out
    *(dict([(g, i * MIB + at)]) for g in ("dq", "dk", "dv") for i in (1, 3) for at in (16, 256, 512, -16)),
    dict(dq=6 * MIB), dict(dk=7 * MIB), dict(dv=8 * MIB),  # lse, lengths
    dict(dk=9 * MIB), dict(dv=10 * MIB + 256), dict(dv=9 * MIB + 7 * 1024),  # one another
    dict(dq=1 << 30), dict(workspace=2 * MIB),
    dict(batch=2, dv_stride_b=256), dict(batch=2, dq_stride_b=0),
], ids=str)
def test_attention_gradients_refuse_overlaps(ogx_lib, change):
    _refused(ogx_lib, "ogx_attention_bwd", {**BWD_OWN, **change}, "grads_alias")


NORM_OVERLAPS = [
    dict(q_out=2 * MIB, k_out=1 * MIB, kv_heads=4, k_stride_t=512, k_out_stride_t=512),  # swapped
    dict(q_out=2 * MIB), dict(k_out=1 * MIB), dict(q_out=1 * MIB + 16), dict(q_out=1 * MIB, q_out_stride_t=520),
    dict(k_out=2 * MIB + 512), dict(q_out=3 * MIB), dict(k_out=4 * MIB), dict(q_out=5 * MIB), dict(k_out=6 * MIB + 16),
    dict(k_out=7 * MIB), dict(k_out=7 * MIB + 1008), dict(q_out_stride_t=504), dict(batch=2, k_out_stride_b=256),
]


@pytest.mark.parametrize("change", NORM_OVERLAPS, ids=str)
def test_norm_rotation_refuses_overlaps(ogx_lib, change):
    _refused(ogx_lib, "ogx_qk_norm_rope", {**QK_OWN, "stream": None, **change}, "out_alias")


@pytest.mark.parametrize("change", [
    dict(q_out=2 * MIB, k_out=1 * MIB, kv_heads=4, k_stride_t=512, k_out_stride_t=512, dk_out_stride_t=512),
    dict(q_out=4 * MIB, k_out=3 * MIB, kv_heads=4, k_stride_t=512, k_out_stride_t=512, dk_out_stride_t=512),
    dict(q_out=1 * MIB + 16), dict(q_out=3 * MIB + 1024), dict(k_out=3 * MIB), dict(k_out=4 * MIB + 512),
    dict(q_out=5 * MIB), dict(k_out=6 * MIB), dict(q_out=7 * MIB), dict(k_out=8 * MIB), dict(k_out=9 * MIB + 512),
    dict(dq_weight=3 * MIB), dict(dk_weight=11 * MIB), dict(dq_weight=9 * MIB), dict(workspace=1 * MIB),
    dict(q_out=1 << 30), dict(k_out_stride_t=248),
], ids=str)
def test_norm_rotation_gradients_refuse_overlaps(ogx_lib, change):
    _refused(ogx_lib, "ogx_qk_norm_rope_bwd", {**QKB_OWN, **change}, "out_alias")


@pytest.mark.parametrize("change,reason", NORM_REFUSALS + [(dict(q_out=None), "output"), (dict(k_out=8), "output")], ids=str)
def test_packed_calls_hand_on_the_norm_rotation_arguments(ogx_lib, change, reason):
    _refused(ogx_lib, "ogx_qk_norm_rope", {**QK_OWN, "stream": None, **change}, reason)
    _refused(ogx_lib, "ogx_qk_norm_rope_bwd", {**QKB_OWN, **change}, reason)


@pytest.mark.parametrize("change,reason", [
    (dict(dq_out=None), "output_gradients"), (dict(dk_out_stride_b=4), "output_gradients"),
    (dict(dk_weight=None), "weight_gradients"), (dict(dq_weight=2), "weight_gradients"), (dict(workspace=None), "workspace"),
    (dict(workspace_bytes=8), "workspace"),
], ids=str)
def test_packed_calls_hand_on_the_gradients_arguments(ogx_lib, change, reason):
    _refused(ogx_lib, "ogx_qk_norm_rope_bwd", {**QKB_OWN, **change}, reason)
