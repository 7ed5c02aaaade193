"""Refusals of the training-pass operators: the Python checks on CPU tensors and the C entries' own guards (no GPU:
every call here is turned down before the device is touched)."""

import ctypes

import pytest
import torch

from opengenie_b200 import _lib, ltx_ops

BF = torch.bfloat16


def _err(lib):
    return lib.ogx_last_error().decode()


def test_python_surface_refuses_cpu_tensors():
    x = torch.zeros((1, 4, 256), dtype=BF)
    cos = torch.zeros((1, 4, 64))
    with pytest.raises(ValueError, match="qkv_device_or_dtype"):
        ltx_ops.attention_with_lse(x, x, x, 2)
    with pytest.raises(ValueError, match="qkv_device_or_dtype"):
        ltx_ops.attention_backward(x, x, x, x, x, torch.zeros((1, 2, 4)), 2)
    with pytest.raises(ValueError, match="qk_device_or_dtype"):
        ltx_ops.fused_qk_norm_rope(x, x, None, None, 1e-6, cos, cos, 2, norm="none")
    with pytest.raises(ValueError, match="qk_device_or_dtype"):
        ltx_ops.fused_qk_norm_rope_backward(x, x, x, x, None, None, 1e-6, cos, cos, 2, norm="none")
    with pytest.raises(ValueError, match="norm"):
        ltx_ops.fused_qk_norm_rope(x, x, None, None, 1e-6, cos, cos, 2, norm="layer")


# ogx_attention_fwd_lse arguments by name, a call that every guard accepts up to the tensor maps
FWD = dict(q=16, k=16, v=16, batch=1, q_tokens=8, kv_tokens=8, heads=4, kv_heads=2, head_dim=128, q_stride_b=4096,
           q_stride_t=512, k_stride_b=2048, k_stride_t=256, v_stride_b=2048, v_stride_t=256, scale=0.1, causal_block=0, q_lengths=None, kv_lengths=None,
           out=16, out_stride_b=4096, out_stride_t=512, lse=16, workspace=None, workspace_bytes=0, stream=None)


@pytest.mark.parametrize("change,reason", [
    (dict(q=None), "null_pointer"), (dict(head_dim=64), "head_dim"), (dict(q_tokens=0), "shape"),
    (dict(kv_tokens=0), "shape"), (dict(kv_tokens=(1 << 29) + 1), "shape"), (dict(heads=65536, kv_heads=1), "shape"),
    (dict(kv_heads=3), "kv_heads"), (dict(causal_block=-1), "causal_block"), (dict(scale=0.0), "softmax_scale"),
    (dict(scale=-1.0), "softmax_scale"), (dict(scale=float("nan")), "softmax_scale"),
    (dict(scale=float("inf")), "softmax_scale"), (dict(q_stride_t=511), "stride"), (dict(q_stride_t=504), "stride"),
    (dict(k_stride_t=248), "stride"), (dict(v_stride_t=248), "stride"), (dict(q_stride_b=-8), "stride"), (dict(q_stride_t=1 << 38), "stride"),
    (dict(k=8), "alignment"), (dict(out=None), "output"), (dict(out=24), "output"), (dict(out_stride_t=256), "output"),
    (dict(lse=None), "lse"), (dict(lse=18), "lse"), (dict(kv_lengths=18), "lengths"),
], ids=str)
def test_attention_entry_refusals(ogx_lib, change, reason):
    assert ogx_lib.ogx_attention_fwd_lse(*{**FWD, **change}.values()) == -1
    assert _err(ogx_lib).split(":")[0] == reason


BWD = dict(dout=16, q=16, k=16, v=16, out=16, lse=16, batch=1, q_tokens=8, kv_tokens=8, heads=4, kv_heads=2,
           head_dim=128, dout_stride_b=4096, dout_stride_t=512, q_stride_b=4096, q_stride_t=512, k_stride_b=2048,
           k_stride_t=256, v_stride_b=2048, v_stride_t=256, out_stride_b=4096, out_stride_t=512, scale=0.1, causal_block=0, q_lengths=None,
           kv_lengths=None, workspace=16, workspace_bytes=1 << 40, dq=16, dq_stride_b=4096, dq_stride_t=512, dk=16,
           dk_stride_b=2048, dk_stride_t=256, dv=16, dv_stride_b=2048, dv_stride_t=256, stream=None)


@pytest.mark.parametrize("change,reason", [
    (dict(v=None), "null_pointer"), (dict(dout=None), "dout_or_out"), (dict(out=8), "dout_or_out"),
    (dict(dout_stride_t=256), "dout_or_out"), (dict(lse=None), "lse"), (dict(dq=None), "gradients"),
    (dict(dk=8), "gradients"), (dict(dk_stride_t=128), "gradients"), (dict(dv_stride_t=128), "gradients"), (dict(workspace=None), "workspace"),
    (dict(workspace_bytes=15), "workspace"), (dict(workspace=8), "workspace"), (dict(scale=0.0), "softmax_scale"),
    (dict(q_lengths=2), "lengths"),
], ids=str)
def test_attention_gradient_entry_refusals(ogx_lib, change, reason):
    assert ogx_lib.ogx_attention_bwd(*{**BWD, **change}.values()) == -1
    assert _err(ogx_lib).split(":")[0] == reason


def test_few_queries_over_many_keys_need_a_workspace(ogx_lib):
    n = ctypes.c_int64(-1)
    assert ogx_lib.ogx_attention_fwd_lse_workspace(4, 9216, 9216, 32, 32, ctypes.addressof(n)) == 0 and n.value == 0
    assert ogx_lib.ogx_attention_fwd_lse_workspace(1, 1, 20000, 4, 4, ctypes.addressof(n)) == 0 and n.value > 0
    call = {**FWD, "q_tokens": 1, "kv_tokens": 20000, "workspace": 16, "workspace_bytes": n.value - 1}
    assert ogx_lib.ogx_attention_fwd_lse(*call.values()) == -1 and _err(ogx_lib) == "workspace"
    assert ogx_lib.ogx_attention_fwd_lse_workspace(1, 0, 20000, 4, 4, ctypes.addressof(n)) == -1
    assert ogx_lib.ogx_attention_fwd_lse_workspace(1, 1, 20000, 4, 3, ctypes.addressof(n)) == -1
    assert ogx_lib.ogx_attention_fwd_lse_workspace(1, 1, (1 << 25) + 1, 4, 4, ctypes.addressof(n)) == -1
    assert ogx_lib.ogx_attention_bwd_workspace(1, 1 << 62, 1, 4, 4, ctypes.addressof(n)) == -1
    assert ogx_lib.ogx_attention_fwd_lse_workspace(1, 1, 20000, 4, 4, None) == -1


def test_attention_gradient_workspace_size(ogx_lib):
    n = ctypes.c_int64(0)
    assert ogx_lib.ogx_attention_bwd_workspace(2, 129, 5, 4, 2, ctypes.addressof(n)) == 0
    assert n.value >= 2 * 4 * 129 * 8
    call = {**BWD, "batch": 2, "q_tokens": 129, "kv_tokens": 5, "workspace_bytes": n.value - 1}
    assert ogx_lib.ogx_attention_bwd(*call.values()) == -1 and _err(ogx_lib) == "workspace"
    assert ogx_lib.ogx_attention_bwd_workspace(0, 129, 5, 4, 2, ctypes.addressof(n)) == -1
    assert ogx_lib.ogx_attention_bwd_workspace(2, 129, 5, 4, 2, None) == -1


NORM = dict(q=16, k=16, batch=1, tokens=3, heads=4, kv_heads=2, head_dim=128, q_stride_b=1536, q_stride_t=512,
            k_stride_b=768, k_stride_t=256, q_weight=16, k_weight=16, weight_dtype=0, norm=1, eps=1e-6, cos=16, sin=16,
            cs_dtype=1, rotary=128, interleaved=0, cs_stride_b=0, cs_stride_h=0, cs_stride_t=64)
NORM_OUT = dict(q_out=16, q_out_stride_b=1536, q_out_stride_t=512, k_out=16, k_out_stride_b=768, k_out_stride_t=256)
NORM_REFUSALS = [
    (dict(k=None), "null_pointer"), (dict(head_dim=96), "head_dim"), (dict(tokens=0), "qk_shape"),
    (dict(heads=127, kv_heads=2), "qk_shape"), (dict(q_stride_t=508), "qk_noncontiguous"), (dict(norm=3), "norm"),
    (dict(q_weight=None), "qk_weight_shape"), (dict(weight_dtype=2), "qk_weight_shape"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(cos=None), "rope_shape"), (dict(cs_dtype=2), "rope_shape"),
    (dict(rotary=8), "rope_shape"), (dict(rotary=144), "rope_shape"), (dict(rotary=40), "rope_shape"),
    (dict(cs_stride_t=60), "rope_shape"), (dict(cs_stride_h=64), "rope_shape"), (dict(q=8), "alignment"),
    (dict(sin=8), "alignment"),
]


@pytest.mark.parametrize("change,reason", NORM_REFUSALS + [(dict(q_out=None), "output"), (dict(k_out=8), "output"),
                                                           (dict(k_out_stride_t=4), "output")], ids=str)
def test_norm_rotation_entry_refusals(ogx_lib, change, reason):
    assert ogx_lib.ogx_qk_norm_rope(*{**NORM, **NORM_OUT, **change}.values(), None) == -1
    assert _err(ogx_lib).split(":")[0] == reason


@pytest.mark.parametrize("change,reason", NORM_REFUSALS + [
    (dict(dq_out=None), "output_gradients"), (dict(dk_out_stride_b=4), "output_gradients"), (dict(q_out=None), "output"),
    (dict(dk_weight=None), "weight_gradients"), (dict(workspace=None), "workspace"), (dict(workspace_bytes=8), "workspace"),
], ids=str)
def test_norm_rotation_gradient_entry_refusals(ogx_lib, change, reason):
    grads = dict(dq_out=16, dq_out_stride_b=1536, dq_out_stride_t=512, dk_out=16, dk_out_stride_b=768,
                 dk_out_stride_t=256)
    rest = dict(dq_weight=16, dk_weight=16, workspace=16, workspace_bytes=1 << 40, stream=None)
    call = {**grads, **NORM, **NORM_OUT, **rest, **change}
    assert ogx_lib.ogx_qk_norm_rope_bwd(*call.values()) == -1
    assert _err(ogx_lib).split(":")[0] == reason


def test_refused_calls_leave_python_errors():
    with pytest.raises(_lib.OgxError, match="null_pointer"):
        _lib.call("ogx_attention_fwd_lse", *{**FWD, "q": None}.values())


def test_packed_calls_reach_the_entry_points(ogx_lib):
    """The packed form hands every argument on: each refusal of the plain form comes back from it."""
    for name, base, change, reason in [
        ("ogx_attention_fwd_lse", FWD, dict(scale=-1.0), "softmax_scale"),
        ("ogx_attention_fwd_lse", FWD, dict(lse=None), "lse"),
        ("ogx_attention_bwd", BWD, dict(dv=None), "gradients"),
        ("ogx_attention_bwd", BWD, dict(workspace_bytes=1), "workspace"),
    ]:
        with pytest.raises(_lib.OgxError, match=reason):
            _lib.call_packed(name, *(0 if v is None else v for v in {**base, **change}.values()))
    slots = (ctypes.c_int64 * 64)()
    for entry, at, count in ((0, slots, 5), (4, slots, 29), (-1, slots, 29), (0, None, 29)):
        assert ogx_lib.ogx_call_packed(entry, at, count) == -1
