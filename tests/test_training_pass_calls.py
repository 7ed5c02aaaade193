"""How the training-pass operators reach the library (no GPU): the device and the stream of a call."""

import contextlib
import ctypes

import pytest
import torch

from opengenie_b200 import ltx_ops


@pytest.mark.parametrize("current,index", [(0, 0), (0, 1), (1, 0)])
def test_a_call_runs_on_the_tensors_device_and_its_current_stream(monkeypatch, current, index):
    now = [current]
    entered = []

    @contextlib.contextmanager
    def device(i):
        before, now[0] = now[0], i
        entered.append(i)
        yield
        now[0] = before

    calls = []
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: now[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 100 + i, raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(ltx_ops._lib, "call_packed", lambda name, *args: calls.append((now[0], name, args)))
    ltx_ops._call_on(torch.device("cuda", index), "entry", 1, 2)
    assert calls == [(index, "entry", (1, 2, 100 + index))] and now == [current]
    assert entered == ([] if current == index else [index])


def test_workspace_sizes_are_kept_for_each_device(monkeypatch):
    asked = []
    now = [0]

    @contextlib.contextmanager
    def device(i):
        now[0] = i
        yield

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(ltx_ops._lib, "call", lambda name, *args: asked.append((now[0], name, args[:-1])))
    ltx_ops._workspace_bytes.cache_clear()
    for index in (0, 1, 0, 1):
        ltx_ops._workspace_bytes("entry", index, 3, 4)
    ltx_ops._workspace_bytes.cache_clear()
    assert asked == [(0, "entry", (3, 4)), (1, "entry", (3, 4))]


@pytest.mark.parametrize("batch,tokens", [(1, (1 << 30) + 1), (1 << 16, 1 << 15), (1 << 40, 1 << 40), ((1 << 30) + 1, 1)])
def test_workspace_query_refuses_sizes_that_the_call_refuses(ogx_lib, batch, tokens):
    size = ctypes.c_int64(-1)
    assert ogx_lib.ogx_qk_norm_rope_bwd_workspace(batch, tokens, 4, 2, 128, 1, ctypes.addressof(size)) == -1
    assert ogx_lib.ogx_last_error().decode().split(":")[0] == "qk_shape" and size.value == -1


@pytest.mark.gpu
def test_tensors_on_another_device_than_the_current_one(ogx_lib):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    q, k, v, dout = (torch.randn((1, 70, 256), device="cuda:1").to(torch.bfloat16) for _ in range(4))
    angle = torch.rand((1, 70, 64), device="cuda:1")

    def step():
        a, b = ltx_ops.fused_qk_norm_rope(q, k, None, None, 0.0, angle.cos(), angle.sin(), 2, norm="none")
        out, lse = ltx_ops.attention_with_lse(a, b, v, 2)
        grads = ltx_ops.attention_backward(dout, a, b, v, out, lse, 2)
        return out, lse, *grads, *ltx_ops.fused_qk_norm_rope_backward(
            *grads[:2], q, k, None, None, 0.0, angle.cos(), angle.sin(), 2, norm="none")[:2]

    with torch.cuda.device(1):
        want = step()
        torch.cuda.synchronize()
    with torch.cuda.device(0):
        got = step()
        assert torch.cuda.current_device() == 0
    torch.cuda.synchronize(1)
    assert all(a.device.index == 1 and torch.equal(a, b) for a, b in zip(got, want))
