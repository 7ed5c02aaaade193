"""The fused branches have no backward pass: they decline where a graph has to run through them, and only there."""

import types

import pytest
import torch

from opengenie_b200 import attention_backend as ab


def _stop(*args, **kwargs):
    raise NotImplementedError("built")


@pytest.fixture
def msa(monkeypatch):
    monkeypatch.setattr(ab._MSA_BLOCKS, "get", _stop)  # a call that does not decline gets as far as the weights
    lin = types.SimpleNamespace()
    attn = types.SimpleNamespace(to_q=lin, to_k=lin, to_v=lin, to_out=[lin], q_norm=types.SimpleNamespace(weight=None),
                                 k_norm=types.SimpleNamespace(weight=None))
    block = types.SimpleNamespace(attn1=attn, scale_shift_table=None)

    def call(vx, timesteps):
        video = types.SimpleNamespace(timesteps=timesteps, positional_embeddings=(None, None))
        return ab.video_msa_branch(block, video, vx)

    return call


@pytest.fixture
def text(monkeypatch):
    monkeypatch.setattr(ab._TEXT_BRANCHES, "get", _stop)
    lin = types.SimpleNamespace()
    attn = types.SimpleNamespace(to_q=lin, to_k=lin, to_v=lin, to_out=[lin], q_norm=types.SimpleNamespace(weight=None),
                                 k_norm=types.SimpleNamespace(weight=None))
    block = types.SimpleNamespace(cross_attention_adaln=True, prompt_scale_shift_table=torch.zeros(2, 4),
                                  scale_shift_table=torch.zeros(9, 4))
    return lambda x, context, timestep, prompt: ab.video_text_cross_attention_branch(block, x, context, attn, timestep,
                                                                                     prompt)


def _given(shapes, wants):
    return [torch.zeros(s).requires_grad_(i == wants) for i, s in enumerate(shapes)]


MSA = [(1, 8, 4096), (1, 8, 9)]
TEXT = [(1, 8, 4096), (1, 5, 4096), (1, 1, 9), (1, 1, 2)]


@pytest.mark.parametrize("wants", range(len(MSA)))
def test_self_attention_branch_declines_where_a_gradient_is_needed(msa, wants):
    before = ab.collect_video_msa_branch_stats()["fallback_reasons"].get("requires_grad", 0)
    assert msa(*_given(MSA, wants)) is None
    assert ab.collect_video_msa_branch_stats()["fallback_reasons"]["requires_grad"] == before + 1


@pytest.mark.parametrize("wants", range(len(TEXT)))
def test_text_branch_declines_where_a_gradient_is_needed(text, wants):
    before = ab.collect_video_text_branch_stats()["fallback_reasons"].get("requires_grad", 0)
    assert text(*_given(TEXT, wants)) is None
    assert ab.collect_video_text_branch_stats()["fallback_reasons"]["requires_grad"] == before + 1


def test_branches_run_where_no_gradient_is_needed(msa, text):
    for call, shapes in ((msa, MSA), (text, TEXT)):
        with pytest.raises(NotImplementedError):  # nothing asks for one
            call(*_given(shapes, -1))
        for mode in (torch.no_grad, torch.inference_mode):
            given = _given(shapes, 0)
            with mode(), pytest.raises(NotImplementedError):
                call(*given)
