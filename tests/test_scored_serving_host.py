"""Host side of scored attention and logit controls in the serving loop (CPU)."""
import types

import pytest
import torch

from baby_sglang_amd import sampling as smp


@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 64, 100])
def test_pack_token_mask(vocab):
    allowed = torch.rand(3, vocab, generator=torch.Generator().manual_seed(vocab)) > 0.5
    words = smp.pack_token_mask(allowed)
    assert words.dtype == torch.int32 and words.shape == (3, (vocab + 31) // 32)
    t = torch.arange(vocab)
    assert torch.equal(((words.long() & 0xFFFFFFFF)[:, t // 32] >> (t % 32)) & 1 == 1, allowed)
    assert torch.equal(smp.pack_token_mask(torch.ones(vocab, dtype=torch.bool))[0] & 1, torch.tensor(1, dtype=torch.int32))


def test_controls_are_asked_for_by_the_new_parameters_only():
    assert not smp.SamplingParams(repetition_penalty=1.3, do_sample=True, top_k=4).needs_controls()
    for kw in (dict(presence_penalty=0.1), dict(frequency_penalty=-0.1), dict(logit_bias={1: 2.0}), dict(allowed_token_ids=[])):
        assert smp.SamplingParams(**kw).needs_controls()


def test_controls_need_a_gpu():
    with pytest.raises(NotImplementedError):
        smp.LogitControls(smp.SamplingParams(presence_penalty=0.1), 2, 4, 64, torch.device("cpu"))


class _Model(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.w = torch.nn.Parameter(torch.zeros(1))
        self.config = types.SimpleNamespace(num_key_value_heads=1, hidden_size=4, num_attention_heads=1, num_hidden_layers=1, vocab_size=8)


def test_loop_refusals():
    from baby_sglang_amd.serving_loop import ServingLoop

    for kw in (dict(kv_budget=0), dict(kv_budget=4, kv_sinks=-1), dict(kv_budget=4, kv_sinks=2, kv_recent=3), dict(kv_budget=4, kv_recent=-1),
               dict(kv_budget=4, kv_slack=0), dict(kv_budget=8)):
        with pytest.raises(ValueError):
            ServingLoop(_Model(), max_total_tokens=16, max_requests=2, **kw)
    with pytest.raises(NotImplementedError):
        ServingLoop(_Model(), max_total_tokens=16, max_requests=2, kv_budget=4)
    loop = ServingLoop(_Model(), max_total_tokens=16, max_requests=2)
    with pytest.raises(NotImplementedError):
        loop.run_batch([torch.tensor([1])], smp.SamplingParams(presence_penalty=0.5))
    with pytest.raises(NotImplementedError):
        loop.run_batch_overlap([torch.tensor([1])], smp.SamplingParams(presence_penalty=0.5))


def test_attention_shim_checks_its_slopes():
    from baby_sglang_amd.qwen2_hip import BabyRadixAttention

    with pytest.raises(ValueError):
        BabyRadixAttention(4, 64, 0.125, 2, 0, distance_slopes=[0.5, 0.25])
    plain = BabyRadixAttention(4, 64, 0.125, 2, 0)
    assert plain.distance_slopes is None and plain.logit_cap == 0.0 and not plain.state_dict()
    biased = BabyRadixAttention(2, 64, 0.125, 2, 0, logit_cap=30.0, distance_slopes=[0.3, 0.1]).to(torch.bfloat16)
    assert biased.distance_slopes.dtype == torch.float32 and not biased.state_dict()
    assert torch.equal(biased.distance_slopes, torch.tensor([0.3, 0.1]))


def _budget_loop(**kw):
    """A loop on the CPU with a budget's settings put in by hand: what it refuses, it refuses before any model or kernel runs."""
    from baby_sglang_amd.serving_loop import ServingLoop

    loop = ServingLoop(_Model(), max_total_tokens=64, max_requests=2)
    loop.kv_budget, loop.kv_recent, loop.kv_sinks, loop.kv_slack = 8, 2, 1, 2
    for k, v in kw.items():
        setattr(loop, k, v)
    return loop


def test_budget_refuses_prompts_that_fill_their_row():
    """A row has 32 columns: the next token of a prompt of 32 would stand in column 32, in the row behind it."""
    loop = _budget_loop()
    for n, new in ((32, 2), (33, 1), (33, 5)):
        with pytest.raises(ValueError, match="request 1"):
            loop.run_batch([torch.tensor([1, 2]), torch.arange(n) % 8], smp.SamplingParams(max_new_tokens=new))
        assert not loop.waiting and loop.req_to_token_pool.available_size() == 2


def test_a_full_row_is_told_on_the_host():
    from baby_sglang_amd.serving_loop import Sequence_, ServingLoop

    loop = ServingLoop(_Model(), max_total_tokens=64, max_requests=2)
    s = Sequence_(input_ids=[1] * 32, max_new_tokens=3, eos_id=-1)
    s.row, s.seq_len, s.table, s.output_ids = 0, 32, list(range(1, 33)), [3]
    with pytest.raises(RuntimeError, match="row of 32"):
        loop._decode_batch([s])
    assert s.seq_len == 32 and len(s.table) == 32 and loop.token_to_kv_pool.available_size() == 64
