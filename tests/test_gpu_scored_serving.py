"""Scored attention, token weights, eviction and logit controls together, as a serving loop uses them: every attention call,
every eviction and every pick of a run is held against its own definition in 64 bits, from what the call itself was given."""
import types

import pytest
import torch

from conftest import load_golden
from oracle import attn_oracle as orc
from test_gpu_evict import plain as plain_eviction
from test_gpu_logit_controls import definition
from test_gpu_scored_attention import check_rows, score_error

pytestmark = pytest.mark.gpu

U_P = {torch.bfloat16: 2.0**-8, torch.float32: 0.0}  # (extend's; decode's bf16 is finer)


def tiny_model(dev, dtype, cap=None, slopes=None):
    import baby_sglang_amd as pkg

    g = load_golden("tiny_model")
    cfg = types.SimpleNamespace(**g["config"], tie_word_embeddings=False, hidden_act="silu", rope_scaling=None, attn_logit_softcapping=cap,
                                distance_slopes=slopes)
    model = pkg.BabyQwen2ForCausalLM(cfg).eval()
    model.load_state_dict(g["state_dict"], strict=True)
    return model.to(dtype).to(dev)


def held_attention(monkeypatch, counts):
    """SimpleAttentionBackend.forward, each call checked after it ran."""
    from baby_sglang_amd.attn_backend import SimpleAttentionBackend as backend

    real = backend.forward

    def forward(q, k, v, layer, fb, save_kv_cache=True):
        table, weights = fb.req_to_token_pool.req_to_token.cpu(), fb.token_weights
        before = weights.double().cpu() if weights is not None else None
        out = real(q, k, v, layer, fb, save_kv_cache)
        ks, vs = (t.cpu() for t in fb.token_to_kv_pool.get_kv_buffer(layer.layer_id))
        req, lens = fb.req_pool_indices.tolist(), fb.seq_lens.tolist()
        if fb.is_prefill:
            ext, pre = fb.extended_lens.tolist(), fb.prefix_lens.tolist()
            row_req = [i for i, n in enumerate(ext) for _ in range(n)]
            row_pos = [p + j for n, p in zip(ext, pre) for j in range(n)]
        else:
            row_req, row_pos = list(range(len(req))), [n - 1 for n in lens]
        opt = [None if t is None else t.cpu() for t in (layer.distance_slopes, fb.visible_from, fb.visible_to)]
        q3 = q.cpu().view(len(row_req), -1, layer.head_dim)
        want, mass, lse, received, top = orc.scored_exact(q3, ks, vs, table[req], lens, row_req, row_pos, layer.head_dim**-0.5, layer.logit_cap, *opt)
        check_rows(out, want, mass, lse, top, layer.logit_cap, q.dtype, q.dtype, U_P[q.dtype], max(lens), vs.float().abs().max().item(), layer.head_dim)
        if weights is not None and not fb.is_prefill:
            after = weights.double().cpu()
            ds = score_error(top, layer.logit_cap, lse, layer.head_dim)
            for i, (r, n) in enumerate(zip(req, lens)):
                slack = received[i] * (4 * ds[i].max() + 2.0**-20 + n * 2.0**-23)
                expect = before[r, :n] + received[i]
                assert bool(((after[r, :n] - expect).abs() <= slack + 2.0**-23 * expect).all())
                assert torch.equal(after[r, n:], before[r, n:])
                counts["weights"] += 1
        counts["prefill" if fb.is_prefill else "decode"] += 1
        return out

    monkeypatch.setattr(backend, "forward", staticmethod(forward))


def held_pool(pool, counts):
    real = pool.evict_tokens

    def evict(rows, lens, budget, recent=0, sinks=0, max_seq_len=0):
        table, weights = pool.req_to_token.cpu(), pool.token_weights.cpu()
        n = lens.tolist()
        want_t, want_w = table.clone(), weights.clone()
        want_lens, want_gone = plain_eviction(table, weights, rows.cpu(), n, budget, recent, sinks, max(n) - budget, want_t, want_w)
        new_lens, gone = real(rows, lens, budget, recent, sinks, max_seq_len)
        assert torch.equal(new_lens.cpu(), want_lens) and torch.equal(gone.cpu(), want_gone)
        for i, r in enumerate(rows.tolist()):
            assert torch.equal(pool.req_to_token[r, : want_lens[i]].cpu(), want_t[r, : want_lens[i]])
            assert torch.equal(pool.token_weights[r, : want_lens[i]].cpu(), want_w[r, : want_lens[i]])
        counts["evict"] += 1
        return new_lens, gone

    pool.evict_tokens = evict


def held_picks(loop, sp, allowed_now, counts):
    """The ids picked (greedy) against the definition over the tokens each request has produced."""
    real = loop._pick

    def pick(logits, batch):
        ids = real(logits, batch)
        n = len(batch)
        past = [list(s.output_ids) for s in batch]
        history = torch.zeros((n, max(1, max(map(len, past)))), dtype=torch.int32)
        for i, t in enumerate(past):
            history[i, : len(t)] = torch.tensor(t, dtype=torch.int32)
        keys = sorted(sp.logit_bias or {})
        bias = torch.tensor([keys] * n, dtype=torch.int32), torch.tensor([[sp.logit_bias[t] for t in keys]] * n) if keys else None
        x, slack = definition(logits.cpu(), history, None, [len(t) for t in past], None, [sp.repetition_penalty] * n, [sp.presence_penalty] * n,
                              [sp.frequency_penalty] * n, bias[0] if keys else None, bias[1], None, None)
        for i, s in enumerate(batch):
            allowed = allowed_now(s)
            x[i, ~allowed] = float("-inf")
            got = int(ids[i])
            assert bool(allowed[got])
            u = torch.finfo(logits.dtype).eps / 2
            best = x[i].max()
            # (both may be off by the bound, and round to the logits' type)
            assert best - x[i, got] <= 2 * slack[i].max() + 2 * u * best.abs().clamp(min=x[i, got].abs())
            assert len(loop._controls.history) == loop.max_requests
            counts["picks"] += 1
        return ids

    loop._pick = pick


def accounted(loop, total):
    assert loop.req_to_token_pool.available_size() == loop.max_requests
    free = loop.token_to_kv_pool.free_slots.tolist()
    assert len(set(free)) == len(free)
    assert len(free) + loop.tree_cache.evictable_size() == total


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("chunk", [None, 7])
def test_everything_together(gpu, monkeypatch, dtype, chunk):
    """Capped and biased attention, a cache budget, penalties, biases and a mask that changes with every token; five prompts
    over three page-table rows, twice (the second run finds the prompts in the prefix tree)."""
    from baby_sglang_amd import sampling as smp
    from baby_sglang_amd.serving_loop import ServingLoop

    model = tiny_model(gpu, dtype, cap=20.0, slopes=[0.25, 0.0625])
    prompts = load_golden("driver_traces")["tiny_model_e2e"]["prompts"]
    sp = smp.SamplingParams(max_new_tokens=40, repetition_penalty=1.1, presence_penalty=0.4, frequency_penalty=0.2, logit_bias={5: 1.5, 56: -2.0, 63: -float("inf")})
    loop = ServingLoop(model, max_total_tokens=384, max_requests=3, chunked_prefill_size=chunk, kv_budget=24, kv_recent=6, kv_sinks=2, kv_slack=5)

    def allowed_now(s):  # a grammar of two states: even ids, then odd ones
        return torch.arange(64) % 2 == len(s.output_ids) % 2

    loop.token_mask_fn = lambda batch: smp.pack_token_mask(torch.stack([allowed_now(s) for s in batch]))
    counts = dict(prefill=0, decode=0, weights=0, evict=0, picks=0)
    held_attention(monkeypatch, counts)
    held_pool(loop.req_to_token_pool, counts)
    held_picks(loop, sp, allowed_now, counts)
    seen = []
    loop.on_batch = lambda mode, fb: seen.append((mode, fb.positions.tolist(), fb.seq_lens.tolist()))
    for again in range(2):
        outs = loop.run_batch(prompts, sp)
        assert all(len(o) == 40 for o in outs)
        assert all(t % 2 == j % 2 for o in outs for j, t in enumerate(o))
        accounted(loop, 384)
    assert min(counts.values()) > 0 and counts["evict"] >= 10
    decodes = [(p, n) for mode, p, n in seen if mode == "decode"]
    assert max(max(n) for _, n in decodes) == 29  # budget + slack, and no more
    assert max(max(p) for p, _ in decodes) == 16 + 40 - 2  # the true position of the longest request's last fed token


def test_budget_that_is_never_reached_changes_nothing(gpu):
    """The plain loop's ids (fp32), its page tables and its prefix tree; the weights are there all the same."""
    from baby_sglang_amd.serving_loop import SamplingParams, ServingLoop

    e2e = load_golden("driver_traces")["tiny_model_e2e"]
    loop = ServingLoop(tiny_model(gpu, torch.float32), max_total_tokens=e2e["max_total_tokens"], max_requests=e2e["max_requests"], kv_budget=50)
    sp = SamplingParams(max_new_tokens=e2e["max_new_tokens"], eos_id=e2e["eos_id"])
    assert [list(o) for o in loop.run_batch(e2e["prompts"], sp)] == [o.tolist() for o in e2e["output_ids"]]
    assert loop.req_to_token_pool.token_weights.max() > 0
    assert int(loop.tree_cache.evictable_size()) > sum(len(p) for p in e2e["prompts"]) - 4 * 10
    accounted(loop, e2e["max_total_tokens"])


def test_budget_lets_a_request_outgrow_its_page_table_row(gpu):
    """32 columns a row, 90 tokens produced; and a pool that sends requests back to the queue."""
    from baby_sglang_amd.serving_loop import SamplingParams, ServingLoop

    model = tiny_model(gpu, torch.float32)
    prompts = load_golden("driver_traces")["tiny_model_e2e"]["prompts"]
    loop = ServingLoop(model, max_total_tokens=96, max_requests=3, kv_budget=24, kv_slack=4)
    outs = loop.run_batch(prompts, SamplingParams(max_new_tokens=90))
    assert all(len(o) == 90 for o in outs)
    accounted(loop, 96)


def test_prompt_longer_than_the_budget(gpu):
    from baby_sglang_amd.serving_loop import SamplingParams, ServingLoop

    model = tiny_model(gpu, torch.float32)
    prompt = torch.randint(0, 64, (50,), generator=torch.Generator().manual_seed(2))
    loop = ServingLoop(model, max_total_tokens=256, max_requests=2, kv_budget=1, kv_recent=1, kv_sinks=0, kv_slack=1)
    lens = []
    loop.on_batch = lambda mode, fb: lens.append(fb.seq_lens.tolist())
    (out,) = loop.run_batch([prompt], SamplingParams(max_new_tokens=6))
    assert len(out) == 6 and lens == [[50], [51], [2], [2], [2], [2]]
    accounted(loop, 256)


def test_penalties_alone_and_sampling(gpu):
    """Draws stay inside the mask; a repetition penalty alone goes the old way and gives the same ids as among the controls."""
    from baby_sglang_amd.serving_loop import SamplingParams, ServingLoop

    model = tiny_model(gpu, torch.float32)
    prompts = load_golden("driver_traces")["tiny_model_e2e"]["prompts"]
    run = lambda **kw: ServingLoop(model, max_total_tokens=384, max_requests=3).run_batch(prompts, SamplingParams(max_new_tokens=12, **kw))  # noqa: E731
    assert run(repetition_penalty=1.3) == run(repetition_penalty=1.3, logit_bias={0: 0.0})
    assert run() != run(frequency_penalty=2.0)
    drawn = run(do_sample=True, allowed_token_ids=[3, 31, 32, 63], temperature=3.0)
    assert {t for o in drawn for t in o} <= {3, 31, 32, 63}


def test_controls_that_leave_nothing_are_refused(gpu):
    from baby_sglang_amd import sampling as smp
    from baby_sglang_amd.serving_loop import ServingLoop

    loop = ServingLoop(tiny_model(gpu, torch.float32), max_total_tokens=384, max_requests=3)
    prompt = [torch.tensor([1, 2, 3])]
    with pytest.raises(ValueError, match="no token"):
        loop.run_batch(prompt, smp.SamplingParams(do_sample=True, allowed_token_ids=[5], logit_bias={5: -float("inf")}))
    for bad in (dict(allowed_token_ids=[]), dict(allowed_token_ids=[64]), dict(logit_bias={64: 1.0}), dict(logit_bias={-1: 1.0})):
        with pytest.raises(ValueError):
            loop.run_batch(prompt, smp.SamplingParams(**bad))
    loop.token_mask_fn = lambda batch: torch.ones((len(batch), 64), dtype=torch.bool)
    with pytest.raises(ValueError, match="int32"):
        loop.run_batch(prompt)
    for kw in (dict(frequency_penalty=0.5), dict(allowed_token_ids=[1])):
        with pytest.raises(NotImplementedError):
            loop.run_batch_overlap(prompt, smp.SamplingParams(**kw))
    with pytest.raises(NotImplementedError):
        ServingLoop(tiny_model(gpu, torch.float32), max_total_tokens=384, max_requests=3, kv_budget=8).run_batch_overlap(prompt)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cap,slopes", [(None, None), (15.0, None), (None, [0.5, 0.125])])
def test_model_with_windows(gpu, monkeypatch, dtype, cap, slopes):
    """Prefill and decode batches with intervals of their own through the model: a window, a document's start, a prefix that
    all its tokens see, and a row that sees nothing."""
    import baby_sglang_amd as pkg

    model = tiny_model(gpu, dtype, cap, slopes)
    lens, pre = [20, 9, 1, 30], [0, 4, 0, 12]
    pool = pkg.ReqToTokenPool(5, 40, str(gpu))
    kv = pkg.MHATokenToKVPool(128, dtype, 1, 64, 2, str(gpu))
    rows = torch.tensor([3, 0, 4, 1], device=gpu)
    slots = (torch.randperm(100, generator=torch.Generator().manual_seed(1)) + 1).to(torch.int32)
    at = 0
    for r, n in zip(rows.tolist(), lens):
        pool.req_to_token[r, : n + 1] = slots[at : at + n + 1].to(gpu)
        at += n + 1
    counts = dict(prefill=0, decode=0, weights=0)
    held_attention(monkeypatch, counts)
    # the prefixes first, as calls of their own
    for part, (first, last) in enumerate(((None, pre), (pre, lens))):
        live = [i for i in range(4) if last[i] > (first[i] if first else 0)]
        starts = [first[i] if first else 0 for i in live]
        pos = [p for i, s in zip(live, starts) for p in range(s, last[i])]
        loc = torch.cat([pool.req_to_token[rows[i], s : last[i]] for i, s in zip(live, starts)])
        ids = torch.randint(0, 64, (len(pos),), device=gpu)
        fb = pkg.SimplifiedForwardBatch.create_prefill_batch(
            input_ids=ids, req_pool_indices=rows[live], seq_lens=torch.tensor([last[i] for i in live], device=gpu), out_cache_loc=loc,
            req_to_token_pool=pool, token_to_kv_pool=kv, prefix_lens=torch.tensor(starts, device=gpu))
        if part:
            fb.visible_from = torch.tensor([max(0, p - 6) for p in pos], dtype=torch.int32, device=gpu)
            fb.visible_to = torch.tensor([max(p + 1, 8) if j != 3 else 0 for j, p in enumerate(pos)], dtype=torch.int32, device=gpu)
        with torch.no_grad():
            model(ids, fb.positions, fb)
    seq = torch.tensor([n + 1 for n in lens], device=gpu)
    ids = torch.randint(0, 64, (4,), device=gpu)
    fb = pkg.SimplifiedForwardBatch.create_decode_batch(
        input_ids=ids, req_pool_indices=rows, seq_lens=seq, out_cache_loc=pool.req_to_token[rows, seq - 1], req_to_token_pool=pool, token_to_kv_pool=kv)
    fb.visible_from = torch.tensor([15, 0, 2, 30], dtype=torch.int32, device=gpu)
    fb.token_weights = pool.enable_token_weights()
    with torch.no_grad():
        model(ids, fb.positions, fb)
    assert counts == dict(prefill=4, decode=2, weights=8)


def test_slopes_stay_in_32_bits_and_out_of_the_state(gpu):
    model = tiny_model(gpu, torch.bfloat16, slopes=[0.3, 0.1])
    attn = model.model.layers[0].self_attn.attn
    assert attn.distance_slopes.dtype == torch.float32 and attn.distance_slopes.device.type == "cuda"
    assert torch.equal(attn.distance_slopes.cpu(), torch.tensor([0.3, 0.1]))
    assert not any("slopes" in k for k in model.state_dict())


def test_prompts_as_long_as_their_row(gpu):
    """32 columns a row: a prompt of 31 leaves room for the next token and is then cut; one of 32 runs where nothing follows it."""
    from baby_sglang_amd.serving_loop import SamplingParams, ServingLoop

    loop = ServingLoop(tiny_model(gpu, torch.float32), max_total_tokens=64, max_requests=2, kv_budget=8, kv_slack=2)
    lens = []
    loop.on_batch = lambda mode, fb: lens.append(fb.seq_lens.tolist())
    prompt = torch.randint(0, 64, (32,), generator=torch.Generator().manual_seed(3))
    (out,) = loop.run_batch([prompt[:31]], SamplingParams(max_new_tokens=5))
    assert len(out) == 5 and lens == [[31], [32], [9], [10], [9]]
    (out,) = loop.run_batch([prompt], SamplingParams(max_new_tokens=1))
    assert len(out) == 1
    with pytest.raises(ValueError, match="row of 32"):
        loop.run_batch([prompt], SamplingParams(max_new_tokens=2))
    accounted(loop, 64)


@pytest.mark.parametrize("chunk", [None, 9])
def test_budget_gives_the_slots_of_long_prompts_back(gpu, chunk):
    """Prompts of four times the budget: once they have been cut, the pool holds what the requests hold, N + slack each, and the tree
    nothing of them; a prompt within the budget is in the tree as ever, and a long one may begin with it."""
    from baby_sglang_amd.serving_loop import SamplingParams, ServingLoop

    model = tiny_model(gpu, torch.float32)
    g = torch.Generator().manual_seed(4)
    short = torch.randint(0, 64, (10,), generator=g)
    prompts = [torch.randint(0, 64, (50,), generator=g), torch.cat((short, torch.randint(0, 64, (40,), generator=g)))]
    loop = ServingLoop(model, max_total_tokens=192, max_requests=3, chunked_prefill_size=chunk, kv_budget=12, kv_slack=4)
    loop.run_batch([short], SamplingParams(max_new_tokens=3))
    in_tree = int(loop.tree_cache.evictable_size())
    assert in_tree >= 10
    held = []
    loop.on_batch = lambda mode, fb: held.append((mode, 192 - loop.token_to_kv_pool.available_size(), fb.seq_lens.tolist()))
    outs = loop.run_batch(prompts, SamplingParams(max_new_tokens=30))
    assert [len(o) for o in outs] == [30, 30]
    for mode, used, lens in held[-20:]:
        assert mode == "decode" and max(lens) <= 16
        assert used <= in_tree + 2 * 16, (used, lens)
    accounted(loop, 192)
    assert int(loop.tree_cache.evictable_size()) == in_tree
    loop.run_batch([short], SamplingParams(max_new_tokens=3))  # (what the tree had is still right)
    accounted(loop, 192)
