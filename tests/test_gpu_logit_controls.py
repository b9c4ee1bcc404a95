"""Penalties, biases and token masks on logits against the definition in 64 bits.

Off by at most: x * (1 / rep) (two roundings) or x * rep, freq * n, its subtraction, the presence, the sum of b biases and its
addition, each a rounding of 2^-24 of a magnitude that A = |x| max(rep, 1 / rep) + freq n + pres + sum |bias| bounds:
(6 + b) 2^-24 A, then one rounding to the output's type."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def definition(x, history, rows, lens, prompt, rep, pres, freq, ids, vals, mask, mask_rows):
    x = x.double().clone()
    batch, vocab = x.shape
    mag = x.abs().nan_to_num(posinf=0.0)
    most = 0
    for i in range(batch):
        if history is not None:
            past = [int(t) for t in history[rows[i] if rows is not None else i, : max(0, min(lens[i], history.shape[1]))]]
            for t in set(past):
                if not 0 <= t < vocab:
                    continue
                n = sum(1 for at, u in enumerate(past) if u == t and at >= (prompt[i] if prompt is not None else 0))
                r = float(rep[i]) if rep is not None else 1.0
                p, f = (float(v[i]) if v is not None else 0.0 for v in (pres, freq))
                x[i, t] = (x[i, t] / r if x[i, t] > 0 else x[i, t] * r) - f * n - (p if n else 0.0)
                mag[i, t] = mag[i, t] * max(r, 1 / r) + abs(f) * n + abs(p)
        if ids is not None:
            for t, v in zip(ids[i].tolist(), vals[i].tolist()):
                if 0 <= t < vocab:
                    x[i, t] += v
                    mag[i, t] += abs(v)
                    most = max(most, ids[i].tolist().count(t))
        m = (mask_rows[i] if mask_rows is not None else i) if mask is not None else -1
        if mask is not None and 0 <= m < mask.shape[0]:
            words = mask[m].long() & 0xFFFFFFFF
            t = torch.arange(vocab)
            x[i, ((words[t // 32] >> (t % 32)) & 1) == 0] = float("-inf")
    return x, mag * (6 + most) * 2.0**-24


def check(got, want, slack):
    dtype = got.dtype
    got, lim = got.double().cpu(), torch.finfo(dtype).max
    assert torch.equal(got.isneginf(), want.isneginf() | (want < -lim * (1 + U[dtype])))
    live = ~want.isneginf() & (want.abs() <= lim)
    bound = U[dtype] * want.abs() + slack * (1 + U[dtype]) + (2.0**-25 if dtype == torch.float16 else 1e-40)
    assert bool(((got - want).abs() <= bound)[live].all()), ((got - want).abs() / bound)[live].max()


def case(gpu, batch, vocab, dtype, seed=0, hist=0, prompt=True, bias=0, mask=None, rows=True, row_pad=0, offset=0, in_place=False, id_lo=0, id_hi=None,
         scalars=False, mask_rows=True):
    from baby_sglang_amd import _hip

    g = torch.Generator().manual_seed(seed)
    x = (4 * torch.randn(batch, vocab, generator=g)).to(dtype)
    a = dict(history=None, rows=None, lens=None, prompt=None, rep=None, pres=None, freq=None, ids=None, vals=None, mask=None, mask_rows=None)
    kw = {}
    if hist:
        n_rows = batch + 2
        a["history"] = (torch.rand(n_rows, hist, generator=g) ** 3 * ((id_hi or vocab) - id_lo) + id_lo).to(torch.int32)
        a["rows"] = torch.randperm(n_rows, generator=g)[:batch].tolist() if rows else None
        a["lens"] = [hist if i == 0 else int(torch.randint(0, hist + 1, (1,), generator=g)) for i in range(batch)]
        a["prompt"] = [min(n, int(torch.randint(0, hist + 1, (1,), generator=g))) for n in a["lens"]] if prompt else None
        if scalars:
            a["rep"], a["pres"], a["freq"] = [1.2] * batch, [0.5] * batch, [0.25] * batch
            kw = dict(repetition=torch.tensor(1.2).item(), presence=0.5, frequency=0.25)
            a["rep"] = torch.tensor(a["rep"])
        else:
            a["rep"], a["pres"], a["freq"] = 0.8 + torch.rand(batch, generator=g), torch.randn(batch, generator=g), torch.randn(batch, generator=g)
            kw = dict(repetition=a["rep"].to(gpu), presence=a["pres"].to(gpu), frequency=a["freq"].to(gpu))
        kw.update(history=a["history"].to(gpu), history_lens=torch.tensor(a["lens"], device=gpu))
        if rows:
            kw["history_rows"] = torch.tensor(a["rows"], device=gpu)
        if prompt:
            kw["prompt_lens"] = torch.tensor(a["prompt"], device=gpu)
    if bias:
        a["ids"] = torch.randint(-2, vocab + 2, (batch, bias), generator=g, dtype=torch.int32)
        a["ids"][:, : bias // 3] = a["ids"][:, :1]  # the same id many times
        a["vals"] = torch.randn(batch, bias, generator=g)
        kw.update(bias_ids=a["ids"].to(gpu), bias_values=a["vals"].to(gpu))
    if mask is not None:
        bits = torch.rand(batch, (vocab + 31) // 32, 32, generator=g) < mask
        words = (bits.long() << torch.arange(32)).sum(-1)
        a["mask"] = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
        kw["token_mask"] = a["mask"].to(gpu)
        if mask_rows:
            a["mask_rows"] = [int(torch.randint(-1, batch + 1, (1,), generator=g)) for _ in range(batch)]
            kw["mask_rows"] = torch.tensor(a["mask_rows"], dtype=torch.int32, device=gpu)
    base = torch.zeros(batch * (vocab + row_pad) + offset, dtype=dtype, device=gpu)
    d = base[offset:].view(batch, vocab + row_pad)[:, :vocab]
    d.copy_(x)
    got = _hip.logit_controls(d, out=d if in_place else None, **kw)
    torch.cuda.synchronize()
    want, slack = definition(x, **a)
    check(got, want, slack)
    if not in_place:
        assert torch.equal(d.cpu(), x)
    if row_pad:
        assert not bool(base[offset:].view(batch, vocab + row_pad)[:, vocab:].any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 31, 33, 1000, 4096, 4097, 9001, 16384])
def test_vocabularies_and_types(gpu, vocab, dtype):
    case(gpu, 3, vocab, dtype, seed=vocab, hist=37, bias=9, mask=0.5)


@pytest.mark.parametrize("kw", [dict(hist=1), dict(hist=300, prompt=False), dict(hist=2049, rows=False), dict(bias=1), dict(bias=300), dict(bias=700), dict(mask=0.01),
                                dict(mask=0.0, mask_rows=False), dict(mask=1.0), dict(), dict(hist=500, bias=300, mask=0.9), dict(hist=64, scalars=True),
                                dict(hist=64, id_lo=-50, id_hi=9000), dict(hist=257, id_hi=1), dict(hist=70, row_pad=8), dict(hist=70, row_pad=3, bias=5),
                                dict(hist=70, offset=1, mask=0.5), dict(hist=70, in_place=True, bias=5, mask=0.5), dict(hist=70, offset=1, in_place=True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_parts_and_layouts(gpu, kw, dtype):
    case(gpu, 5, 8200, dtype, seed=3, **kw)


def test_the_whole_vocabulary(gpu):
    case(gpu, 4, 151936, torch.bfloat16, seed=4, hist=400, bias=40, mask=0.3)


def test_agrees_with_the_torch_penalty(gpu):
    """The loop's repetition penalty, which is pinned to the reference's, bit for bit in f32."""
    from baby_sglang_amd import _hip
    from baby_sglang_amd.sampling import apply_repetition_penalty_

    x = 3 * torch.randn(6, 5000, device=gpu)
    hist = torch.randint(0, 5000, (6, 90), dtype=torch.int32)
    lens = [90, 0, 1, 45, 89, 90]
    want = apply_repetition_penalty_(x.clone(), [h[:n].tolist() for h, n in zip(hist, lens)], 1.3)
    got = _hip.logit_controls(x, history=hist.to(gpu), history_lens=torch.tensor(lens, device=gpu), repetition=1.3)
    # x * (1 / 1.3) is two roundings of half a step, 2^-24, torch's quotient one, and 1.3 itself is rounded once on either side
    assert bool(((got - want).abs() <= 5 * 2.0**-24 * want.abs()).all())
    assert torch.equal(got == x, want == x)


def test_special_values(gpu):
    from baby_sglang_amd import _hip

    x = torch.tensor([[float("nan"), float("inf"), float("-inf"), torch.finfo(torch.float32).min, 0.0, -0.0, 1.0, -1.0]], device=gpu)
    h = torch.arange(8, dtype=torch.int32, device=gpu)[None].contiguous()
    got = _hip.logit_controls(x, history=h, history_lens=torch.tensor([8], device=gpu), repetition=2.0)
    assert bool(got[0, 0].isnan()) and got[0, 1:].tolist() == [float("inf"), float("-inf"), float("-inf"), 0.0, 0.0, 0.5, -2.0]
    allowed = torch.tensor([[0b11111100]], dtype=torch.int32, device=gpu)
    got = _hip.logit_controls(x, token_mask=allowed)
    assert got[0, :3].tolist() == [float("-inf")] * 3 and got[0, 6].item() == 1.0  # masked NaN and inf do not come through


def test_same_result_every_time_and_in_a_graph(gpu):
    from baby_sglang_amd import _hip

    g = torch.Generator().manual_seed(5)
    x = torch.randn(8, 20000, generator=g).to(gpu)
    kw = dict(history=torch.randint(0, 50, (8, 3000), generator=g, dtype=torch.int32).to(gpu), history_lens=torch.full((8,), 3000, device=gpu),
              repetition=torch.full((8,), 1.1, device=gpu), frequency=torch.full((8,), 0.01, device=gpu),
              bias_ids=torch.randint(0, 9, (8, 500), generator=g, dtype=torch.int32).to(gpu), bias_values=torch.randn(8, 500, generator=g).to(gpu))
    first = _hip.logit_controls(x, **kw)
    out = torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _hip.logit_controls(x, out=out, **kw)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _hip.logit_controls(x, out=out, **kw)
    for i in range(4):
        out.zero_()
        eager = _hip.logit_controls(x, **kw)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        if i == 0:
            assert torch.equal(out, first)
        x.mul_(1.25)


def test_random(gpu):
    r = random.Random(2)
    for seed in range(30):
        case(gpu, r.randint(1, 7), r.choice([5, 100, 4095, 4100, 12345]), r.choice([torch.bfloat16, torch.float16, torch.float32]), seed=seed,
             hist=r.choice([0, 3, 200, 1030]), bias=r.choice([0, 2, 260]), mask=r.choice([None, 0.1, 0.9]), in_place=r.random() < 0.5,
             row_pad=r.choice([0, 0, 1, 8]), prompt=r.random() < 0.5)


def test_refusals(gpu):
    from baby_sglang_amd import _hip

    x = torch.zeros(2, 64, device=gpu)
    h, n = torch.zeros(2, 4, dtype=torch.int32, device=gpu), torch.tensor([1, 2], device=gpu)
    m = torch.zeros(2, 2, dtype=torch.int32, device=gpu)
    for kw in [dict(history=h), dict(history_lens=n), dict(repetition=1.2), dict(history=h.long(), history_lens=n), dict(history=h, history_lens=n[:1]),
               dict(history=h[:1], history_lens=n), dict(history=h, history_lens=n, repetition=torch.ones(3, device=gpu)),
               dict(bias_ids=h), dict(bias_ids=h, bias_values=torch.zeros(2, 3, device=gpu)), dict(bias_ids=h, bias_values=torch.zeros(2, 4, device=gpu).double()),
               dict(token_mask=m[:, :1]), dict(token_mask=m[:1]), dict(mask_rows=n), dict(token_mask=m.long()), dict(out=torch.zeros(2, 63, device=gpu)),
               dict(out=x.half())]:
        with pytest.raises(ValueError):
            _hip.logit_controls(x, **kw)
    with pytest.raises(ValueError):
        _hip.logit_controls(x.t())
    with pytest.raises(NotImplementedError):
        _hip.logit_controls(x.double())
    with pytest.raises(RuntimeError):
        _hip.logit_controls(x.cpu())
    assert _hip.logit_controls(x[:0]).shape == (0, 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinite_penalties_touch_produced_tokens_only(gpu, dtype):
    """A penalty of inf forbids what was produced; the prompt's tokens and biased ones stay numbers."""
    from baby_sglang_amd import _hip

    x = torch.ones(1, 64, dtype=dtype, device=gpu)
    h = torch.tensor([[3, 4, 5]], dtype=torch.int32, device=gpu)
    ids, vals = torch.tensor([[9]], dtype=torch.int32, device=gpu), torch.tensor([[2.0]], device=gpu)
    inf = float("inf")
    for kw in (dict(frequency=inf), dict(presence=inf)):
        got = _hip.logit_controls(x, history=h, history_lens=torch.tensor([3], device=gpu), prompt_lens=torch.tensor([2], device=gpu), bias_ids=ids,
                                  bias_values=vals, **kw)[0]
        want = torch.ones(64)
        want[5], want[9] = -inf, 3.0
        assert torch.equal(got.float().cpu(), want)


def test_as_many_biases_as_are_taken(gpu):
    case(gpu, 2, 9000, torch.float32, seed=11, bias=4096, hist=20)


def test_a_history_without_columns(gpu):
    from baby_sglang_amd import _hip

    x = torch.randn(2, 40, device=gpu)
    got = _hip.logit_controls(x, history=torch.zeros((2, 0), dtype=torch.int32, device=gpu), history_lens=torch.zeros(2, dtype=torch.int64, device=gpu),
                              repetition=1.5, presence=1.0)
    assert torch.equal(got, x)


def test_the_repetition_penalty_is_the_quotient(gpu):
    """x / repetition in 32 bits, rounded once, is one number: that of the torch division, for ordinary penalties and for those whose
    reciprocal is no normal number or none at all; in 16 bits it is rounded a second time, as the torch one is."""
    from baby_sglang_amd import _hip

    vocab = 5000
    for rep in (1.3, 1.1, 0.7, 3.0, 1e-38, 2e-39, 1e-44, 1e38, 3e38):
        r = torch.tensor(rep, dtype=torch.float32)
        for dtype in (torch.float32, torch.bfloat16, torch.float16):
            x = (3 * torch.randn(4, vocab, generator=torch.Generator().manual_seed(5))).to(dtype)
            x[0, :4] = torch.tensor([0.0, -0.0, 65504.0, 6e-8]).to(dtype)
            hist = torch.arange(vocab, dtype=torch.int32).repeat(4, 1)
            lens = [vocab, 3000, 1, 0]
            want = x.clone()
            for i, n in enumerate(lens):
                f = x[i, :n].float()
                want[i, :n] = torch.where(f > 0, f / r, f * r).to(dtype)
            got = _hip.logit_controls(x.to(gpu), history=hist.to(gpu), history_lens=torch.tensor(lens, device=gpu), repetition=torch.full((4,), r.item(), device=gpu))
            ok = (got.cpu() == want) | (f_tiny(want) & f_tiny(got.cpu()))
            assert bool(ok.all()), (rep, dtype, got.cpu()[~ok][:4], want[~ok][:4])


def f_tiny(t):
    """(subnormal results may be flushed)"""
    return t.float().abs() < 2.0**-126
