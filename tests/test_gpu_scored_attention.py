"""Scored attention (capped, distance-biased scores over an interval of positions) and the token weights
it leaves, on the GPU against the float64 definition (oracle/attn_oracle.py: scored_exact).

What an element may be off, from the arithmetic (u(t) = half a step of type t, relative):
  score   ds = (D + 4) 2^-23 top + 2^-22 (|cap| + |score|): top = scale sum |q_d k_d| bounds a sum of D products
          in 32 bits, truncated; the cap's tanh is good to 2^-22 of the cap; scaling by log2 e, the bias and the
          exponent's own argument each round once, relative to the score
  prob.   relative: 2 ds (its own score and the normaliser) and 2^-21 for exp2, reciprocal and log2
  output  u(out) |o| + (2 ds + 2^-21 + u_p + n 2^-23) sum p |v|, where u_p is the rounding of the probabilities
          that enter the second product: f32 none; f16 2^-11 and 2^-25 per token absolute (a step of the
          subnormals); bf16 decode 2^-16 (hi + lo pairs), bf16 extend 2^-8
"""
import math
import random

import pytest
import torch

from oracle import attn_oracle as orc

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
HEADS = {"1.5b": (12, 2, 128), "7b": (28, 4, 128), "0.5b": (14, 2, 64), "mha": (3, 3, 128), "one": (16, 1, 128), "d64": (4, 4, 64)}


def make(seed, heads, dtype, lens, layout="interleaved", pad_cols=5, q_rows=None, q_scale=2.0):
    g = torch.Generator().manual_seed(seed)
    hq, hkv, dim = HEADS[heads]
    total = sum(lens)
    kv = torch.randn(total + 3, 2, hkv, dim, generator=g).to(dtype)
    if layout == "interleaved":
        k, v = kv[:, 0], kv[:, 1]
    else:
        k, v = kv[:, 0].contiguous(), kv[:, 1].contiguous()
    perm = (torch.randperm(total, generator=g) + 1).to(torch.int32)
    n_rows = len(lens) + 2
    table = torch.randint(0, total + 1, (n_rows, max(lens) + pad_cols), generator=g, dtype=torch.int32)
    req = torch.randperm(n_rows, generator=g)[: len(lens)]
    at = 0
    for r, n in zip(req.tolist(), lens):
        table[r, :n] = perm[at : at + n]
        at += n
    q = (q_scale * torch.randn(q_rows if q_rows is not None else len(lens), hq, dim, generator=g)).to(dtype)
    return dict(hq=hq, hkv=hkv, dim=dim, dtype=dtype, q=q, k=k, v=v, table=table, req=req, lens=lens, g=g)


def to_gpu(c, dev):
    kv = {}
    if c["k"].is_contiguous():
        kv["k"], kv["v"] = c["k"].to(dev), c["v"].to(dev)
    else:
        both = torch.stack((c["k"], c["v"]), 1).to(dev)
        kv["k"], kv["v"] = both[:, 0], both[:, 1]
    return dict(c, q=c["q"].to(dev), table=c["table"].to(dev), req=c["req"].to(dev), seq=torch.tensor(c["lens"], dtype=torch.int64, device=dev), **kv)


def slopes_of(hq):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)])


def score_error(top, cap, lse, dim):
    big = top + abs(cap)
    return (dim + 4) * 2.0**-23 * top + 2.0**-22 * (abs(cap) + torch.where(lse.isinf(), torch.zeros_like(lse), lse.abs()) + big)


def check_rows(out, want, mass, lse, top, cap, dtype, out_dtype, u_p, n_max, v_max, dim):
    ds = score_error(top, cap, lse, dim)[..., None]
    rel = 2 * ds + 2.0**-21 + u_p + n_max * 2.0**-23
    bound = U[out_dtype] * want.abs() + rel * mass * (1 + U[out_dtype]) + 1e-30
    if dtype == torch.float16:
        bound = bound + n_max * 2.0**-25 * v_max + 2.0**-25
    err = (out.double().cpu().view_as(want) - want).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} outside; worst ratio {(err / bound).max().item():.2f}, err {err[bad].max().item():.3e}"


def decode_case(gpu, heads, dtype, lens, cap=0.0, slopes=False, start=None, stop=None, weights=True, seed=0, out_f32=False, layout="interleaved", **kw):
    from baby_sglang_amd import _hip

    c = make(seed, heads, dtype, lens, layout)
    d = to_gpu(c, gpu)
    sl = slopes_of(c["hq"]) if slopes else None
    st = torch.tensor(start, dtype=torch.int32) if start is not None else None
    sp = torch.tensor(stop, dtype=torch.int32) if stop is not None else None
    scale = c["dim"] ** -0.5
    old = torch.rand(c["table"].shape, generator=c["g"])
    w = old.to(gpu)
    lse = torch.empty((len(lens), c["hq"]), device=gpu)
    out = _hip.paged_decode_scored(
        d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"], scale=scale, logit_cap=cap, slopes=sl.to(gpu) if slopes else None,
        visible_from=st.to(gpu) if st is not None else None, visible_to=sp.to(gpu) if sp is not None else None,
        token_weights=w if weights else None, lse=lse, out_dtype=torch.float32 if out_f32 else None, **kw)
    torch.cuda.synchronize()
    want, mass, lse64, received, top = orc.scored_exact(
        c["q"], c["k"], c["v"], c["table"][c["req"]], lens, range(len(lens)), [n - 1 for n in lens], scale, cap, sl, st, sp)
    u_p = {torch.bfloat16: 2.0**-16, torch.float16: 2.0**-11, torch.float32: 0.0}[dtype]
    check_rows(out, want, mass, lse64, top, cap, dtype, torch.float32 if out_f32 else dtype, u_p, max(lens), c["v"].abs().max().item(), c["dim"])
    ds = score_error(top, cap, lse64, c["dim"])
    live = ~lse64.isinf()
    assert torch.equal(lse.cpu().isinf(), ~live)
    assert bool(((lse.cpu().double() - lse64)[live].abs() <= (2 * ds + 2.0**-20 + max(lens) * 2.0**-23 + 2.0**-21 * lse64.abs())[live]).all())
    if weights:
        got = w.cpu()
        expect = old.double().clone()
        slack = torch.zeros_like(expect)
        for i, n in enumerate(lens):
            r = int(c["req"][i])
            expect[r, :n] += received[i]
            slack[r, :n] += received[i] * (4 * ds[i].max() + 2.0**-20 + max(lens) * 2.0**-23)
        bound = slack + 2.0**-23 * expect.abs()
        untouched = torch.ones_like(old, dtype=torch.bool)
        for i, n in enumerate(lens):
            lo = 0 if start is None else max(0, min(start[i], n))
            hi = n if stop is None else max(lo, min(stop[i], n))
            untouched[int(c["req"][i]), lo:hi] = False
        assert torch.equal(got[untouched], old[untouched])
        assert bool(((got.double() - expect).abs() <= bound).all())
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads", list(HEADS))
def test_decode_types_and_heads(gpu, heads, dtype):
    hq, hkv, _ = HEADS[heads]
    if hq // hkv > 8 and dtype == torch.float32:
        pytest.skip("f32 kernels take up to 8 q heads per kv head")
    decode_case(gpu, heads, dtype, [1, 2, 15, 16, 17, 300, 33, 64], cap=8.0, slopes=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cap,slopes", [(0.0, False), (0.0, True), (3.0, False), (50.0, True)])
def test_decode_score_shapes(gpu, dtype, cap, slopes):
    decode_case(gpu, "1.5b", dtype, [700, 5, 1301], cap=cap, slopes=slopes, seed=3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_decode_intervals(gpu, dtype):
    """From and to at, inside and outside the request's ends; empty and upside-down intervals; ragged."""
    lens = [1, 40, 40, 600, 600, 600, 1100, 17, 90, 33]
    start = [0, 39, 40, 0, 599, 100, 513, 9, -5, 50]
    stop = [1, 40, 40, 1, 700, 612, 1090, 3, 1 << 30, -3]
    decode_case(gpu, "7b", dtype, lens, cap=20.0, slopes=True, start=start, stop=stop, seed=4)
    decode_case(gpu, "0.5b", dtype, lens, cap=20.0, start=start, stop=stop, seed=5)


def test_decode_nothing_visible_at_all(gpu):
    out = decode_case(gpu, "1.5b", torch.bfloat16, [5, 60, 200], start=[5, 60, 200], seed=6)
    assert not bool(out.any())


@pytest.mark.parametrize("kw", [dict(n_splits=1), dict(n_splits=7), dict(n_splits=64), dict(variant=1), dict(variant=2), dict(max_seq_len=256),
                                dict(out_f32=True), dict(out_f32=True, n_splits=1), dict(layout="split"), dict(weights=False), dict(variant=0x200)])
def test_decode_launch_forms(gpu, kw):
    lens = [200, 256, 129] if "max_seq_len" in kw else [2000, 1, 777, 1536]
    decode_case(gpu, "1.5b", torch.bfloat16, lens, cap=5.0, slopes=True, start=[3, 0, 20, 1000][: len(lens)], seed=7, **kw)


@pytest.mark.parametrize("batch,n", [(1, 5003), (40, 130), (200, 70), (70, 600)])
def test_decode_batches(gpu, batch, n):
    r = random.Random(batch)
    lens = [r.randint(1, n) for _ in range(batch)]
    lens[0] = n
    decode_case(gpu, "one" if batch == 200 else "1.5b", torch.bfloat16, lens, cap=30.0, start=[r.randint(0, x) for x in lens], seed=8)


def test_decode_without_changes_is_the_plain_decode(gpu):
    from baby_sglang_amd import _hip

    for heads, dtype in (("1.5b", torch.bfloat16), ("0.5b", torch.float16), ("7b", torch.float32)):
        d = to_gpu(make(9, heads, dtype, [1, 500, 37, 1025]), gpu)
        args = (d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"])
        assert torch.equal(_hip.paged_decode_scored(*args), _hip.paged_decode(*args))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_decode_reads_nothing_outside_the_interval(gpu, dtype):
    """NaN, infinities and the type's lowest value in every cached row that may not be seen."""
    from baby_sglang_amd import _hip

    lens, start, stop = [100, 333, 48], [10, 100, 0], [90, 333, 17]
    c = make(10, "1.5b", dtype, lens)
    d = to_gpu(c, gpu)
    st, sp = (torch.tensor(x, dtype=torch.int32, device=gpu) for x in (start, stop))
    kw = dict(logit_cap=10.0, visible_from=st, visible_to=sp)
    clean = _hip.paged_decode_scored(d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"], **kw)
    hidden = torch.ones(d["k"].shape[0], dtype=torch.bool, device=gpu)
    for i in range(3):
        hidden[d["table"][d["req"][i], start[i] : stop[i]].long()] = False
    for bad in (float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).min):
        d["k"][hidden] = bad
        d["v"][hidden] = bad
        w = torch.zeros(d["table"].shape, device=gpu)
        assert torch.equal(clean, _hip.paged_decode_scored(d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"], token_weights=w, **kw))
        assert bool(w.isfinite().all())


def test_decode_requests_on_the_same_row_add_up(gpu):
    from baby_sglang_amd import _hip

    c = make(11, "1.5b", torch.bfloat16, [400, 90, 300])
    d = to_gpu(c, gpu)
    req = torch.stack((d["req"][0], d["req"][1], d["req"][0], d["req"][0]))
    seq = torch.tensor([400, 90, 250, 399], dtype=torch.int64, device=gpu)
    st = torch.tensor([100, 0, 20, 390], dtype=torch.int32, device=gpu)
    q = torch.randn(4, 12, 128, device=gpu).to(torch.bfloat16)
    old = torch.rand(d["table"].shape, device=gpu)
    w_out = torch.full_like(old, -7.0)
    _hip.paged_decode_scored(q, d["k"], d["v"], d["table"], req, seq, visible_from=st, token_weights=old, token_weights_out=w_out)
    one = torch.zeros((4,) + tuple(old.shape), device=gpu)
    for i in range(4):
        _hip.paged_decode_scored(q[i : i + 1], d["k"], d["v"], d["table"], req[i : i + 1], seq[i : i + 1], visible_from=st[i : i + 1],
                                 token_weights=one[i])
    total = old.double() + one.double().sum(0)
    touched = torch.zeros(old.shape, dtype=torch.bool, device=gpu)
    for i in range(4):
        touched[req[i], int(st[i]) : int(seq[i])] = True
    assert bool((w_out[~touched] == -7.0).all())
    assert bool(((w_out.double() - total).abs()[touched] <= 1e-5).all())  # (12 heads, 4 sums in 32 bits: 2^-20 of at most 48)


def test_decode_writes_the_new_rows(gpu):
    """Fused and separate KV write: the slabs hold the new rows and attention has read them."""
    from baby_sglang_amd import _hip

    for heads, dtype in (("1.5b", torch.bfloat16), ("0.5b", torch.float32)):
        c = make(12, heads, dtype, [33, 512, 1])
        outs = []
        for fuse in (False, True):
            d = to_gpu(c, gpu)
            g = torch.Generator().manual_seed(1)
            kn, vn = (torch.randn(3, c["hkv"], c["dim"], generator=g).to(dtype).to(gpu) for _ in range(2))
            loc = torch.stack([d["table"][d["req"][i], c["lens"][i] - 1] for i in range(3)])
            outs.append(_hip.paged_decode_scored(d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"], logit_cap=4.0, k_new=kn, v_new=vn,
                                                 out_cache_loc=loc, fuse_kv_write=fuse))
            assert torch.equal(d["k"][loc.long()], kn) and torch.equal(d["v"][loc.long()], vn)
        assert torch.equal(outs[0], outs[1])
        c["k"][loc.cpu().long()], c["v"][loc.cpu().long()] = kn.cpu(), vn.cpu()
        want, mass, lse, _, top = orc.scored_exact(c["q"], c["k"], c["v"], c["table"][c["req"]], c["lens"], range(3), [n - 1 for n in c["lens"]],
                                                   c["dim"] ** -0.5, 4.0)
        check_rows(outs[0], want, mass, lse, top, 4.0, dtype, dtype, 2.0**-16, 512, 6.0, c["dim"])


def test_decode_graph_replays_and_streams(gpu):
    """A captured decode with weights, replayed with eager work in between; another stream's workspace is another one."""
    from baby_sglang_amd import _hip

    c = make(13, "1.5b", torch.bfloat16, [900, 64, 333])
    d = to_gpu(c, gpu)
    n_splits = _hip.decode_num_splits(3, 2, d["table"].shape[1])
    ws = _hip.new_decode_workspace(_hip.decode_scored_workspace_bytes(3, 12, 128, n_splits, d["table"].shape[1], True), gpu)
    out, w, w2 = torch.zeros(3, 12 * 128, device=gpu, dtype=torch.bfloat16), torch.zeros(d["table"].shape, device=gpu), torch.zeros(d["table"].shape, device=gpu)

    def call(out, w, ws):
        return _hip.paged_decode_scored(d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"], logit_cap=9.0, token_weights=w, out=out, workspace=ws,
                                        n_splits=n_splits)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(out, w, ws)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out, w, ws)
    for i in range(4):
        d["q"].copy_(torch.randn_like(d["q"]))
        w.zero_()
        w2.zero_()
        eager = call(torch.zeros_like(out), w2, None)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(w, w2), i


def test_decode_long_rows_and_far_slots(gpu):
    """One request of 131072 tokens in a pool whose used slots stand at its far end."""
    from baby_sglang_amd import _hip

    n, hq, hkv, dim = 131072, 12, 2, 128
    far = 6_000_000  # 6 M slots x 1 KiB: offsets pass 32 bits
    kv = torch.zeros((far, 2, hkv, dim), dtype=torch.bfloat16, device=gpu)
    kv[far - n :].normal_()
    table = (torch.randperm(n, device=gpu) + (far - n)).to(torch.int32)[None].contiguous()
    q = torch.randn(1, hq, dim, device=gpu).to(torch.bfloat16)
    req, seq = torch.zeros(1, dtype=torch.int64, device=gpu), torch.tensor([n], device=gpu)
    w = torch.zeros((1, n), device=gpu)
    out = _hip.paged_decode_scored(q, kv[:, 0], kv[:, 1], table, req, seq, logit_cap=20.0, token_weights=w).view(hq, dim)
    k, v = (kv[:, i][table[0].long()].float() for i in (0, 1))
    for h in (0, 5, 11):
        s = 20.0 * torch.tanh((k[:, h // 6].double() @ q[0, h].double()) * dim**-0.5 / 20.0)
        p = torch.softmax(s, 0)
        want = p @ v[:, h // 6].double()
        # ds <= 132 * 2^-23 * top + 2^-22 (cap + lse + ...) < 132 * 2^-23 * 20 + 2^-22 * 60 = 3.3e-4; the sum of 131072 tokens adds
        # its own rounding (16-token tiles, 32 bits: relative 8192 steps of 2^-23 = 1e-3 at the very worst)
        mass = p @ v[:, h // 6].double().abs()
        assert bool(((out[h].double() - want).abs() <= 2.0**-8 * want.abs() + 2e-3 * mass).all())
    assert abs(w.double().sum().item() - hq) < 2e-3 * hq


def test_decode_refusals(gpu):
    from baby_sglang_amd import _hip

    d = to_gpu(make(14, "1.5b", torch.bfloat16, [20, 30]), gpu)
    args = (d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"])
    for bad in (dict(logit_cap=-1.0), dict(logit_cap=float("nan")), dict(logit_cap=float("inf")), dict(slopes=torch.zeros(11, device=gpu)),
                dict(slopes=torch.zeros(12, device=gpu, dtype=torch.float16)), dict(visible_from=torch.zeros(3, dtype=torch.int32, device=gpu)),
                dict(visible_to=torch.zeros(2, device=gpu)), dict(token_weights=torch.zeros(d["table"].shape, device=gpu).half()),
                dict(token_weights=torch.zeros(2, 2, device=gpu)), dict(token_weights_out=torch.zeros(d["table"].shape, device=gpu)),
                dict(out=torch.zeros(2, 12 * 64, device=gpu, dtype=torch.bfloat16)), dict(lse=torch.zeros(2, device=gpu)),
                dict(k_new=d["k"][:2]), dict(n_splits=65)):
        with pytest.raises(ValueError):
            _hip.paged_decode_scored(*args, **bad)
    with pytest.raises(ValueError):
        _hip.paged_decode_scored(d["q"].half(), *args[1:])
    with pytest.raises(RuntimeError):
        _hip.paged_decode_scored(d["q"].cpu(), *args[1:])
    assert math.isfinite(_hip.paged_decode_scored(*args).float().sum().item())
