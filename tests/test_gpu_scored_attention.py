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
        # cut alike, bit for bit; by default a scored call may cut a long request finer, and then two sums of the same
        # probabilities (rounded to f16, or to hi + lo bf16) in 32 bits over up to 1025 tokens, normalised and merged in another
        # order, are rounded once each: 2 u |o| + (2 u_p + 2 * 1030 * 2^-23) sum p |v|, and sum p |v| <= max |v|
        uniform = _hip.DECODE_UNIFORM_SPLITS
        assert torch.equal(_hip.paged_decode_scored(*args, variant=uniform), _hip.paged_decode(*args, variant=uniform))
        got, want = _hip.paged_decode_scored(*args).double(), _hip.paged_decode(*args).double()
        u_p = {torch.bfloat16: 2.0**-16, torch.float16: 2.0**-11, torch.float32: 0.0}[dtype]
        slack = (2 * u_p + 2060 * 2.0**-23) * d["v"].double().abs().max()
        assert bool(((got - want).abs() <= 2 * U[dtype] * want.abs() + slack).all())


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


# --------------------------------------------------------------------------- extend
def intervals(kind, lens, ext, seed):
    """Per extend row: {start, stop} lists of the mask kinds, or None."""
    r = random.Random(seed)
    start, stop = [], []
    for n, e in zip(lens, ext):
        cuts = sorted(r.randrange(n) for _ in range(3)) if n else []
        for i in range(n - e, n):
            a, b = 0, i + 1
            if kind == "window":
                a = max(0, i + 1 - max(1, n // 4))
            elif kind == "prefix":
                b = max(b, n // 2)
            elif kind == "document":
                a = max([0] + [c for c in cuts if c <= i])
            elif kind == "both":  # a document read in both directions
                a = max([0] + [c for c in cuts if c <= i])
                b = min([n] + [c for c in cuts if c > i])
            elif kind == "empty" and r.random() < 0.3:
                b = a
            elif kind == "wild":
                a, b = r.randint(-5, n + 5), r.randint(-5, n + 5)
            start.append(a)
            stop.append(b)
    return start, stop


def extend_case(gpu, heads, dtype, ext, prefix, cap=0.0, slopes=False, kind=None, seed=0, layout="interleaved", extra_rows=0, only=None, poison=None, pad_cols=5, **kw):
    from baby_sglang_amd import _hip

    lens = [a + b for a, b in zip(ext, prefix)]
    c = make(seed, heads, dtype, lens, layout, pad_cols=pad_cols, q_rows=sum(ext) + extra_rows)
    st = sp = None
    if kind is not None:
        st, sp = (torch.tensor(x, dtype=torch.int32) for x in intervals(kind, lens, ext, seed))
        st, sp = (torch.cat((x, torch.zeros(extra_rows, dtype=torch.int32))) for x in (st, sp))
    row_req = [i for i, e in enumerate(ext) for _ in range(e)]
    row_pos = [n - e + j for n, e in zip(lens, ext) for j in range(e)]
    rows = list(range(sum(ext)))
    scale = c["dim"] ** -0.5
    sl = slopes_of(c["hq"]) if slopes else None
    if poison is not None:
        poison(c, row_req, row_pos, st, sp)
    d = to_gpu(c, gpu)
    out = torch.full((sum(ext) + extra_rows, c["hq"] * c["dim"]), -3.0, dtype=dtype, device=gpu)
    got = _hip.paged_prefill_scored(
        d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"], torch.tensor(prefix, device=gpu), torch.tensor(ext, device=gpu), scale=scale,
        logit_cap=cap, slopes=sl.to(gpu) if slopes else None, visible_from=st.to(gpu) if st is not None else None,
        visible_to=sp.to(gpu) if sp is not None else None, out=out, **kw)
    torch.cuda.synchronize()
    assert got is out
    if extra_rows:
        assert bool((out[sum(ext):] == -3.0).all())
    if only is not None and len(rows) > only:
        rows = sorted(random.Random(seed).sample(rows, only - 2) + [0, len(rows) - 1])
    pick = lambda x: x[rows] if x is not None else None  # noqa: E731
    want, mass, lse, _, top = orc.scored_exact(c["q"][rows], c["k"], c["v"], c["table"][c["req"]], lens, [row_req[r] for r in rows], [row_pos[r] for r in rows],
                                               scale, cap, sl, pick(st), pick(sp))
    u_p = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 0.0}[dtype]
    finite = c["v"][c["v"].isfinite()].abs().max().item()
    # (f16: probabilities stand against a reference up to 2^6 below the maximum, so the subnormal step is not scaled up)
    check_rows(out[rows], want, mass, lse, top, cap, dtype, dtype, u_p, max(lens), finite, c["dim"])
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("ext,prefix", [([3, 1, 0, 17, 40], [0, 5, 9, 33, 600]), ([130, 64, 1, 200], [0, 31, 70, 513])])
def test_extend_types_and_heads(gpu, heads, dtype, ext, prefix):
    hq, hkv, _ = HEADS[heads]
    if hq // hkv > 8 and dtype == torch.float32:
        pytest.skip("f32 kernels take up to 8 q heads per kv head")
    extend_case(gpu, heads, dtype, ext, prefix, cap=8.0, slopes=True, only=60)


@pytest.mark.parametrize("heads", ["1.5b", "0.5b"])
@pytest.mark.parametrize("cap,slopes", [(0.0, False), (0.0, True), (3.0, False), (50.0, False), (50.0, True)])
@pytest.mark.parametrize("kind", [None, "window", "prefix", "document", "both", "empty", "wild"])
def test_extend_masks_and_shapes(gpu, heads, cap, slopes, kind):
    extend_case(gpu, heads, torch.bfloat16, [150, 70, 33], [0, 100, 700], cap=cap, slopes=slopes, kind=kind, seed=20, only=70)
    extend_case(gpu, heads, torch.float16, [9, 20, 33, 1], [0, 100, 40, 700], cap=cap, slopes=slopes, kind=kind, seed=21, only=40)


@pytest.mark.parametrize("kind", [None, "document", "wild"])
def test_extend_f32_masks(gpu, kind):
    extend_case(gpu, "7b", torch.float32, [50, 20, 3], [0, 33, 300], cap=10.0, slopes=True, kind=kind, seed=22, only=40)


@pytest.mark.parametrize("kw", [dict(layout="split"), dict(extra_rows=5), dict(variant=1), dict(variant=2)])
def test_extend_launch_forms(gpu, kw):
    extend_case(gpu, "7b", torch.bfloat16, [65, 100, 7], [513, 0, 64], cap=30.0, kind="document", seed=23, only=50, **kw)


@pytest.mark.parametrize("heads,dtype", [("7b", torch.bfloat16), ("0.5b", torch.float16), ("d64", torch.bfloat16), ("1.5b", torch.float32), ("one", torch.float16),
                                         ("mha", torch.bfloat16)])
@pytest.mark.parametrize("ext,prefix,kind", [([1], [0], None), ([1], [2500], None), ([3, 0, 2], [700, 9, 0], "both"), ([7, 11], [1300, 40], "document"),
                                             ([5, 9, 20], [0, 600, 33], "wild"), ([8], [4000], "prefix")])
def test_extend_a_few_tokens(gpu, heads, dtype, ext, prefix, kind):
    """So few new tokens that they run as rows of the decode kernel; rows that no request owns stay as they were."""
    if heads == "one" and dtype == torch.float32:
        pytest.skip("f32 kernels take up to 8 q heads per kv head")
    extend_case(gpu, heads, dtype, ext, prefix, cap=20.0, slopes=True, kind=kind, seed=36, extra_rows=3)


@pytest.mark.parametrize("heads,dtype", [("1.5b", torch.bfloat16), ("0.5b", torch.bfloat16), ("7b", torch.float32)])
def test_extend_unowned_rows(gpu, heads, dtype):
    extend_case(gpu, heads, dtype, [150, 130], [0, 30], cap=20.0, seed=37, extra_rows=70, only=40)


@pytest.mark.parametrize("heads,dtype", [("1.5b", torch.bfloat16), ("0.5b", torch.float16), ("7b", torch.float16), ("one", torch.bfloat16)])
@pytest.mark.parametrize("ext,prefix,kind,cap", [([300], [2000], None, 20.0), ([260, 0, 90], [1500, 40, 700], "document", 0.0), ([280], [1800], "wild", 70.0),
                                                 ([200, 150], [0, 2100], "prefix", 0.0), ([513], [1100], "empty", 30.0)])
def test_extend_long_streams_in_pieces(gpu, heads, dtype, ext, prefix, kind, cap):
    """Few blocks over long prefixes: the streams are cut and merged (page table of more than 2000 columns); short requests beside
    long ones leave pieces empty; rows that no request owns stay as they were."""
    extend_case(gpu, heads, dtype, ext, prefix, cap=cap, slopes=cap != 20.0, kind=kind, seed=38, extra_rows=9, only=24, pad_cols=800)


def test_extend_pieces_keep_hidden_tokens_out(gpu):
    """A NaN value in one piece of a cut stream: rows that do not see it are right, whichever piece it is in."""
    def poison(c, row_req, row_pos, st, sp):
        for at in (3, 700, 2100):
            c["v"][c["table"][c["req"][0], at].long()] = float("nan")
        st[:], sp[:] = torch.tensor([[4, 700], [701, 2100], [2101, 2300], [10, 600]]).t().repeat(1, 70)[:, : len(st)].to(torch.int32)

    extend_case(gpu, "1.5b", torch.bfloat16, [280], [2020], cap=20.0, kind="wild", seed=39, only=30, poison=poison, pad_cols=800)


def test_extend_long(gpu):
    """Several blocks of page-table entries, many steps; ring and entry staging wrap."""
    extend_case(gpu, "one", torch.bfloat16, [700, 64], [2100, 1500], cap=20.0, slopes=True, seed=24, only=24)
    extend_case(gpu, "mha", torch.float16, [1300], [0], kind="window", slopes=True, seed=25, only=24)


def test_extend_many_requests(gpu):
    r = random.Random(3)
    ext = [r.choice([0, 1, 2, 5, 30, 64, 65, 129]) for _ in range(90)]
    extend_case(gpu, "1.5b", torch.bfloat16, ext, [r.randint(0, 90) for _ in ext], cap=12.0, kind="document", seed=26, only=80)
    ext = [r.randint(0, 20) for _ in range(130)]
    extend_case(gpu, "7b", torch.float16, ext, [r.randint(0, 90) for _ in ext], slopes=True, kind="both", seed=27, only=80)


def test_extend_all_rows_empty(gpu):
    from baby_sglang_amd import _hip

    c = make(28, "1.5b", torch.bfloat16, [70, 20], q_rows=90)
    d = to_gpu(c, gpu)
    out = _hip.paged_prefill_scored(d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"], torch.zeros(2, dtype=torch.int64, device=gpu), d["seq"],
                                    logit_cap=5.0, visible_to=torch.zeros(90, dtype=torch.int32, device=gpu))
    assert not bool(out.any())


@pytest.mark.parametrize("scale", [0.0, -0.11])
def test_extend_scale_of_any_sign(gpu, scale):
    from baby_sglang_amd import _hip

    c = make(29, "1.5b", torch.bfloat16, [100], q_rows=100)
    d = to_gpu(c, gpu)
    for cap in (0.0, 6.0):
        out = _hip.paged_prefill_scored(d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"], torch.zeros(1, dtype=torch.int64, device=gpu), d["seq"],
                                        scale=scale, logit_cap=cap)
        want, mass, lse, _, top = orc.scored_exact(c["q"], c["k"], c["v"], c["table"][c["req"]], [100], [0] * 100, range(100), scale, cap)
        check_rows(out, want, mass, lse, top.abs(), cap, torch.bfloat16, torch.bfloat16, 2.0**-8, 100, 6.0, 128)


@pytest.mark.parametrize("cap", [60.0, 61.0, 100.0])
@pytest.mark.parametrize("side", [-1.0, 1.0])
def test_extend_scores_at_the_cap(gpu, cap, side):
    """Every visible score at one end of the cap's range, for some rows: the exponentials' range is the cap's (bf16 takes a
    fixed reference up to 60); the others see ordinary scores."""
    def poison(c, row_req, row_pos, st, sp):
        c["k"][:] = c["k"].abs()  # so that a row of one sign has scores of one sign
        c["q"][::2] = (c["q"][::2].abs() * 40.0 * side).to(c["q"].dtype)

    extend_case(gpu, "1.5b", torch.bfloat16, [90, 33], [0, 70], cap=cap, seed=34, poison=poison)
    extend_case(gpu, "1.5b", torch.bfloat16, [9, 3], [0, 70], cap=cap, slopes=True, seed=35, poison=poison)


@pytest.mark.parametrize("heads,dtype", [("1.5b", torch.bfloat16), ("0.5b", torch.float16), ("7b", torch.float32)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), "lowest"])
def test_extend_nothing_leaks_from_hidden_tokens(gpu, heads, dtype, bad):
    """A document whose keys and values are not finite beside documents that must not see it, in the same blocks;
    rows that do see it are not looked at."""
    from baby_sglang_amd import _hip

    val = torch.finfo(dtype).min if bad == "lowest" else bad
    lens, ext = [200, 90], [200, 90]
    c = make(30, heads, dtype, lens, q_rows=290)
    lo, hi = 70, 101  # the bad document of request 0
    start = [0 if i < lo else lo if i < hi else hi for i in range(200)] + [0] * 90
    stop = [lo if i < lo else hi if i < hi else 200 for i in range(200)] + [90] * 90
    st, sp = (torch.tensor(x, dtype=torch.int32, device=gpu) for x in (start, stop))
    zero = torch.zeros(2, dtype=torch.int64, device=gpu)

    def call(d):
        return _hip.paged_prefill_scored(d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"], zero, d["seq"], logit_cap=9.0, slopes=slopes_of(c["hq"]).to(gpu),
                                         visible_from=st, visible_to=sp)

    clean = call(to_gpu(c, gpu))
    slots = c["table"][c["req"][0], lo:hi].long()
    for what in ("k", "v"):
        d = to_gpu(c, gpu)
        d[what][slots.to(gpu)] = val
        out = call(d)
        rows = [i for i in range(290) if not lo <= i < hi]
        assert bool(out[rows].isfinite().all())
        # (rows that were computed again went through another order of sums: held to the definition)
        want, mass, lse, _, top = orc.scored_exact(c["q"][rows], c["k"], c["v"], c["table"][c["req"]], lens, [0 if i < 200 else 1 for i in rows],
                                                   [i if i < 200 else i - 200 for i in rows], c["dim"] ** -0.5, 9.0, slopes_of(c["hq"]),
                                                   torch.tensor(start)[rows], torch.tensor(stop)[rows])
        u_p = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 0.0}[dtype]
        check_rows(out[rows], want, mass, lse, top, 9.0, dtype, dtype, u_p, 200, 6.0, c["dim"])
        if what == "v" and isinstance(bad, float) and bad != bad:
            assert bool(out[lo:hi].isnan().all())  # ... and who sees NaN gets NaN
    assert bool(clean.isfinite().all())


def test_extend_without_changes_agrees_with_the_plain_extend(gpu):
    from baby_sglang_amd import _hip

    for heads in ("1.5b", "7b", "0.5b"):
        c = make(31, heads, torch.bfloat16, [300, 77, 610], q_rows=377)
        d = to_gpu(c, gpu)
        args = (d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"], torch.tensor([0, 0, 610], device=gpu), torch.tensor([300, 77, 0], device=gpu))
        a, b = _hip.paged_prefill_scored(*args).float(), _hip.paged_prefill(*args).float()
        assert bool(((a - b).abs() <= 2.0**-7 * b.abs() + 2.0**-6).all())  # (two roundings of p and of the result, mass <= 2)


def test_extend_graph_replays_with_the_list_of_a_batch(gpu):
    from baby_sglang_amd import _hip

    c = make(32, "1.5b", torch.bfloat16, [200, 90, 333], q_rows=400)
    d = to_gpu(c, gpu)
    pre, ext = torch.tensor([0, 13, 210], device=gpu), torch.tensor([200, 77, 123], device=gpu)
    st = torch.zeros(400, dtype=torch.int32, device=gpu)
    ws = torch.empty(_hip.prefill_workspace_bytes(3, 400, 12, 128), dtype=torch.uint8, device=gpu)
    out = torch.zeros(400, 12 * 128, dtype=torch.bfloat16, device=gpu)

    def call(o, w, **kw):
        return _hip.paged_prefill_scored(d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"], pre, ext, logit_cap=9.0, visible_from=st, out=o, workspace=w, **kw)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = call(out, ws).clone()
        assert torch.equal(call(torch.zeros_like(out), ws, list_ready=True), first)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out, ws)
    for i in range(4):
        d["q"].copy_(torch.randn_like(d["q"]))
        st.fill_(i * 20)
        eager = call(torch.zeros_like(out), None)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), i


def test_extend_refusals(gpu):
    from baby_sglang_amd import _hip

    d = to_gpu(make(33, "1.5b", torch.bfloat16, [20, 30], q_rows=50), gpu)
    args = (d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"], torch.zeros(2, dtype=torch.int64, device=gpu), d["seq"])
    for bad in (dict(logit_cap=-1.0), dict(slopes=torch.zeros(11, device=gpu)), dict(visible_from=torch.zeros(2, dtype=torch.int32, device=gpu)),
                dict(visible_to=torch.zeros(50, device=gpu)), dict(out=torch.zeros(49, 1536, dtype=torch.bfloat16, device=gpu)), dict(list_ready=True)):
        with pytest.raises(ValueError):
            _hip.paged_prefill_scored(*args, **bad)
    with pytest.raises(ValueError):
        _hip.paged_prefill_scored(*args[:6], args[6][:1], args[7])
    with pytest.raises(RuntimeError):
        _hip.paged_prefill_scored(*args[:7], args[7].cpu())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_decode_writes_new_rows_nobody_sees(gpu, dtype):
    """Intervals that end before the new token, and empty ones: its K/V row is written all the same, fused or not."""
    from baby_sglang_amd import _hip

    lens = [40, 700, 1, 90]
    c = make(51, "1.5b", dtype, lens)
    st, sp = (torch.tensor(x, dtype=torch.int32, device=gpu) for x in ([0, 30, 1, 60], [39, 600, 1, 20]))
    for fuse in (False, True):
        d = to_gpu(c, gpu)
        kn, vn = torch.full((4, 2, 128), 3.0, dtype=dtype, device=gpu), torch.full((4, 2, 128), float("nan"), dtype=dtype, device=gpu)
        loc = torch.stack([d["table"][d["req"][i], lens[i] - 1] for i in range(4)])
        w = torch.zeros(d["table"].shape, device=gpu)
        out = _hip.paged_decode_scored(d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"], logit_cap=8.0, visible_from=st, visible_to=sp, k_new=kn,
                                       v_new=vn, out_cache_loc=loc, fuse_kv_write=fuse, token_weights=w)
        assert torch.equal(d["k"][loc.long()], kn) and bool(d["v"][loc.long()].isnan().all())
        assert bool(out.isfinite().all()) and not bool(out[2:].any()) and bool(w.isfinite().all())


@pytest.mark.parametrize("cap", [2.0**-20, 1e-3, 16384.0])
def test_smallest_and_largest_caps(gpu, cap):
    decode_case(gpu, "1.5b", torch.bfloat16, [300, 20], cap=cap, seed=52)
    decode_case(gpu, "mha", torch.float32, [300, 20], cap=cap, seed=53)
    extend_case(gpu, "1.5b", torch.bfloat16, [90, 33], [0, 70], cap=cap, seed=54)
    extend_case(gpu, "1.5b", torch.bfloat16, [90, 33], [0, 70], cap=cap, slopes=True, seed=55)


def test_extend_tiny_scale_with_a_bias(gpu):
    from baby_sglang_amd import _hip

    c = make(56, "1.5b", torch.bfloat16, [100], q_rows=100)
    d = to_gpu(c, gpu)
    sl = slopes_of(12)
    for scale in (1e-36, 1e-20):
        out = _hip.paged_prefill_scored(d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"], torch.zeros(1, dtype=torch.int64, device=gpu), d["seq"],
                                        scale=scale, slopes=sl.to(gpu))
        want, mass, lse, _, top = orc.scored_exact(c["q"], c["k"], c["v"], c["table"][c["req"]], [100], [0] * 100, range(100), scale, 0.0, sl)
        check_rows(out, want, mass, lse, top + 100.0, 0.0, torch.bfloat16, torch.bfloat16, 2.0**-8, 100, 6.0, 128)


@pytest.mark.parametrize("kw", [dict(), dict(n_splits=1), dict(n_splits=3), dict(n_splits=64), dict(variant=0x200), dict(variant=1)])
@pytest.mark.parametrize("heads", ["1.5b", "d64", "7b"])
def test_decode_f32_launch_forms(gpu, heads, kw):
    """The matrix-core form in one piece, some and as many as there are, and the generic kernel."""
    decode_case(gpu, heads, torch.float32, [1, 2, 15, 16, 17, 63, 64, 65, 300, 900], cap=8.0, slopes=True, seed=61, **kw)


def test_decode_f32_up_to_16_heads_per_kv_head(gpu):
    decode_case(gpu, "one", torch.float32, [1, 33, 700], cap=8.0, slopes=True, seed=62)
    decode_case(gpu, "one", torch.float32, [50, 33, 700], start=[0, 33, 650], stop=[50, 33, 651], seed=63)


@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_decode_f32_numbers_that_are_none(gpu, where, bad):
    """A value that is not finite in the last visible token (which also stands in for the places behind it) spreads as the
    definition has it and stays in its request."""
    from baby_sglang_amd import _hip

    c = make(64, "mha", torch.float32, [37, 100])
    d = to_gpu(c, gpu)
    clean = _hip.paged_decode_scored(d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"]).view(2, 3, 128)
    d[where][d["table"][d["req"][0], 36].long()] = bad
    got = _hip.paged_decode_scored(d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"]).view(2, 3, 128)
    assert torch.equal(got[1], clean[1])
    if where == "v":
        assert bool(got[0].isinf().all() if bad == float("inf") else got[0].isnan().all())
    elif bad != bad:
        assert bool(got[0].isnan().all())


def test_decode_f32_more_rows_than_tickets(gpu):
    """8200 requests of 3 kv heads in two pieces each: their results are merged by a launch of its own."""
    from baby_sglang_amd import _hip

    r = random.Random(65)
    lens = [r.randint(1, 3) for _ in range(8200)]
    lens[4000], lens[8199] = 150, 0
    g = torch.Generator().manual_seed(65)
    k, v = (torch.randn(500, 3, 128, generator=g) for _ in range(2))
    table = torch.randint(0, 500, (8200, 160), generator=g, dtype=torch.int32)
    q = torch.randn(8200, 3, 128, generator=g)
    out = _hip.paged_decode_scored(q.to(gpu), k.to(gpu), v.to(gpu), table.to(gpu), torch.arange(8200, device=gpu), torch.tensor(lens, device=gpu),
                                   logit_cap=9.0, n_splits=2)
    rows = [0, 4000, 8198, 8199] + r.sample(range(8200), 60)
    want, mass, lse, _, top = orc.scored_exact(q[rows], k, v, table[rows], [lens[i] for i in rows], range(len(rows)), [lens[i] - 1 for i in rows], 128**-0.5, 9.0)
    check_rows(out[rows], want, mass, lse, top, 9.0, torch.float32, torch.float32, 0.0, 150, 6.0, 128)


@pytest.mark.parametrize("heads", ["1.5b", "0.5b", "one"])
@pytest.mark.parametrize("ext,prefix", [([1], [0]), ([31, 33, 64, 65], [0, 5, 64, 1]), ([200], [900]), ([3, 0, 1, 2], [1000, 5, 0, 31])])
def test_extend_f32_blocks_and_pieces(gpu, heads, ext, prefix):
    for kind in (None, "window", "wild"):
        extend_case(gpu, heads, torch.float32, ext, prefix, cap=7.0, slopes=True, kind=kind, seed=66)


@pytest.mark.parametrize("heads,dtype", [("1.5b", torch.bfloat16), ("one", torch.float16), ("d64", torch.float32)])
@pytest.mark.parametrize("batch", [65, 129, 1500])
def test_decode_ragged_batches_of_many_rows(gpu, heads, dtype, batch):
    """Pieces dealt out over more rows than a wave has lanes, and over more than are looked through (1024): long rows among short and
    empty ones, at the ends and at the lanes' border; sampled rows against the definition."""
    from baby_sglang_amd import _hip

    r = random.Random(batch)
    lens = [r.randint(1, 60) for _ in range(batch)]
    for at, n in ((0, 900), (63, 2300), (64, 1700), (batch - 1, 700)):
        lens[at] = n
    c = make(67, heads, dtype, [1], q_rows=batch)
    g = torch.Generator().manual_seed(68)
    table = torch.randint(0, 3000, (batch, 2400), generator=g, dtype=torch.int32)
    k, v = (torch.randn(3000, c["hkv"], c["dim"], generator=g).to(dtype) for _ in range(2))
    st = torch.tensor([r.choice([0, 0, n // 2, n]) for n in lens], dtype=torch.int32)
    st[[0, 63, 64, batch - 1]] = torch.tensor([0, 5, 0, 100], dtype=torch.int32)
    w = torch.zeros((batch, 2400), device=gpu)
    out = _hip.paged_decode_scored(c["q"].to(gpu), k.to(gpu), v.to(gpu), table.to(gpu), torch.arange(batch, device=gpu), torch.tensor(lens, device=gpu),
                                   logit_cap=9.0, visible_from=st.to(gpu), token_weights=w)
    rows = sorted({0, 1, 62, 63, 64, batch - 1, *r.sample(range(batch), 40)})
    want, mass, lse, received, top = orc.scored_exact(c["q"][rows], k, v, table[rows], [lens[i] for i in rows], range(len(rows)), [lens[i] - 1 for i in rows],
                                                      c["dim"] ** -0.5, 9.0, None, st[rows])
    u_p = {torch.bfloat16: 2.0**-16, torch.float16: 2.0**-11, torch.float32: 0.0}[dtype]
    check_rows(out[rows], want, mass, lse, top, 9.0, dtype, dtype, u_p, 2300, v.abs().max().item(), c["dim"])
    ds = score_error(top, 9.0, lse, c["dim"])
    for i, row in enumerate(rows):
        n = lens[row]
        got = w[row, :n].double().cpu()
        assert bool(((got - received[i]).abs() <= received[i] * (4 * ds[i].max() + 2.0**-20 + n * 2.0**-23)).all())


@pytest.mark.parametrize("hint", [1, 64, 130, 5000])
def test_decode_hints_that_are_wrong_change_nothing(gpu, hint):
    for batch in (2, 70):
        lens = [900, 300] + [5] * (batch - 2)
        decode_case(gpu, "1.5b", torch.bfloat16, lens, cap=8.0, seed=69, max_seq_len=hint)


@pytest.mark.parametrize("heads,dtype,kind", [("7b", torch.bfloat16, "document"), ("0.5b", torch.float16, "wild"), ("1.5b", torch.float32, "prefix"), ("mha", torch.bfloat16, None)])
def test_extend_many_groups_longest_first(gpu, heads, dtype, kind):
    """Launches whose blocks are sorted by what they stream: ragged, with requests that bring nothing; several rows of one request."""
    r = random.Random(5)
    ext = [r.choice([0, 1, 63, 64, 65, r.randint(1, 400)]) for _ in range(40)]
    prefix = [r.choice([0, 7, r.randint(0, 500)]) for _ in ext]
    extend_case(gpu, heads, dtype, ext, prefix, cap=20.0, slopes=True, kind=kind, seed=50, extra_rows=2, only=80)


@pytest.mark.parametrize("batch", [900, 1000, 1100])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_extend_about_as_many_groups_as_are_sorted(gpu, batch, dtype):
    r = random.Random(batch)
    ext = [r.randint(0, 3) for _ in range(batch - 2)] + [200, 90]
    extend_case(gpu, "1.5b", dtype, ext, [r.randint(0, 20) for _ in ext], cap=20.0, kind="window", seed=51, only=120)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_extend_lengths_that_contradict_the_rows(gpu, dtype):
    """100 requests that all claim the 100 rows: the first one has them, the others' lie behind the last row."""
    from baby_sglang_amd import _hip

    c = make(52, "7b", dtype, [150], q_rows=100)
    d = to_gpu(c, gpu)
    claim = lambda first, rest: torch.tensor([first] + [rest] * 99, device=gpu)  # noqa: E731
    row = int(c["req"][0])
    out = _hip.paged_prefill_scored(d["q"], d["k"], d["v"], d["table"], claim(row, row), claim(150, 150), claim(50, 0), claim(100, 100), logit_cap=9.0, variant=2)
    alone = _hip.paged_prefill_scored(d["q"], d["k"], d["v"], d["table"], *(claim(x, 0)[:1] for x in (row, 150, 50, 100)), logit_cap=9.0, variant=2)
    torch.cuda.synchronize()
    want, mass, lse, _, top = orc.scored_exact(c["q"], c["k"], c["v"], c["table"][c["req"]], [150], [0] * 100, list(range(50, 150)), c["dim"] ** -0.5, 9.0, None, None, None)
    u_p = {torch.bfloat16: 2.0**-8, torch.float32: 0.0}[dtype]
    for got in (out, alone):
        check_rows(got, want, mass, lse, top, 9.0, dtype, dtype, u_p, 150, c["v"].abs().max().item(), c["dim"])


def test_extend_sorted_list_kept_and_replayed(gpu):
    """A kept list under other masks and caps, and a captured pair of calls replayed with other lengths."""
    from baby_sglang_amd import _hip

    r = random.Random(8)
    ext = [r.randint(60, 300) for _ in range(20)]
    pre = [r.randint(0, 300) for _ in ext]
    c = make(53, "7b", torch.bfloat16, [a + b for a, b in zip(ext, pre)], q_rows=sum(ext))
    d = to_gpu(c, gpu)
    pre_t, ext_t = torch.tensor(pre, device=gpu), torch.tensor(ext, device=gpu)
    args = (d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"], pre_t, ext_t)
    ws = torch.empty(_hip.prefill_workspace_bytes(20, sum(ext), 28, 128), dtype=torch.uint8, device=gpu)
    st, sp = (torch.tensor(x, dtype=torch.int32, device=gpu) for x in intervals("both", c["lens"], ext, 3))
    first = _hip.paged_prefill_scored(*args, logit_cap=10.0, workspace=ws)
    kept = _hip.paged_prefill_scored(*args, logit_cap=30.0, visible_from=st, visible_to=sp, workspace=ws, list_ready=True)
    assert torch.equal(first, _hip.paged_prefill_scored(*args, logit_cap=10.0))
    assert torch.equal(kept, _hip.paged_prefill_scored(*args, logit_cap=30.0, visible_from=st, visible_to=sp))
    out = torch.empty_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _hip.paged_prefill_scored(*args, logit_cap=10.0, workspace=ws, out=torch.empty_like(first))
        _hip.paged_prefill_scored(*args, logit_cap=30.0, visible_from=st, visible_to=sp, workspace=ws, list_ready=True, out=out)
    for turn in range(3):
        e2 = ext[turn:] + ext[:turn]
        ext_t.copy_(torch.tensor(e2))
        pre_t.copy_(torch.tensor([n - e if n > e else 0 for n, e in zip(c["lens"], e2)]))
        out.zero_()
        eager = _hip.paged_prefill_scored(*args, logit_cap=30.0, visible_from=st, visible_to=sp)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


@pytest.mark.parametrize("cap", [30.0, 60.0])
@pytest.mark.parametrize("side,power", [(1.0, 60), (1.0, 100), (-1.0, -60)])
def test_extend_values_of_the_whole_range(gpu, cap, side, power):
    """Scores at one end of the cap's range and values far from 1: 2^power times a probability of 2^(cap log2 e) is no bf16, nor is what
    2^-60 times 2^-(cap log2 e) leaves of it, and the result is as finite as the values are.  (Products of 2^10 with up to 103 values of 5.5 x
    2^100 stay below 2^120.)"""
    def poison(c, row_req, row_pos, st, sp):
        c["k"][:] = c["k"].abs()
        c["q"][::2] = (c["q"][::2].abs() * 40.0 * side).to(c["q"].dtype)
        c["v"] *= 2.0**power

    extend_case(gpu, "1.5b", torch.bfloat16, [90, 33], [0, 70], cap=cap, seed=70, poison=poison, variant=2)
    extend_case(gpu, "1.5b", torch.bfloat16, [9, 3], [0, 70], cap=cap, seed=71, poison=poison, variant=2)


@pytest.mark.parametrize("ext", [1, 40, 300])
@pytest.mark.parametrize("cap", [0.0, 40.0])
def test_f16_long_flat_tails(gpu, ext, cap):
    """Tokens of score 18.5 among 60000 of score 0, which are 2^-26.7 of one of them each: a probability that f16 cannot hold beside 1, all
    together a part of the row that it can.  The values of the few are 0, so that the tail is all there is of the result.  Extend: one such
    token, ahead of the new ones (the stream goes from the last one back); decode: four in every 512, in f32, so that every piece has some.

    A probability is rounded to 2^-11 of itself, or to a step of 2^-25 where it is below 2^-14: the kernels hold the largest at 2^6 or more, so a
    token of 2^-26.7 stands at 2^-20.7 and is off by 2^-4.3 of itself at most, all of them alike; the rest of the bound is as above (score
    error: products of 128 terms, all but one of them 0, a top of 20)."""
    from baby_sglang_amd import _hip

    n, hq, hkv, dim = 60000, 2, 1, 128
    s = cap * math.tanh(18.5 / cap) if cap else 18.5
    ds = score_error(torch.tensor(20.0), cap, torch.tensor(s), dim).item()
    rel = 2.0**-4.3 + 2 * ds + 2.0**-21 + n * 2.0**-23
    table = torch.arange(n + ext, dtype=torch.int32, device=gpu)[None].contiguous()
    q = torch.zeros((ext, hq, dim), dtype=torch.float16, device=gpu)
    q[:, :, 0] = 1.0
    req, seq = torch.zeros(1, dtype=torch.int64, device=gpu), torch.tensor([n + ext], device=gpu)
    for decode in (False, True):
        kv = torch.zeros((n + ext, 2, hkv, dim), dtype=torch.float16, device=gpu)
        kv[:, 1] = 1.0
        few = torch.tensor([i + 5 + 16 * w for i in range(0, n - 64, 512) for w in range(4)] if decode else [n - 1], device=gpu)
        kv[few, 0, 0, 0], kv[few, 1] = 18.5, 0.0
        if decode:
            out = _hip.paged_decode_scored(q[:1], kv[:, 0], kv[:, 1], table, req, seq, scale=1.0, logit_cap=cap, out_dtype=torch.float32)
        else:
            out = _hip.paged_prefill_scored(q, kv[:, 0], kv[:, 1], table, req, seq, seq - ext, torch.tensor([ext], device=gpu), scale=1.0, logit_cap=cap,
                                            variant=2 if ext > 1 else 0)
        rows = [n + ext] if decode else [n + i + 1 for i in range(ext)]
        want = torch.tensor([(m - len(few)) / (m - len(few) + len(few) * math.exp(s)) for m in rows], dtype=torch.float64)[:, None]
        step = 0.0 if decode else 2.0**-11 * want + 2.0**-25
        assert bool(((out.double().cpu() - want).abs() <= step + rel * want).all()), (decode, (out.double().cpu() / want).aminmax())


@pytest.mark.parametrize("power", [-14, 15])
def test_f16_values_at_the_ends_of_the_type(gpu, power):
    """Probabilities that stand high in f16 do not make large values infinite, nor small ones less exact than f16 is."""
    def poison(c, row_req, row_pos, st, sp):
        c["v"][:] = (c["v"].clamp(-1.9, 1.9) * 2.0**power).to(c["v"].dtype)

    for heads, ext, pre in (("1.5b", [90, 33], [0, 70]), ("0.5b", [9, 3], [0, 700]), ("7b", [1, 2], [300, 20])):
        extend_case(gpu, heads, torch.float16, ext, pre, cap=20.0, seed=72, poison=poison)
        extend_case(gpu, heads, torch.float16, ext, pre, slopes=True, seed=73, poison=poison)


@pytest.mark.parametrize("variant", [0, 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("same_row", [False, True])
def test_weights_of_scores_that_are_all_minus_infinity(gpu, dtype, variant, same_row):
    """-inf in every visible key of kv head 0: its q heads get zeros and give no weight; those of the other kv head give theirs.  A request of
    one row and two requests of the same row (which are added up another way)."""
    from baby_sglang_amd import _hip

    c = make(74, "1.5b", dtype, [90, 300], q_rows=3)
    c["q"] = c["q"].abs() + 0.5
    c["k"][c["table"][c["req"][0], :90].long(), 0, 5] = float("-inf")
    d = to_gpu(c, gpu)
    pick = torch.tensor([0, 1, 0] if same_row else [0, 1], device=gpu)
    n = len(pick)
    old = torch.rand(d["table"].shape, device=gpu)
    w = old.clone()
    out = _hip.paged_decode_scored(d["q"][:n], d["k"], d["v"], d["table"], d["req"][pick], d["seq"][pick], token_weights=w, variant=variant).view(n, 12, 128)
    finite = {k: v.clone() for k, v in c.items() if torch.is_tensor(v)}
    finite["k"][~finite["k"].isfinite()] = 0.0
    rows = c["table"][c["req"]][pick.cpu()]
    want, mass, lse, received, top = orc.scored_exact(finite["q"][:n], finite["k"], finite["v"], rows, [c["lens"][i] for i in pick.tolist()], range(n),
                                                      [c["lens"][i] - 1 for i in pick.tolist()], 128**-0.5)
    ds = score_error(top, 0.0, lse, 128).max().item()
    expect = old.double().cpu()
    slack = torch.zeros_like(expect)
    for i, at in enumerate(pick.tolist()):
        m, r = c["lens"][at], int(c["req"][at])
        if at == 0:
            assert not bool(out[i, :6].any())
            q, k = finite["q"][i, 6:].double(), finite["k"][rows[i, :m].long()][:, 1].double()
            got = torch.softmax(q @ k.t().contiguous() * 128**-0.5, -1).sum(0)
        else:
            got = received[i]
        expect[r, :m] += got
        slack[r, :m] += got * (4 * ds + 2.0**-20 + m * 2.0**-23)
    assert bool(out.isfinite().all())
    assert bool(((w.double().cpu() - expect).abs() <= slack + 2.0**-22 * expect).all())


@pytest.mark.parametrize("heads,dtype", [("1.5b", torch.bfloat16), ("0.5b", torch.float16), ("1.5b", torch.float32)])
@pytest.mark.parametrize("what", ["k", "v", "one value"])
def test_extend_that_sees_a_nan_takes_no_longer(gpu, heads, dtype, what):
    """A NaN in the prefix, in front of every row: the rows are NaN (in its column, where it is one value) and the launch takes what it
    takes without.  20 times that and a millisecond is far from noise, and from rows computed again one by one."""
    from baby_sglang_amd import _hip

    c = make(75, heads, dtype, [4300], q_rows=300)
    d = to_gpu(c, gpu)
    args = (d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"], torch.tensor([4000], device=gpu), torch.tensor([300], device=gpu))

    def timed():
        best = float("inf")
        for _ in range(4):
            t0, t1 = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            t0.record()
            out = _hip.paged_prefill_scored(*args, logit_cap=10.0, variant=2)
            t1.record()
            torch.cuda.synchronize()
            best = min(best, t0.elapsed_time(t1))
        return out.view(300, c["hq"], c["dim"]), best

    clean, before = timed()
    slot = c["table"][c["req"][0], 5].long().item()
    if what == "one value":
        d["v"][slot, :, 3] = float("nan")
    else:
        d[what][slot] = float("nan")
    got, after = timed()
    if what == "one value":
        assert bool(got[:, :, 3].isnan().all())
        rest = [i for i in range(c["dim"]) if i != 3]
        assert torch.equal(got[:, :, rest], clean[:, :, rest])
    else:
        assert bool(got.isnan().all())
    assert after <= 20 * before + 1.0, (before, after)


@pytest.mark.parametrize("heads,dtype", [("1.5b", torch.bfloat16), ("0.5b", torch.float16), ("7b", torch.float32), ("one", torch.bfloat16)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("at", [0, 31, 32, 100, 149, 205, 299])
def test_extend_rows_around_a_value_that_is_no_number(gpu, heads, dtype, bad, at):
    """One such value: causal rows before it, and the rows of windows that have left it behind, are right to the bit of their own sums; who sees it
    has it in that column and nowhere else."""
    from baby_sglang_amd import _hip

    n = 300
    c = make(76, heads, dtype, [n], q_rows=n)
    start, stop = [max(0, i - 120) for i in range(n)], [i + 1 for i in range(n)]
    st, sp = (torch.tensor(x, dtype=torch.int32) for x in (start, stop))
    slot = c["table"][c["req"][0], at].long()
    finite = {k: (v.clone() if torch.is_tensor(v) else v) for k, v in c.items()}
    c["v"][slot, :, 7] = bad
    d = to_gpu(c, gpu)
    out = _hip.paged_prefill_scored(d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"], torch.zeros(1, dtype=torch.int64, device=gpu), d["seq"], logit_cap=9.0,
                                    visible_from=st.to(gpu), visible_to=sp.to(gpu), variant=2).view(n, c["hq"], c["dim"]).cpu()
    sees = torch.tensor([a <= at < b for a, b in zip(start, stop)])
    assert bool((out[sees][:, :, 7].isnan() if bad != bad else out[sees][:, :, 7].isinf()).all())
    want, mass, lse, _, top = orc.scored_exact(finite["q"], finite["k"], finite["v"], finite["table"][finite["req"]], [n], [0] * n, range(n), c["dim"] ** -0.5, 9.0,
                                               None, st, sp)
    u_p = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 0.0}[dtype]
    keep = torch.ones(c["dim"], dtype=torch.bool)
    keep[7] = False
    check_rows(out[:, :, keep], want[:, :, keep], mass[:, :, keep], lse, top, 9.0, dtype, dtype, u_p, n, 6.0, c["dim"])
    check_rows(out[~sees], want[~sees], mass[~sees], lse[~sees], top[~sees], 9.0, dtype, dtype, u_p, n, 6.0, c["dim"])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n_splits,variant", [(3, 0), (7, 0x200), (3, 1), (64, 0)])
def test_decode_infinite_values_in_every_piece(gpu, dtype, n_splits, variant):
    """An infinite value shows in its column and nowhere else, whichever piece of the request it is in: the pieces that a merge reads twice to
    fill a round among them.  Where every probability meets the values once, as a positive number, the column is infinite; as the
    sum of two (bf16), or by the generic kernel, it may be NaN."""
    from baby_sglang_amd import _hip

    lens = [900, 40, 2000]
    for at in (0, 450, 899):
        c = make(77, "1.5b", dtype, lens)
        c["v"][c["table"][c["req"][0], at].long(), :, 7] = float("inf")
        d = to_gpu(c, gpu)
        out = _hip.paged_decode_scored(d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"], logit_cap=5.0, n_splits=n_splits, variant=variant).view(3, 12, 128)
        once = dtype != torch.bfloat16 and variant != 1
        assert bool((out[0, :, 7] == float("inf")).all() if once else (~out[0, :, 7].isfinite()).all())
        out[0, :, 7] = 0.0
        assert bool(out.isfinite().all())


@pytest.mark.parametrize("heads,dtype", [("7b", torch.bfloat16), ("7b", torch.float32)])
def test_extend_list_taken_over_from_a_call_of_another_path(gpu, heads, dtype):
    """Layers of one batch that differ in their cap, with a scale that only the generic kernel takes without one (16 bits): the list that the first
    call left is right for the second, sorted or not, either way round."""
    from baby_sglang_amd import _hip

    r = random.Random(9)
    ext = [r.randint(60, 300) for _ in range(31)]  # (with the end of the sums on a border of the workspace's parts: 31 + 1 entries of 8 bytes)
    pre = [r.randint(0, 300) for _ in ext]
    c = make(78, heads, dtype, [a + b for a, b in zip(ext, pre)], q_rows=sum(ext))
    d = to_gpu(c, gpu)
    args = (d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"], torch.tensor(pre, device=gpu), torch.tensor(ext, device=gpu))
    ws = torch.empty(_hip.prefill_workspace_bytes(len(ext), sum(ext), c["hq"], c["dim"]), dtype=torch.uint8, device=gpu)
    generic = dict(scale=-0.09) if dtype != torch.float32 else dict(scale=0.09)
    forms = [dict(generic, logit_cap=0.0), dict(generic, logit_cap=10.0), dict(generic, logit_cap=30.0)]
    want = [_hip.paged_prefill_scored(*args, **kw) for kw in forms]
    for first, *later in ((0, 1, 2, 0, 1), (1, 0, 1, 2), (2, 2, 1)):
        assert torch.equal(_hip.paged_prefill_scored(*args, workspace=ws, **forms[first]), want[first])
        for i in later:
            assert torch.equal(_hip.paged_prefill_scored(*args, workspace=ws, list_ready=True, **forms[i]), want[i]), (first, i)


def test_f32_of_16_heads_per_kv_head_everywhere(gpu):
    """The sizes that the tests above leave out for it: f32 takes up to 16 q heads per kv head in every form."""
    decode_case(gpu, "one", torch.float32, [1, 2, 15, 16, 17, 300, 33, 64], cap=8.0, slopes=True)
    for ext, prefix in (([3, 1, 0, 17, 40], [0, 5, 9, 33, 600]), ([130, 64, 1, 200], [0, 31, 70, 513])):
        extend_case(gpu, "one", torch.float32, ext, prefix, cap=8.0, slopes=True, only=60)
    for ext, prefix, kind in (([1], [0], None), ([1], [2500], None), ([3, 0, 2], [700, 9, 0], "both"), ([7, 11], [1300, 40], "document"),
                              ([5, 9, 20], [0, 600, 33], "wild"), ([8], [4000], "prefix")):
        extend_case(gpu, "one", torch.float32, ext, prefix, cap=20.0, slopes=True, kind=kind, seed=36, extra_rows=3)


@pytest.mark.parametrize("heads", ["1.5b", "0.5b", "7b"])
def test_decode_f32_is_as_exact_as_f32_is(gpu, heads):
    """The results' distance from the definition, beside that of elementary operations in 32 bits (products, exp, sums by torch on the same
    tensors): both round some 130 times on the way to a score, so neither should be far ahead; 1.35 times is allowed."""
    from baby_sglang_amd import _hip

    lens = [300, 900, 555, 731, 402, 618, 850, 333]
    c = make(79, heads, torch.float32, lens, q_scale=3.0)
    d = to_gpu(c, gpu)
    hq, hkv, dim = c["hq"], c["hkv"], c["dim"]
    got = _hip.paged_decode_scored(d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"]).view(len(lens), hq, dim).double()
    kernel = plain = 0.0
    for i, n in enumerate(lens):
        slots = d["table"][d["req"][i], :n].long()
        k, v = d["k"][slots].transpose(0, 1).contiguous(), d["v"][slots].transpose(0, 1).contiguous()  # [Hkv, n, D]
        q = d["q"][i].view(hkv, hq // hkv, dim)
        outs = []
        for t in (torch.float64, torch.float32):
            s = torch.matmul(q.to(t), k.to(t).transpose(1, 2).contiguous()) * dim**-0.5
            p = torch.exp(s - s.amax(-1, keepdim=True))
            outs.append((torch.matmul(p, v.to(t)) / p.sum(-1, keepdim=True)).reshape(hq, dim).double())
        kernel += (got[i] - outs[0]).square().sum().item()
        plain += (outs[1] - outs[0]).square().sum().item()
    assert kernel <= 1.35**2 * plain, (kernel / plain) ** 0.5


@pytest.mark.parametrize("heads,dtype", [("1.5b", torch.bfloat16), ("0.5b", torch.float16), ("one", torch.float16), ("1.5b", torch.float32)])
@pytest.mark.parametrize("ext", [[150, 70], [9, 20]])
@pytest.mark.parametrize("cap,slopes", [(0.0, False), (0.0, True), (900.0, False), (900.0, True)])
def test_extend_scores_that_rise_away_from_the_row(gpu, heads, dtype, ext, cap, slopes):
    """Keys that grow by leaps with the distance: scores exceed all before them by 2^3 to 2^1000 of probability inside steps that every row sees
    whole, where nobody looks for a maximum beforehand; and fall back again."""
    def poison(c, row_req, row_pos, st, sp):
        for r, n in zip(c["req"].tolist(), c["lens"]):
            for lo, hi, by in ((600, 700, 1.5), (400, 520, 4.0), (330, 331, 12.0), (200, 280, 25.0), (100, 101, 60.0), (10, 40, 0.1)):
                slots = c["table"][r, lo : min(hi, n)].long()
                c["k"][slots] = (c["k"][slots].float() * by).to(dtype)

    extend_case(gpu, heads, dtype, ext, [700, 640], cap=cap, slopes=slopes, seed=80, poison=poison, variant=2, only=60)
    extend_case(gpu, heads, dtype, ext, [700, 640], cap=cap, slopes=slopes, kind="document", seed=81, poison=poison, variant=2, only=60)
