"""Eviction by accumulated weight against a plain sort: everything is exact."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def plain(table, weights, req, lens, budget, recent, sinks, width, out_table, out_weights):
    """Per request: the stable descending sort of the middle decides (torch puts NaN first, as the kernel does)."""
    gone = torch.full((len(lens), width), -1, dtype=torch.int32)
    for i, n in enumerate(lens):
        r = int(req[i])
        if r in [int(x) for x in req[:i]]:
            continue
        stay = torch.ones(n, dtype=torch.bool)
        if n > budget:
            mid = weights[r, sinks : n - recent]
            order = torch.sort(mid + 0.0, descending=True, stable=True).indices
            stay[sinks + order[budget - sinks - recent :]] = False
            left = table[r, :n][~stay][:width]
            gone[i, : len(left)] = left
        m = int(stay.sum())
        kept_t, kept_w = table[r, :n][stay].clone(), weights[r, :n][stay].clone()
        out_table[r, :m], out_weights[r, :m] = kept_t, kept_w
    return torch.tensor([min(n, budget) for n in lens]), gone


def case(gpu, lens, budget, recent=0, sinks=0, seed=0, weights=None, in_place=True, width=None, pad=9, row_pad=0, offset=0, max_seq_len=0, rows=None):
    from baby_sglang_amd import _hip

    g = torch.Generator().manual_seed(seed)
    cols = max(max(lens) + pad, 1)
    n_rows = len(lens) + 3
    req = torch.randperm(n_rows, generator=g)[: len(lens)] if rows is None else torch.tensor(rows)
    table = torch.randint(0, 1 << 30, (n_rows, cols), generator=g, dtype=torch.int32)
    w = torch.exp(2 * torch.randn(n_rows, cols, generator=g)) * (torch.rand(n_rows, cols, generator=g) > 0.2)
    if weights is not None:
        w = weights(w, g)
    want_t, want_w = (table.clone(), w.clone()) if in_place else (torch.full_like(table, -5), torch.full_like(w, -5.0))
    wid = max(0, cols - budget) if width is None else width
    new_lens, gone = plain(table, w, req, lens, budget, recent, sinks, wid, want_t, want_w)

    def place(t):  # on the GPU, with the row stride and the start asked for
        base = torch.zeros(n_rows * (cols + row_pad) + offset, dtype=t.dtype, device=gpu)
        view = base[offset:].view(n_rows, cols + row_pad)[:, :cols]
        view.copy_(t)
        return view

    dt, dw = place(table), place(w)
    kw = {}
    if not in_place:
        kw = dict(out_table=place(torch.full_like(table, -5)), out_weights=place(torch.full_like(w, -5.0)))
    if width is not None:
        kw["evicted"] = torch.zeros((len(lens), width), dtype=torch.int32, device=gpu)
    got_lens, got_gone = _hip.evict_tokens(dt, dw, req.to(gpu), torch.tensor(lens, device=gpu), budget, recent, sinks, max_seq_len=max_seq_len, **kw)
    torch.cuda.synchronize()
    if width is None and max_seq_len:
        gone = gone[:, : got_gone.shape[1]]
    assert torch.equal(got_lens.cpu(), new_lens)
    assert torch.equal(got_gone.cpu(), gone)
    ot, ow = kw.get("out_table", dt), kw.get("out_weights", dw)
    assert torch.equal(ot.cpu(), want_t)
    assert torch.equal(ow.cpu().view(torch.int32), want_w.view(torch.int32))


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("lens,budget,recent,sinks", [
    ([1, 0, 2, 5, 9], 4, 0, 0), ([1, 0, 2, 5, 9], 4, 2, 2), ([7], 1, 0, 0), ([7], 1, 1, 0), ([7], 1, 0, 1), ([300, 261, 256, 255], 256, 32, 4),
    ([1024, 1023, 1025], 1000, 100, 7), ([4096, 2500, 4095], 2048, 256, 4), ([2000] * 40, 3, 1, 1), ([16384, 16383], 9000, 0, 0),
    ([16385, 20000, 33000], 9000, 1000, 4), ([70001], 69999, 3, 3), ([131072], 100, 0, 4), ([900, 1100], 1, 0, 0)])
def test_sizes(gpu, lens, budget, recent, sinks, in_place):
    case(gpu, lens, budget, recent, sinks, seed=len(lens) + budget, in_place=in_place)


def _special(w, g):
    w = torch.round(w)  # many ties
    for r in range(w.shape[0]):
        idx = torch.randint(0, w.shape[1], (8,), generator=g)
        w[r, idx] = torch.tensor([float("nan"), float("inf"), float("-inf"), -0.0, torch.finfo(torch.float32).min, torch.finfo(torch.float32).max,
                                  1e-40, -1.5])
    return w


@pytest.mark.parametrize("lens", [[50, 200, 1000], [5000, 3000], [40000]])
@pytest.mark.parametrize("make", [lambda w, g: torch.zeros_like(w), lambda w, g: torch.full_like(w, 3.0), _special,
                                  lambda w, g: torch.full_like(w, float("nan")), lambda w, g: -w, lambda w, g: (torch.rand(w.shape, generator=g) > 0.5).float(),
                                  lambda w, g: w * 0 + torch.arange(w.shape[1]).float(), lambda w, g: w * 0 - torch.arange(w.shape[1]).float()])
def test_ties_and_special_values(gpu, lens, make):
    case(gpu, lens, max(8, min(lens) // 3), recent=3, sinks=2, seed=5, weights=make)


@pytest.mark.parametrize("kw", [dict(width=0), dict(width=1), dict(width=7), dict(width=5000), dict(row_pad=3), dict(offset=1), dict(offset=3, row_pad=1),
                                dict(max_seq_len=700), dict(max_seq_len=10), dict(pad=0)])
def test_layouts_and_hints(gpu, kw):
    if kw.get("max_seq_len") == 10:  # a hint that is wrong costs the tail of `evicted`, whose width it sets, and nothing else
        kw = dict(kw, width=600)
    case(gpu, [700, 650, 64, 333], 100, recent=20, sinks=4, seed=6, **kw)


def test_a_row_named_twice_is_compacted_once(gpu):
    case(gpu, [500, 400, 500, 90], 100, seed=7, rows=[2, 0, 2, 1])


def test_random(gpu):
    r = random.Random(1)
    for seed in range(40):
        n = r.randint(1, 12)
        top = r.choice([3, 64, 500, 1500, 20000])
        lens = [r.randint(0, top) for _ in range(n)]
        budget = r.randint(1, top + 1)
        recent = r.randint(0, budget)
        case(gpu, lens, budget, recent, r.randint(0, budget - recent), seed=seed, in_place=r.random() < 0.5)


def test_graph_replays(gpu):
    """Captured in place: every replay compacts what the table then holds."""
    from baby_sglang_amd import _hip

    table = torch.arange(3 * 600, dtype=torch.int32, device=gpu).view(3, 600).contiguous()
    w = torch.rand(3, 600, device=gpu)
    req, lens = torch.tensor([2, 0], device=gpu), torch.tensor([600, 431], device=gpu)
    new_lens, gone = torch.zeros(2, dtype=torch.int64, device=gpu), torch.zeros((2, 600), dtype=torch.int32, device=gpu)
    t0, w0 = table.clone(), w.clone()

    def call(t, x):
        return _hip.evict_tokens(t, x, req, lens, 200, recent=10, sinks=1, new_lens=new_lens, evicted=gone)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(table.clone(), w.clone())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(table, w)
    for i in range(3):
        table.copy_(t0)
        w.copy_(w0 * (i + 1) + i)
        et, ew = table.clone(), w.clone()
        want = [x.clone() for x in call(et, ew)]
        gone.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(table, et) and torch.equal(w, ew) and torch.equal(gone, want[1]) and torch.equal(new_lens, want[0])


def test_refusals(gpu):
    from baby_sglang_amd import _hip

    t, w = torch.zeros(4, 32, dtype=torch.int32, device=gpu), torch.zeros(4, 32, device=gpu)
    req, lens = torch.tensor([0, 1], device=gpu), torch.tensor([30, 3], device=gpu)
    for args, kw in [((t, w, req, lens, 0), {}), ((t, w, req, lens, 4), dict(recent=3, sinks=2)), ((t, w, req, lens, 4), dict(recent=-1)),
                     ((t.long(), w, req, lens, 4), {}), ((t, w.double(), req, lens, 4), {}), ((t, w[:, :31], req, lens, 4), {}),
                     ((t, w, req, lens[:1], 4), {}), ((t, w, req, lens, 4), dict(out_table=torch.zeros(4, 31, dtype=torch.int32, device=gpu))),
                     ((t, w, req, lens, 4), dict(evicted=torch.zeros(1, 3, dtype=torch.int32, device=gpu))),
                     ((t, w, req, lens, 4), dict(new_lens=torch.zeros(2, dtype=torch.int32, device=gpu)))]:
        with pytest.raises(ValueError):
            _hip.evict_tokens(*args, **kw)
    with pytest.raises(RuntimeError):
        _hip.evict_tokens(t.cpu(), w, req, lens, 4)
    got, gone = _hip.evict_tokens(t, w, req[:0], lens[:0], 4)
    assert got.shape == (0,) and gone.shape == (0, 28)


def test_long_rows_in_a_graph_and_on_two_streams(gpu):
    """The form over several workgroups: replays with a workspace of their own, and two calls at once on two streams."""
    from baby_sglang_amd import _hip

    g = torch.Generator().manual_seed(9)
    cols, budget = 40000, 9000
    t0 = torch.randint(0, 1 << 30, (2, cols), generator=g, dtype=torch.int32).to(gpu)
    w0 = torch.rand(2, cols, generator=g).to(gpu)
    req, lens = torch.tensor([1, 0], device=gpu), torch.tensor([39999, 25000], device=gpu)
    ws = [torch.empty(_hip.evict_workspace_bytes(2, cols, budget), dtype=torch.uint8, device=gpu) for _ in range(2)]
    table, w = t0.clone(), w0.clone()
    new_lens, gone = torch.zeros(2, dtype=torch.int64, device=gpu), torch.zeros((2, cols - budget), dtype=torch.int32, device=gpu)

    def call(t, x, ws, **kw):
        return _hip.evict_tokens(t, x, req, lens, budget, recent=100, sinks=4, workspace=ws, **kw)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(t0.clone(), w0.clone(), ws[0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(table, w, ws[0], new_lens=new_lens, evicted=gone)
    for i in range(3):
        table.copy_(t0)
        w.copy_((w0 * (i + 1)).frac())
        et, ew = table.clone(), w.clone()
        want = call(et, ew, None)
        gone.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(table, et) and torch.equal(w, ew) and torch.equal(gone, want[1]) and torch.equal(new_lens, want[0])
    pairs = [(t0.clone(), w0.clone()) for _ in range(2)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(*pairs[0], ws[0])
    call(*pairs[1], ws[1])
    torch.cuda.synchronize()
    assert torch.equal(pairs[0][0], pairs[1][0]) and torch.equal(pairs[0][1], pairs[1][1])


def test_new_lengths_over_the_old_ones_are_refused(gpu):
    from baby_sglang_amd import _hip

    t, w = torch.zeros(4, 32, dtype=torch.int32, device=gpu), torch.zeros(4, 32, device=gpu)
    lens = torch.tensor([30, 3], device=gpu)
    with pytest.raises(ValueError, match="overlap"):
        _hip.evict_tokens(t, w, torch.tensor([0, 1], device=gpu), lens, 4, new_lens=lens)


def test_evicted_rows_that_share_memory_are_refused(gpu):
    """Through the fast way as well, which leaves such a tensor to the wrapper."""
    from baby_sglang_amd import _hip

    t, w = torch.zeros(4, 32, dtype=torch.int32, device=gpu), torch.zeros(4, 32, device=gpu)
    req, lens = torch.tensor([0, 1, 2], device=gpu), torch.tensor([30, 3, 20], device=gpu)
    one, new = torch.empty(7, dtype=torch.int32, device=gpu), torch.zeros(3, dtype=torch.int64, device=gpu)
    for bad in (one.expand(3, 7), torch.as_strided(one, (3, 3), (2, 1))):
        for kw in ({}, dict(new_lens=new)):
            with pytest.raises(ValueError, match="evicted"):
                _hip.evict_tokens(t, w, req, lens, 4, evicted=bad, **kw)
