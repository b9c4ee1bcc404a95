"""The fast way into the small calls (csrc/fast_calls.cpp): it is taken for the ordinary case, left alone otherwise, and the wrappers
give the same results without it."""
import pytest
import torch

import test_gpu_evict as ev
import test_gpu_logit_controls as lg
import test_gpu_scored_attention as sa

pytestmark = pytest.mark.gpu


class Spy:
    def __init__(self, real):
        self.real, self.taken, self.left = real, 0, 0

    def __getattr__(self, name):
        fn = getattr(self.real, name)

        def call(*a):
            rc = fn(*a)
            self.taken += rc is not None
            self.left += rc is None
            return rc

        return call


def run_some(gpu):
    out = [sa.decode_case(gpu, "1.5b", torch.bfloat16, [200, 1, 777], cap=5.0, slopes=True, start=[3, 0, 20], seed=7)]
    out.append(sa.decode_case(gpu, "0.5b", torch.float32, [20, 33], weights=False, seed=8))
    ev.case(gpu, [500, 400, 90], 100, recent=7, sinks=2, seed=7)
    ev.case(gpu, [500, 400, 90], 100, in_place=False, width=12, seed=8)
    lg.case(gpu, 3, 9001, torch.bfloat16, seed=5, hist=37, bias=9, mask=0.5)
    lg.case(gpu, 3, 4096, torch.float32, seed=6, hist=37, scalars=True, in_place=True)
    return out


def test_same_results_with_and_without(gpu, monkeypatch):
    from baby_sglang_amd import _hip

    assert _hip._fast is not None, "build baby-sglang_amd/_fast_calls.so (make -C baby-sglang_amd/csrc)"
    with_it = run_some(gpu)
    monkeypatch.setattr(_hip, "_fast", None)
    for a, b in zip(with_it, run_some(gpu)):
        assert torch.equal(a, b)


def test_what_it_takes_and_what_it_leaves(gpu, monkeypatch):
    from baby_sglang_amd import _hip

    spy = Spy(_hip._fast)
    monkeypatch.setattr(_hip, "_fast", spy)
    d = sa.to_gpu(sa.make(9, "1.5b", torch.bfloat16, [30, 500]), gpu)
    args = (d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"])
    ws = _hip.new_decode_workspace(_hip.decode_scored_workspace_bytes(2, 12, 128, 4, d["table"].shape[1], True), gpu)
    kn = torch.randn(2, 4, 128, device=gpu).to(torch.bfloat16)
    loc = torch.stack([d["table"][d["req"][i], n - 1] for i, n in enumerate((30, 500))])
    w = torch.zeros(d["table"].shape, device=gpu)

    def taken(fn, yes):
        before = spy.taken
        fn()
        assert (spy.taken - before == 1) is yes

    scored = _hip.paged_decode_scored
    taken(lambda: scored(*args, n_splits=4, workspace=ws, logit_cap=3, token_weights=w, k_new=kn[:, :2], v_new=kn[:, 2:], out_cache_loc=loc, fuse_kv_write=True), True)
    assert torch.equal(d["k"][loc.long()], kn[:, :2]) and torch.equal(d["v"][loc.long()], kn[:, 2:])
    taken(lambda: scored(*args, n_splits=4, workspace=ws[:100]), False)  # too small: the wrapper makes one
    taken(lambda: scored(*args, workspace=ws), False)  # splits to be found
    taken(lambda: scored(*args[:4], d["req"].int(), d["seq"], n_splits=4, workspace=ws), False)  # to be converted
    taken(lambda: scored(*args, n_splits=4, workspace=ws, visible_from=torch.zeros(2, dtype=torch.int64, device=gpu)), False)
    taken(lambda: scored(d["q"].transpose(0, 1).contiguous().transpose(0, 1), *args[1:], n_splits=4, workspace=ws), False)
    ext = torch.tensor([1, 3], device=gpu)
    q4 = torch.randn(4, 12, 128, device=gpu).to(torch.bfloat16)
    pre = (q4, *args[1:], d["seq"] - ext, ext)
    pws = torch.empty(_hip.prefill_workspace_bytes(2, 4, 12, 128), dtype=torch.uint8, device=gpu)
    taken(lambda: _hip.paged_prefill_scored(*pre, workspace=pws, logit_cap=4.0), True)
    taken(lambda: _hip.paged_prefill_scored(*pre, logit_cap=4.0), False)
    taken(lambda: _hip.paged_prefill_scored(*pre[:-1], ext.int(), workspace=pws), False)
    a = _hip.paged_prefill_scored(*pre, workspace=pws, logit_cap=4.0, visible_to=torch.tensor([9, 9, 0, 400], dtype=torch.int32, device=gpu))
    b = _hip.paged_prefill_scored(*pre, logit_cap=4.0, visible_to=torch.tensor([9, 9, 0, 400], dtype=torch.int32, device=gpu))
    assert torch.equal(a, b)
    x, h, n = torch.zeros(2, 64, device=gpu), torch.zeros(2, 4, dtype=torch.int32, device=gpu), torch.tensor([1, 2], device=gpu)
    taken(lambda: _hip.logit_controls(x, history=h, history_lens=n, repetition=torch.full((2,), 1.5, device=gpu)), True)
    taken(lambda: _hip.logit_controls(x, history=h, history_lens=n, repetition=1.5), False)
    taken(lambda: _hip.logit_controls(x, history=h[:, :0], history_lens=n), False)
    table, weights = torch.zeros(3, 64, dtype=torch.int32, device=gpu), torch.zeros(3, 64, device=gpu)
    new, gone = torch.zeros(2, dtype=torch.int64, device=gpu), torch.zeros((2, 9), dtype=torch.int32, device=gpu)
    taken(lambda: _hip.evict_tokens(table, weights, d["req"][:2] * 0 + n - 1, n * 20, 8, evicted=gone, new_lens=new), True)
    taken(lambda: _hip.evict_tokens(table, weights, n - 1, n * 20, 8), False)  # results to be made
    for fn in (lambda: scored(*args, n_splits=4, workspace=ws, logit_cap=1e9), lambda: _hip.evict_tokens(table, weights, n - 1, n, 8, recent=9, evicted=gone, new_lens=new),
               lambda: _hip.logit_controls(x, token_mask=h[:, :1]),
               lambda: _hip.paged_prefill_scored(*pre, workspace=pws, logit_cap=-1.0)):
        with pytest.raises(ValueError):
            fn()


def test_on_a_stream_of_its_own_and_captured(gpu):
    from baby_sglang_amd import _hip

    x = torch.randn(4, 5000, device=gpu)
    mask = torch.randint(-(2**31), 2**31 - 1, (4, 157), dtype=torch.int32, device=gpu)
    out = torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _hip.logit_controls(x, token_mask=mask, out=out)
    side.synchronize()
    assert torch.equal(out, _hip.logit_controls(x, token_mask=mask))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _hip.logit_controls(x, token_mask=mask, out=out)
    for _ in range(3):
        x.mul_(-1.5)
        out.zero_()
        eager = _hip.logit_controls(x, token_mask=mask)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


SLOW = """
#include <unistd.h>
int slow(void) { usleep(400000); return 0; }
"""


def test_other_threads_run_while_a_call_waits(gpu, monkeypatch, tmp_path):
    """A launch that has to wait (here: a function of 0.4 s in an entry point's place) does not stop the process's other threads."""
    import ctypes
    import subprocess
    import threading
    import time

    from baby_sglang_amd import _hip

    src, so = tmp_path / "slow.c", tmp_path / "slow.so"
    src.write_text(SLOW)
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-o", str(so), str(src)])
    slow = ctypes.CDLL(str(so))
    d = sa.to_gpu(sa.make(9, "1.5b", torch.bfloat16, [30, 500]), gpu)
    args = (d["q"], d["k"], d["v"], d["table"], d["req"], d["seq"])
    ws = _hip.new_decode_workspace(_hip.decode_scored_workspace_bytes(2, 12, 128, 4, d["table"].shape[1], True), gpu)
    ext = torch.tensor([1, 1], device=gpu)
    pws = torch.empty(_hip.prefill_workspace_bytes(2, 2, 12, 128), dtype=torch.uint8, device=gpu)
    x, mask = torch.zeros(2, 64, device=gpu), torch.zeros(2, 2, dtype=torch.int32, device=gpu)
    table, weights = torch.zeros(3, 64, dtype=torch.int32, device=gpu), torch.zeros(3, 64, device=gpu)
    new, gone = torch.zeros(2, dtype=torch.int64, device=gpu), torch.zeros((2, 9), dtype=torch.int32, device=gpu)
    calls = (lambda: _hip.paged_decode_scored(*args, n_splits=4, workspace=ws), lambda: _hip.paged_prefill_scored(*args, d["seq"] - ext, ext, workspace=pws),
             lambda: _hip.evict_tokens(table, weights, ext, ext, 8, evicted=gone, new_lens=new), lambda: _hip.logit_controls(x, token_mask=mask))
    for call in calls:
        call()
    try:
        _hip.bind_fast_calls({name: slow.slow for name in ("bsgl_paged_decode_scored", "bsgl_evict_tokens", "bsgl_logit_controls", "bsgl_paged_prefill_scored")})
        for call in calls:
            worker = threading.Thread(target=call)
            t0, gap = time.perf_counter(), 0.0
            worker.start()
            while worker.is_alive():
                t1 = time.perf_counter()
                time.sleep(0.002)
                gap = max(gap, time.perf_counter() - t1)
            assert time.perf_counter() - t0 > 0.3  # (the stand-in was called)
            assert gap < 0.2, gap
    finally:
        _hip.bind_fast_calls()
