"""Refusals and host arithmetic of the scored attention, eviction and logit entry points (CPU only: every one of
them is answered before anything would be launched)."""
import ctypes

import pytest
import torch

from baby_sglang_amd import _hip

lib = _hip.lib
P = ctypes.c_void_p(256)  # a pointer that a refused call never follows


def mods(**kw):
    m = _hip.ScoreMods()
    for k, v in kw.items():
        setattr(m, k, v)
    return ctypes.byref(m)


def decode_call(**kw):
    c = _hip.DecodeCall()
    d = dict(out=256, out_row_stride=1536, q=256, q_row_stride=1536, k_slab=256, v_slab=256, slab_row_stride=512, n_slots=9, req_to_token=256,
             table_row_stride=64, table_rows=2, table_cols=64, req_pool_indices=256, seq_lens=256, batch=2, n_q_heads=12, n_kv_heads=2,
             head_dim=128, scale=0.1, n_splits=1)
    d.update(kw)
    for k, v in d.items():
        setattr(c, k, v)
    return ctypes.byref(c)


def test_scored_decode_refusals():
    f = lib.bsgl_paged_decode_scored
    assert f(None, mods()) == _hip.BSGL_ERR_BAD_ARG and f(decode_call(), None) == _hip.BSGL_ERR_BAD_ARG
    for cap in (-1.0, float("nan"), float("inf")):
        assert f(decode_call(), mods(logit_cap=cap)) == _hip.BSGL_ERR_BAD_ARG and b"logit_cap" in lib.bsgl_last_error()
    assert f(decode_call(), mods(token_weights=256)) == _hip.BSGL_ERR_BAD_ARG
    assert f(decode_call(), mods(token_weights=256, token_weights_out=256, weights_row_stride=63)) == _hip.BSGL_ERR_BAD_ARG
    assert f(decode_call(), mods(token_weights=256, token_weights_out=256, weights_row_stride=64)) == _hip.BSGL_ERR_WORKSPACE
    assert f(decode_call(n_splits=65), mods()) == _hip.BSGL_ERR_BAD_ARG
    assert f(decode_call(q=None), mods()) == _hip.BSGL_ERR_BAD_ARG
    assert f(decode_call(dtype=7, out_dtype=7), mods()) == _hip.BSGL_ERR_UNSUPPORTED
    assert f(decode_call(batch=0), mods(logit_cap=1.0)) == _hip.BSGL_OK  # nothing to do


def test_scored_caps_out_of_range():
    for cap in (1e-9, 2.0**-21, 16385.0, 1e30):
        assert lib.bsgl_paged_decode_scored(decode_call(), mods(logit_cap=cap)) == _hip.BSGL_ERR_BAD_ARG and b"logit_cap" in lib.bsgl_last_error()
    big = decode_call(batch=65536)
    assert lib.bsgl_paged_decode_scored(big, mods(token_weights=256, token_weights_out=256, weights_row_stride=64)) == _hip.BSGL_ERR_UNSUPPORTED


def test_evict_lengths_must_not_overlap():
    def f(seq, new, batch=4, cols=64):
        return lib.bsgl_evict_tokens(P, P, P, cols, P, cols, 2, cols, P, ctypes.c_void_p(seq), ctypes.c_void_p(new), None, 0, 0, batch, 4, 0, 0, 0, None, 0, None)

    for new in (4096, 4096 - 24, 4096 + 24):
        assert f(4096, new) == _hip.BSGL_ERR_BAD_ARG and b"overlap" in lib.bsgl_last_error()
    assert f(4096, 8192, cols=2**31 - 5) == _hip.BSGL_ERR_BAD_ARG


def test_logits_in_place_keep_their_stride():
    c = _hip.LogitCall()
    for k, v in dict(out=256, logits=256, out_row_stride=100, logits_row_stride=104, batch=2, vocab=100, dtype=2).items():
        setattr(c, k, v)
    assert lib.bsgl_logit_controls(ctypes.byref(c)) == _hip.BSGL_ERR_BAD_ARG


def test_scored_decode_workspace():
    plain = _hip.decode_workspace_bytes(4, 12, 128, 32)  # (up to four times the splits for a long request)
    assert _hip.decode_scored_workspace_bytes(4, 12, 128, 8, 1000, False) == plain
    with_weights = _hip.decode_scored_workspace_bytes(4, 12, 128, 8, 1000, True)
    assert with_weights >= plain + 4 * 12 * (1 + 1008) * 4
    # the ticket area stays free of scores where the decode itself needs no workspace
    assert _hip.decode_workspace_bytes(4, 12, 128, 1) == 0
    assert _hip.decode_scored_workspace_bytes(4, 12, 128, 1, 1000, True) >= lib.bsgl_decode_counter_bytes() + 4 * 12 * 1008 * 4


def test_evict_refusals():
    def f(budget=4, recent=1, sinks=1, rows=2, cols=64, ts=64, ws=64, es=8, ec=8, batch=2, table=P):
        return lib.bsgl_evict_tokens(P, P, table, ts, P, ws, rows, cols, P, P, P, P, es, ec, batch, budget, recent, sinks, 0, None, 0, None)

    for kw in (dict(budget=0), dict(budget=-1), dict(recent=-1), dict(sinks=-1), dict(budget=4, recent=2, sinks=3), dict(recent=2**31 - 1, sinks=2),
               dict(rows=0), dict(cols=0), dict(cols=2**31, ts=2**31, ws=2**31), dict(ts=63), dict(ws=63), dict(es=7), dict(ec=-1), dict(batch=-1), dict(table=None)):
        assert f(**kw) == _hip.BSGL_ERR_BAD_ARG, kw
    assert f(batch=0) == _hip.BSGL_OK


def test_logit_refusals():
    def f(**kw):
        c = _hip.LogitCall()
        d = dict(out=256, logits=256, out_row_stride=100, logits_row_stride=100, batch=2, vocab=100, dtype=2)
        d.update(kw)
        for k, v in d.items():
            setattr(c, k, v)
        return lib.bsgl_logit_controls(ctypes.byref(c))

    hist = dict(history=256, history_row_stride=10, history_n_rows=2, history_cols=10, history_lens=256)
    for kw in (dict(out=None), dict(logits=None), dict(out_row_stride=99), dict(logits_row_stride=99), dict(batch=-1), dict(vocab=-1), dict(n_bias=-1),
               dict(n_bias=3), dict(n_bias=3, bias_ids=256, bias_values=256, bias_row_stride=2), dict(repetition=256),
               dict(hist, history_lens=None), dict(hist, history_n_rows=1), dict(hist, history_n_rows=0), dict(hist, history_row_stride=9),
               dict(token_mask=256, mask_n_rows=2, mask_row_stride=3), dict(token_mask=256, mask_n_rows=0, mask_row_stride=4)):
        assert f(**kw) == _hip.BSGL_ERR_BAD_ARG, kw
    assert f(history=256, history_row_stride=1 << 18, history_n_rows=2, history_cols=1 << 18, history_lens=256) == _hip.BSGL_ERR_UNSUPPORTED
    assert f(n_bias=4097, bias_ids=256, bias_values=256, bias_row_stride=4097) == _hip.BSGL_ERR_UNSUPPORTED
    assert f(dtype=5) == _hip.BSGL_ERR_UNSUPPORTED and f(batch=65536) == _hip.BSGL_ERR_UNSUPPORTED
    assert f(batch=0, out=None) == _hip.BSGL_OK and f(vocab=0, out=None) == _hip.BSGL_OK
    assert lib.bsgl_logit_controls(None) == _hip.BSGL_ERR_BAD_ARG


def test_tensors_off_the_gpu_are_refused():
    q = torch.zeros(1, 12, 128, dtype=torch.bfloat16)
    slab = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    table, one = torch.zeros(1, 8, dtype=torch.int32), torch.ones(1, dtype=torch.int64)
    with pytest.raises(RuntimeError):
        _hip.paged_decode_scored(q, slab, slab, table, one, one)
    with pytest.raises(RuntimeError):
        _hip.evict_tokens(table, torch.zeros(1, 8), one, one, 2)
    with pytest.raises(RuntimeError):
        _hip.logit_controls(torch.zeros(1, 8))


def test_evicted_rows_that_share_memory_are_refused(monkeypatch):
    """The wrapper's own check of a given `evicted`, on CPU tensors with the launch caught: rows that overlap never reach the library, and
    the stride that does is the tensor's own."""
    calls = []
    monkeypatch.setattr(_hip, "_need_gpu", lambda *t: None)
    monkeypatch.setattr(_hip, "_same_gpu", lambda *t: None)
    monkeypatch.setattr(_hip, "_launch", lambda index, fn, *args: calls.append(args) or 0)
    table, w = torch.zeros(4, 32, dtype=torch.int32), torch.zeros(4, 32)
    req, lens = torch.tensor([0, 1, 2]), torch.tensor([30, 3, 20])
    one = torch.empty(7, dtype=torch.int32)
    for bad in (one.expand(3, 7), torch.as_strided(one, (3, 3), (2, 1)), one[:1].expand(3, 1), torch.empty(7, 3, dtype=torch.int32).t(),
                torch.empty(2, 7, dtype=torch.int32), torch.empty(3, 7)):
        with pytest.raises(ValueError, match="evicted"):
            _hip.evict_tokens(table, w, req, lens, 4, evicted=bad)
    assert not calls
    wide = torch.empty(3, 9, dtype=torch.int32)
    for good, stride, width in ((wide, 9, 9), (wide[:, :5], 9, 5), (wide[:, 2:3], 9, 1), (wide[:, :0], 9, 0)):
        _hip.evict_tokens(table, w, req, lens, 4, evicted=good)
        # ... (out_table, out_weights, table, stride, weights, stride, rows, columns, requests, lengths, new lengths, evicted, stride, width, ..)
        assert calls[-1][12:14] == (stride, width)
    _hip.evict_tokens(table, w, req[:1], lens[:1], 4, evicted=one.expand(1, 7))
    assert calls[-1][12:14] == (7, 7)


def test_evict_new_lengths_over_the_requests_rows():
    """Later requests look at the rows that earlier ones name."""
    def f(req, new, batch=4, cols=64):
        return lib.bsgl_evict_tokens(P, P, P, cols, P, cols, 2, cols, ctypes.c_void_p(req), ctypes.c_void_p(1 << 20), ctypes.c_void_p(new), None, 0, 0, batch, 4, 0, 0,
                                     0, None, 0, None)

    for new in (4096, 4096 - 24, 4096 + 24):
        assert f(4096, new) == _hip.BSGL_ERR_BAD_ARG and b"req_pool_indices" in lib.bsgl_last_error()


def test_results_that_are_their_inputs_in_part():
    """Shifted by an element, by a row, by a part of a row's gap: refused; in place, beside each other, columns apart: not this refusal's business (what
    answers those calls here is a workspace that is missing, or a type that is none, behind the check)."""
    at = 1 << 20

    def evict(out_t, out_w, rows=5, cols=20000, stride=40000):  # (rows this long need a workspace)
        v = ctypes.c_void_p
        return lib.bsgl_evict_tokens(v(out_t), v(out_w), v(at), stride, v(at), stride, rows, cols, v(64), v(1 << 10), v(1 << 12), None, 0, 0, 2, 4, 0, 0, 0, None, 0, None)

    row = 40000 * 4
    far = at + 100 * row
    for out in (at + 4, at - 4, at + row, at - row, at + 4 * row, at - 4 * row, at + 3 * row + 19999 * 4, at + row - 4, at + 20000 * 4 - 4):
        assert evict(out, far) == _hip.BSGL_ERR_BAD_ARG and b"share no memory" in lib.bsgl_last_error(), out
        assert evict(far, out) == _hip.BSGL_ERR_BAD_ARG and b"share no memory" in lib.bsgl_last_error(), out
    for out in (at, at + 20000 * 4, at - 20000 * 4, at + 5 * row, at + row + 20000 * 4, far):
        assert evict(out, out) == _hip.BSGL_ERR_WORKSPACE, out

    def logits(out, out_stride, in_stride=100, batch=3, vocab=100):
        c = _hip.LogitCall()
        for k, v in dict(out=out, logits=at, out_row_stride=out_stride, logits_row_stride=in_stride, batch=batch, vocab=vocab, dtype=2, repetition=256).items():
            setattr(c, k, v)
        return lib.bsgl_logit_controls(ctypes.byref(c))  # (penalties without a history: refused next)

    for out, stride in ((at + 4, 100), (at + 400, 100), (at - 400, 100), (at + 400, 300), (at - 4, 1000)):
        assert logits(out, stride) == _hip.BSGL_ERR_BAD_ARG and b"share no memory" in lib.bsgl_last_error(), (out, stride)
    for out, stride, kw in ((at, 100, {}), (at + 1200, 100, {}), (at - 1200, 100, {}), (at + 400, 200, dict(in_stride=200)), (at, 500, dict(batch=1)), (at + 800, 100, dict(in_stride=2000, batch=1))):
        assert logits(out, stride, **kw) == _hip.BSGL_ERR_BAD_ARG and b"history" in lib.bsgl_last_error(), (out, stride)
    w = dict(weights_row_stride=64)
    for out in (at + 4, at + 256, at - 252):
        assert lib.bsgl_paged_decode_scored(decode_call(), mods(token_weights=at, token_weights_out=out, **w)) == _hip.BSGL_ERR_BAD_ARG
        assert b"share no memory" in lib.bsgl_last_error()
    assert lib.bsgl_paged_decode_scored(decode_call(), mods(token_weights=at, token_weights_out=at, **w)) == _hip.BSGL_ERR_WORKSPACE
    assert lib.bsgl_paged_decode_scored(decode_call(), mods(token_weights=at, token_weights_out=at + 512, **w)) == _hip.BSGL_ERR_WORKSPACE


def test_the_library_alone_needs_no_python_to_build():
    """`make` is the C library with hipcc; what needs PyTorch and its headers is a target of its own."""
    import os
    import subprocess

    csrc = os.path.join(os.path.dirname(_hip.LIB_PATH), "csrc")
    plan = lambda *goals: subprocess.run(["make", "-n", "-B", "-C", csrc, *goals], capture_output=True, text=True, check=True).stdout  # noqa: E731
    alone = plan()
    assert "libbsgl_attn.so" in alone and "fast_calls" not in alone and "python" not in alone.replace("/python", "")
    both = plan("python")
    assert "libbsgl_attn.so" in both and "fast_calls" in both


def test_the_fast_calls_of_another_version_are_not_taken():
    """Another ABI version, or a descriptor of another size, than the extension was built with."""
    import ctypes as ct

    fast = _hip._fast
    assert fast is not None, "build baby-sglang_amd/_fast_calls.so (make -C baby-sglang_amd/csrc python)"
    right = [_hip.ABI_VERSION] + [ct.sizeof(t) for t in (_hip.DecodeCall, _hip.ScoreMods, _hip.LogitCall)]
    try:
        for i in range(4):
            with pytest.raises(ImportError, match="another version"):
                fast.bind(*(x + (j == i) for j, x in enumerate(right)), *[0] * 7)
        with pytest.raises(ImportError):
            fast.bind(*[0] * 7)
        with pytest.raises(TypeError):
            fast.bind("2", *right[1:], *[0] * 7)
    finally:
        _hip.bind_fast_calls()
