"""Cases and plain forms of the operators around a serving step's scores.

Four operators, all over the pools' own layout (a page table of one-token pages, K and V rows of
a slot side by side):

``decode``   attention of one new token per request over the paged cache, its scores capped by a
             tanh, biased by distance and limited to an interval of positions; optionally the
             attention weight every cached token received is added to a table beside the page table
``extend``   the same scores for the new tokens of a prompt over a cached prefix, with an interval of
             visible positions per new token (causal, prefix, document and window masks)
``evict``    keeping the tokens with the largest accumulated weight of every request: page-table and
             weight rows compacted, the slots of the others handed back
``logits``   penalties for tokens already produced, sparse biases and token bitmasks on the logits

``listed()`` and ``draw()`` give cases, ``prepare()`` the tensors a serving program holds before the
call, ``run()`` one pass: in elementary torch operations, or (``own``) through the framework.
"""

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
VOCAB = 151936  # rows of the vocabulary projection of the models this framework runs
HEADS = [(12, 2, 128), (28, 4, 128), (14, 2, 64), (6, 1, 128)]  # (q heads, kv heads, head_dim)


# --------------------------------------------------------------------------- what a case stands for
def listed():
    return [
        # one chat request early in its answer: latency is all that counts
        dict(name="decode_one", op="decode", batch=1, lo=131, hi=131, heads=0, dtype="bf16", cap=50.0, slopes=False,
             mask="all", weights=False, lens=1),
        # the headline serving batch, with the weights an eviction policy needs
        dict(name="decode_batch", op="decode", batch=64, lo=2048, hi=2048, heads=0, dtype="bf16", cap=30.0, slopes=False,
             mask="all", weights=True, lens=2),
        # a large ragged batch of the wider model: distance bias, packed documents, weights
        dict(name="decode_ragged", op="decode", batch=96, lo=600, hi=4095, heads=1, dtype="f16", cap=0.0, slopes=True,
             mask="document", weights=True, lens=3),
        # 32-bit cache, heads of 64 values
        dict(name="decode_f32", op="decode", batch=9, lo=100, hi=1777, heads=2, dtype="f32", cap=20.0, slopes=True,
             mask="window", weights=True, lens=4),
        # a few short follow-up turns over cached prefixes
        dict(name="extend_turns", op="extend", batch=5, lo=3, hi=41, prefix=333, heads=2, dtype="bf16", cap=50.0,
             slopes=False, mask="causal", lens=5),
        # image or instruction prefixes that are read in both directions
        dict(name="extend_prefix", op="extend", batch=6, lo=700, hi=1501, prefix=0, heads=0, dtype="f16", cap=0.0,
             slopes=True, mask="prefix", lens=6),
        # a chunk of a large prefill over cached prefixes
        dict(name="extend_chunk", op="extend", batch=48, lo=512, hi=512, prefix=1536, heads=1, dtype="bf16", cap=30.0,
             slopes=False, mask="causal", lens=7),
        # the smallest eviction: a few requests just over their budget
        dict(name="evict_few", op="evict", batch=3, lo=261, hi=300, cols=512, budget=256, recent=32, sinks=4, lens=8),
        # the headline batch brought back to half its length
        dict(name="evict_batch", op="evict", batch=64, lo=2500, hi=4096, cols=4096, budget=2048, recent=256, sinks=4, lens=9),
        # a long document or two, cut to a tenth
        dict(name="evict_long", op="evict", batch=2, lo=100003, hi=131072, cols=131072, budget=12500, recent=1000,
             sinks=4, lens=10),
        # one request with a grammar: few tokens allowed
        dict(name="logits_one", op="logits", batch=1, vocab=VOCAB, dtype="bf16", history=150, prompt=40, bias=5, mask="few", lens=11),
        # the headline batch: long histories, biases, a mask for some of the rows
        dict(name="logits_batch", op="logits", batch=64, vocab=VOCAB, dtype="f32", history=2048, prompt=1024, bias=40, mask="some", lens=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "extend", "extend", "evict", "logits"])
    lens = rng.randrange(1 << 30)
    if op == "decode":
        while True:
            batch, hi, heads, dtype = _log(rng, 1, 128), _log(rng, 1, 16384), rng.randrange(4), rng.choice(["bf16", "f16", "f32"])
            _, hkv, dim = HEADS[heads]
            if batch * hi * hkv * dim * BYTES[dtype] <= 96 * 2400 * 4 * 128 * 2:
                break
        return dict(op=op, batch=batch, lo=rng.randint(max(1, hi // 4), hi), hi=hi, heads=heads, dtype=dtype,
                    cap=rng.choice([0.0, 15.0, 30.0, 50.0]), slopes=rng.random() < 0.5,
                    mask=rng.choice(["all", "document", "window", "empty"]), weights=rng.random() < 0.7, lens=lens)
    if op == "extend":
        while True:
            batch, hi, prefix = _log(rng, 1, 48), _log(rng, 1, 2048), rng.choice([0, _log(rng, 1, 8192)])
            heads, dtype = rng.randrange(4), rng.choice(["bf16", "f16", "bf16", "f16", "f32"])
            hq, _, dim = HEADS[heads]
            pairs = batch * hi * (hi + prefix)
            if pairs * hq * dim <= (48 * 512 * 1800 * 28 * 128 if dtype != "f32" else 4 * 300 * 800 * 28 * 128):
                break
        return dict(op=op, batch=batch, lo=rng.randint(max(1, hi // 4), hi), hi=hi, prefix=prefix, heads=heads, dtype=dtype,
                    cap=rng.choice([0.0, 15.0, 30.0, 50.0]), slopes=rng.random() < 0.5,
                    mask=rng.choice(["causal", "prefix", "document", "window", "empty"]), lens=lens)
    if op == "evict":
        while True:
            batch, hi = _log(rng, 1, 128), _log(rng, 4, 131072)
            if batch * hi <= 64 * 4096:
                break
        budget = max(1, int(hi * rng.uniform(0.05, 1.1)))
        recent = rng.randint(0, budget // 2)
        return dict(op=op, batch=batch, lo=rng.randint(max(1, hi // 2), hi), hi=hi, cols=hi + rng.randint(0, 100), budget=budget,
                    recent=recent, sinks=rng.randint(0, min(8, budget - recent)), lens=lens)
    while True:
        batch, vocab = _log(rng, 1, 128), rng.choice([VOCAB, _log(rng, 50, VOCAB)])
        history = rng.choice([0, _log(rng, 1, 16384)])
        if batch * (vocab + 4 * history) <= 64 * (VOCAB + 4 * 2048):
            break
    return dict(op=op, batch=batch, vocab=vocab, dtype=rng.choice(["bf16", "f16", "f32"]), history=history,
                prompt=rng.randint(0, history), bias=rng.choice([0, rng.randint(1, 300)]),
                mask=rng.choice(["none", "few", "some", "most", "empty"]), lens=lens)


def _lens(case, n, lo, hi):
    """The lengths of a case: part of what it IS, so that its work is known without its data."""
    r = random.Random(case["lens"])
    return [r.randint(lo, hi) for _ in range(n)]


def _spans(case, length, rows, r):
    """First and one-past-last visible position of the last ``rows`` of ``length`` positions."""
    i = np.arange(length - rows, length, dtype=np.int64)
    start, stop = np.zeros(rows, np.int64), i + 1
    kind = case["mask"]
    if kind == "window":
        start = np.maximum(i + 1 - max(1, length // 3), 0)
    elif kind == "prefix":  # the first third of the request is read in both directions
        stop = np.maximum(stop, length // 3)
    elif kind == "document":  # up to four documents packed one behind the other
        cuts = np.array(sorted(r.randrange(length) for _ in range(3)), np.int64)
        for c in cuts:
            start = np.where(i >= c, c, start)
    elif kind == "empty":  # a fifth of the rows sees nothing
        none = np.array([r.random() < 0.2 for _ in range(rows)])
        stop = np.where(none, start, stop)
    return start, stop


def _attention_plan(case):
    n, r = case["batch"], random.Random(case["lens"] + 1)
    new = _lens(case, n, case["lo"], case["hi"])
    if case["op"] == "decode":
        lens, rows = new, [1] * n
    else:
        pre = [0 if case["prefix"] == 0 else r.randint(case["prefix"] // 2, case["prefix"]) if case["lo"] != case["hi"] else case["prefix"]
               for _ in range(n)]
        lens, rows = [a + b for a, b in zip(new, pre)], new
    spans = [_spans(case, le, ro, r) for le, ro in zip(lens, rows)]
    return lens, rows, spans


# --------------------------------------------------------------------------- the work of a pass
def work(case):
    if case["op"] in ("decode", "extend"):
        hq, hkv, dim = HEADS[case["heads"]]
        eb = BYTES[case["dtype"]]
        _, rows, spans = _attention_plan(case)
        pairs = sum(int(np.maximum(b - a, 0).sum()) for a, b in spans)
        seen = 0  # cached tokens that some row sees
        for a, b in spans:
            live = b > a
            seen += int(b[live].max() - a[live].min()) if live.any() else 0
        n_bytes = seen * (2 * hkv * dim * eb + 4) + 2 * sum(rows) * hq * dim * eb
        if case.get("weights"):
            n_bytes += 8 * seen
        return {"bytes": n_bytes, "flops": 4 * hq * dim * pairs}
    if case["op"] == "evict":
        n = sum(_lens(case, case["batch"], case["lo"], case["hi"]))
        kept = sum(min(x, case["budget"]) for x in _lens(case, case["batch"], case["lo"], case["hi"]))
        return {"bytes": 8 * n + 8 * kept + 4 * (n - kept), "flops": n}
    eb = BYTES[case["dtype"]]
    mask = 0 if case["mask"] == "none" else case["batch"] * ((case["vocab"] + 31) // 32) * 4
    return {"bytes": 2 * case["batch"] * case["vocab"] * eb + 4 * case["batch"] * case["history"] + 8 * case["batch"] * case["bias"] + mask,
            "flops": 4 * case["batch"] * case["vocab"]}


# --------------------------------------------------------------------------- inputs
def _page_table(lens, cols, n_rows, g):
    """A page table whose used entries are distinct slots in random order, the rest zero."""
    total = sum(lens)
    perm = (torch.randperm(total, generator=g, device=DEV) + 1).to(torch.int32)
    table = torch.zeros((n_rows, cols), dtype=torch.int32, device=DEV)
    row_of = torch.randperm(n_rows, generator=g, device=DEV)[: len(lens)]
    at = 0
    for i, n in enumerate(lens):
        table[row_of[i], :n] = perm[at : at + n]
        at += n
    return table, row_of.to(torch.int64), total + 1


def _prepare_attention(case, g):
    hq, hkv, dim = HEADS[case["heads"]]
    dtype = DTYPES[case["dtype"]]
    lens, rows, spans = _attention_plan(case)
    table, row_of, n_slots = _page_table(lens, max(lens) + 7, len(lens) + 2, g)
    kv = torch.empty((n_slots, 2, hkv, dim), dtype=dtype, device=DEV).normal_(generator=g)
    q = (3.0 * torch.randn((sum(rows), hq, dim), generator=g, device=DEV)).to(dtype)
    st = dict(case=case, hq=hq, hkv=hkv, dim=dim, q=q, k_slab=kv[:, 0], v_slab=kv[:, 1], table=table, row_of=row_of, lens=lens, rows=rows,
              seq_lens=torch.tensor(lens, dtype=torch.int64, device=DEV), scale=dim**-0.5, cap=case["cap"], slopes=None,
              start=None, stop=None, spans=spans)
    if case["slopes"]:
        st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], dtype=torch.float32, device=DEV)
    if case["mask"] in ("document", "window", "empty", "prefix"):
        st["start"] = torch.from_numpy(np.concatenate([a for a, _ in spans]).astype(np.int32)).to(DEV)
        st["stop"] = torch.from_numpy(np.concatenate([b for _, b in spans]).astype(np.int32)).to(DEV)
    st["out"] = torch.zeros((sum(rows), hq * dim), dtype=dtype, device=DEV)
    if case["op"] == "extend":
        st["new"] = torch.tensor(rows, dtype=torch.int64, device=DEV)
        st["prefix"] = st["seq_lens"] - st["new"]
    elif case["weights"]:
        st["weights"] = torch.rand(table.shape, generator=g, device=DEV) * 4.0
        st["weights_out"] = torch.zeros_like(st["weights"])
    if own:
        from baby_sglang_amd import _hip

        if case["op"] == "decode":
            st["n_splits"] = _hip.decode_num_splits(len(lens), hkv, table.shape[1])
            st["workspace"] = _hip.new_decode_workspace(
                _hip.decode_scored_workspace_bytes(len(lens), hq, dim, st["n_splits"], table.shape[1], bool(case["weights"])), DEV)
        else:
            st["workspace"] = torch.empty(_hip.prefill_workspace_bytes(len(lens), sum(rows), hq, dim), dtype=torch.uint8, device=DEV)
    return st


def _prepare_evict(case, g):
    lens = _lens(case, case["batch"], case["lo"], case["hi"])
    table, row_of, _ = _page_table(lens, case["cols"], case["batch"] + 1, g)
    # accumulated weights are heavy-tailed, and some tokens never received any
    weights = torch.exp(2.0 * torch.randn(table.shape, generator=g, device=DEV))
    weights *= (torch.rand(table.shape, generator=g, device=DEV) > 0.1).float()
    width = max(0, case["cols"] - case["budget"])
    st = dict(case=case, table=table, weights=weights, row_of=row_of, lens=lens, seq_lens=torch.tensor(lens, dtype=torch.int64, device=DEV),
              out_table=torch.zeros_like(table), out_weights=torch.zeros_like(weights), new_lens=torch.zeros(len(lens), dtype=torch.int64, device=DEV),
              evicted=torch.zeros((len(lens), width), dtype=torch.int32, device=DEV))
    if own:
        from baby_sglang_amd import _hip

        st["workspace"] = torch.empty(_hip.evict_workspace_bytes(len(lens), table.shape[1], case["budget"]), dtype=torch.uint8, device=DEV)
    return st


def _prepare_logits(case, g):
    n, vocab = case["batch"], case["vocab"]
    r = random.Random(case["lens"])
    logits = (4.0 * torch.randn((n, vocab), generator=g, device=DEV)).to(DTYPES[case["dtype"]])
    st = dict(case=case, logits=logits, history=None, token_mask=None, bias_ids=None, bias_values=None, out=torch.zeros_like(logits))
    if case["history"]:
        cols = case["history"]
        lens = [r.randint(max(1, cols // 2), cols) if i else cols for i in range(n)]
        # text repeats its common words: ids fall off like 1 / rank
        u = torch.rand((n + 1, cols), generator=g, device=DEV)
        st["history"] = (torch.exp(u * math.log(vocab)) - 1.0).to(torch.int32).clamp_(0, vocab - 1)
        st["rows"] = torch.randperm(n + 1, generator=g, device=DEV)[:n].to(torch.int64)
        st["row_list"] = st["rows"].tolist()
        st["lens"] = lens
        st["history_lens"] = torch.tensor(lens, dtype=torch.int64, device=DEV)
        st["prompt"] = [min(case["prompt"], x) for x in lens]
        st["prompt_lens"] = torch.tensor(st["prompt"], dtype=torch.int64, device=DEV)
        st["repetition"] = 1.0 + 0.3 * torch.rand(n, generator=g, device=DEV)
        st["presence"] = torch.rand(n, generator=g, device=DEV)
        st["frequency"] = 0.4 * torch.rand(n, generator=g, device=DEV)
    if case["bias"]:
        st["bias_ids"] = torch.randint(0, vocab, (n, case["bias"]), generator=g, device=DEV, dtype=torch.int32)
        st["bias_ids"][:, -1] = -1  # an unused place
        st["bias_values"] = 5.0 * torch.randn((n, case["bias"]), generator=g, device=DEV)
    if case["mask"] != "none":
        share = {"few": 20.0 / vocab, "some": 0.5, "most": 0.97, "empty": 0.5}[case["mask"]]
        allowed = torch.rand((n, (vocab + 31) // 32, 32), generator=g, device=DEV) < share
        if case["mask"] == "empty":
            allowed[0] = False
        bit = torch.arange(32, device=DEV, dtype=torch.int64)
        words = (allowed.long() << bit).sum(-1)
        st["token_mask"] = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
        st["mask_list"] = [-1 if case["mask"] == "some" and i % 3 == 0 else i for i in range(n)]
        st["mask_rows"] = torch.tensor(st["mask_list"], dtype=torch.int32, device=DEV)
    return st


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] in ("decode", "extend"):
        return _prepare_attention(case, g)
    return _prepare_evict(case, g) if case["op"] == "evict" else _prepare_logits(case, g)


# --------------------------------------------------------------------------- plain forms
def _plain_attention(st):
    """Request by request: gather its K and V rows, scores of all its rows, softmax, product."""
    hq, hkv, dim = st["hq"], st["hkv"], st["dim"]
    group = hq // hkv
    decode = st["case"]["op"] == "decode"
    weights = st.get("weights")
    at = 0
    for i, (n, rows) in enumerate(zip(st["lens"], st["rows"])):
        slots = st["table"][st["row_of"][i], :n].long()
        k = st["k_slab"][slots].float().permute(1, 2, 0).contiguous()  # [kv head, dim, n]
        v = st["v_slab"][slots].float().permute(1, 0, 2).contiguous()  # [kv head, n, dim]
        j = torch.arange(n, device=DEV)
        pos = torch.arange(n - rows, n, device=DEV)[:, None]
        seen = j[None, :] <= pos
        if st["start"] is not None:
            seen = (j[None, :] >= st["start"][at : at + rows, None]) & (j[None, :] < st["stop"][at : at + rows, None])
        step = max(1, (1 << 27) // (n * hq))  # rows at a time, so that the scores stay below 512 MB
        for r0 in range(0, rows, step):
            r1 = min(rows, r0 + step)
            q = st["q"][at + r0 : at + r1].float().view(r1 - r0, hkv, group, dim).permute(1, 2, 0, 3).reshape(hkv, group * (r1 - r0), dim)
            s = (torch.matmul(q, k) * st["scale"]).view(hkv, group, r1 - r0, n)
            if st["cap"] > 0:
                s = st["cap"] * torch.tanh(s / st["cap"])
            if st["slopes"] is not None:
                s = s - st["slopes"].view(hkv, group, 1, 1) * (j[None, :] - pos[r0:r1]).abs().float()
            s = torch.where(seen[r0:r1], s, torch.full_like(s, float("-inf")))
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(top == float("-inf"), torch.zeros_like(top), top))
            total = p.sum(-1, keepdim=True)
            p = torch.where(total > 0, p / total, torch.zeros_like(p))
            o = torch.matmul(p.view(hkv, group * (r1 - r0), n), v).view(hkv, group, r1 - r0, dim).permute(2, 0, 1, 3)
            st["out"][at + r0 : at + r1] = o.reshape(r1 - r0, hq * dim).to(st["out"].dtype)
            if decode and weights is not None:
                row = st["row_of"][i]
                st["weights_out"][row, :n] = torch.where(seen[0], weights[row, :n] + p.sum((0, 1, 2)), st["weights_out"][row, :n])
        at += rows
    return [st["out"], st["weights_out"]] if decode and weights is not None else [st["out"]]


def _plain_evict(st):
    c = st["case"]
    for i, n in enumerate(st["lens"]):
        row = st["row_of"][i]
        slots, w = st["table"][row, :n], st["weights"][row, :n]
        st["evicted"][i] = -1
        keep = torch.ones(n, dtype=torch.bool, device=DEV)
        if n > c["budget"]:
            lo, hi = c["sinks"], n - c["recent"]
            order = torch.sort(w[lo:hi], descending=True, stable=True).indices
            keep[lo + order[c["budget"] - c["sinks"] - c["recent"] :]] = False
            st["evicted"][i, : n - c["budget"]] = slots[~keep]
        m = min(n, c["budget"])
        st["out_table"][row, :m] = slots[keep]
        st["out_weights"][row, :m] = w[keep]
        st["new_lens"][i] = m
    return [st["out_table"], st["out_weights"], st["new_lens"], st["evicted"]]


def _plain_logits(st):
    c = st["case"]
    vocab = c["vocab"]
    for i in range(c["batch"]):
        x = st["logits"][i].float()
        if st["history"] is not None:
            ids = st["history"][st["row_list"][i], : st["lens"][i]].long()
            seen = torch.zeros(vocab, device=DEV)
            seen[ids] = 1.0
            counts = torch.zeros(vocab, device=DEV).index_add_(0, ids[st["prompt"][i] :], torch.ones_like(ids[st["prompt"][i] :], dtype=torch.float32))
            x = torch.where(seen > 0, torch.where(x > 0, x / st["repetition"][i], x * st["repetition"][i]), x)
            x = x - st["frequency"][i] * counts - st["presence"][i] * (counts > 0).float()
        if st["bias_ids"] is not None:
            ok = st["bias_ids"][i] >= 0
            x = x + torch.zeros(vocab, device=DEV).index_add_(0, st["bias_ids"][i].clamp(min=0).long(), torch.where(ok, st["bias_values"][i], 0.0))
        if st["token_mask"] is not None and st["mask_list"][i] >= 0:
            words = st["token_mask"][st["mask_list"][i]].long()
            allowed = ((words[:, None] >> torch.arange(32, device=DEV)) & 1).view(-1)[:vocab]
            x = torch.where(allowed > 0, x, torch.full_like(x, float("-inf")))
        st["out"][i] = x.to(st["out"].dtype)
    return [st["out"]]


# --------------------------------------------------------------------------- one pass
def run(st):
    op = st["case"]["op"]
    if not own:
        return _plain_attention(st) if op in ("decode", "extend") else _plain_evict(st) if op == "evict" else _plain_logits(st)
    from baby_sglang_amd import _hip

    if op == "decode":
        out = _hip.paged_decode_scored(
            st["q"], st["k_slab"], st["v_slab"], st["table"], st["row_of"], st["seq_lens"], scale=st["scale"], logit_cap=st["cap"],
            slopes=st["slopes"], visible_from=st["start"], visible_to=st["stop"], token_weights=st.get("weights"),
            token_weights_out=st.get("weights_out"), n_splits=st["n_splits"], out=st["out"], workspace=st["workspace"],
            max_seq_len=max(st["lens"]))
        return [out] if st.get("weights") is None else [out, st["weights_out"]]
    if op == "extend":
        return [_hip.paged_prefill_scored(
            st["q"], st["k_slab"], st["v_slab"], st["table"], st["row_of"], st["seq_lens"], st["prefix"], st["new"], scale=st["scale"],
            logit_cap=st["cap"], slopes=st["slopes"], visible_from=st["start"], visible_to=st["stop"], out=st["out"],
            workspace=st["workspace"])]
    c = st["case"]
    if op == "evict":
        new_lens, evicted = _hip.evict_tokens(
            st["table"], st["weights"], st["row_of"], st["seq_lens"], c["budget"], recent=c["recent"], sinks=c["sinks"],
            out_table=st["out_table"], out_weights=st["out_weights"], evicted=st["evicted"], new_lens=st["new_lens"],
            max_seq_len=max(st["lens"]), workspace=st["workspace"])
        return [st["out_table"], st["out_weights"], new_lens, evicted]
    args = {}
    if st["history"] is not None:
        args = dict(history=st["history"], history_rows=st["rows"], history_lens=st["history_lens"], prompt_lens=st["prompt_lens"],
                    repetition=st["repetition"], presence=st["presence"], frequency=st["frequency"])
    return [_hip.logit_controls(st["logits"], bias_ids=st["bias_ids"], bias_values=st["bias_values"], token_mask=st["token_mask"],
                                mask_rows=st.get("mask_rows"), out=st["out"], **args)]


# --------------------------------------------------------------------------- the definition in 64 bits
def _exact_attention(case, st):
    hq, hkv, dim = HEADS[case["heads"]]
    ratio = hq // hkv
    out = torch.zeros((sum(st["rows"]), hq, dim), dtype=torch.float64, device=DEV)
    acc = st["weights_out"].double() if st.get("weights") is not None else None
    first = 0
    for i, (n, rows) in enumerate(zip(st["lens"], st["rows"])):
        begin, end = (torch.from_numpy(np.ascontiguousarray(x)).to(DEV) for x in st["spans"][i])
        where = st["table"][st["row_of"][i]][:n].long()
        keys, values = st["k_slab"][where].double(), st["v_slab"][where].double()
        cols = torch.arange(n, device=DEV, dtype=torch.float64)
        own_pos = torch.arange(n - rows, n, device=DEV, dtype=torch.float64)
        visible = (cols >= begin.double()[:, None]) & (cols < end.double()[:, None])
        received = torch.zeros(n, dtype=torch.float64, device=DEV)
        for h in range(hq):
            block = max(1, (1 << 26) // n)
            for r0 in range(0, rows, block):
                r1 = min(rows, r0 + block)
                query = st["q"][first + r0 : first + r1, h].double()
                score = torch.mm(query, keys[:, h // ratio].t().contiguous()) / math.sqrt(dim)
                if case["cap"]:
                    score = torch.tanh(score / case["cap"]) * case["cap"]
                if case["slopes"]:
                    score -= float(st["slopes"][h].item()) * (own_pos[r0:r1, None] - cols[None, :]).abs()
                score.masked_fill_(~visible[r0:r1], float("-inf"))
                norm = torch.logsumexp(score, dim=1, keepdim=True)
                prob = torch.exp(score - norm).nan_to_num_(nan=0.0)
                out[first + r0 : first + r1, h] = torch.mm(prob, values[:, h // ratio].contiguous())
                received += prob.sum(0)
        if acc is not None:
            row = int(st["row_of"][i])
            live = visible[0]
            acc[row, :n][live] = st["weights"][row, :n].double()[live] + received[live]
        first += rows
    res = [out.view(out.shape[0], hq * dim)]
    return res + [acc] if acc is not None else res


def _exact_logits(case, st):
    x = st["logits"].double()
    for i in range(case["batch"]):
        if st["history"] is not None:
            past = st["history"][st["row_list"][i]][: st["lens"][i]].tolist()
            often = {}
            for at, t in enumerate(past):
                often[t] = often.get(t, 0) + (1 if at >= st["prompt"][i] else 0)
            ids = torch.tensor(list(often), device=DEV)
            n = torch.tensor(list(often.values()), device=DEV, dtype=torch.float64)
            rep, pre, fre = (float(st[k][i].item()) for k in ("repetition", "presence", "frequency"))
            y = x[i, ids]
            x[i, ids] = torch.where(y > 0, y / rep, y * rep) - fre * n - pre * (n > 0)
        if st["bias_ids"] is not None:
            add = {}
            for t, b in zip(st["bias_ids"][i].tolist(), st["bias_values"][i].tolist()):
                if t >= 0:
                    add[t] = add.get(t, 0.0) + b
            ids = torch.tensor(list(add), device=DEV, dtype=torch.long)
            x[i, ids] += torch.tensor(list(add.values()), device=DEV, dtype=torch.float64)
        if st["token_mask"] is not None and st["mask_list"][i] >= 0:
            words = st["token_mask"][st["mask_list"][i]].cpu().numpy().view(np.uint8)
            on = np.unpackbits(words, bitorder="little")[: case["vocab"]].astype(bool)
            x[i].masked_fill_(torch.from_numpy(~on).to(DEV), float("-inf"))
    return [x]


def _exact_evict(case, st):
    table, weights, rows = st["table"].cpu().numpy(), st["weights"].cpu().numpy(), st["row_of"].tolist()
    to, wo = np.zeros_like(table), np.zeros(weights.shape, np.float64)
    gone = np.full(st["evicted"].shape, -1, np.int32)
    lens = np.zeros(len(rows), np.int64)
    for i, (row, n) in enumerate(zip(rows, st["lens"])):
        chosen = np.arange(n)
        if n > case["budget"]:
            middle = range(case["sinks"], n - case["recent"])
            w = weights[row]
            best = sorted(middle, key=lambda c: (-w[c], c))[: case["budget"] - case["sinks"] - case["recent"]]
            chosen = np.array(sorted(list(range(case["sinks"])) + best + list(range(n - case["recent"], n))), np.int64)
            rest = np.setdiff1d(np.arange(n), chosen)
            gone[i, : len(rest)] = table[row][rest]
        lens[i] = len(chosen)
        to[row, : len(chosen)], wo[row, : len(chosen)] = table[row][chosen], weights[row][chosen]
    return [torch.from_numpy(t).to(DEV) for t in (to, wo, lens, gone)]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] in ("decode", "extend"):
        return _exact_attention(case, st)
    return _exact_evict(case, st) if case["op"] == "evict" else _exact_logits(case, st)
