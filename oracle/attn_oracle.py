"""CPU oracle for the paged-attention path.  TEST INFRASTRUCTURE ONLY.

Nothing under ``baby-sglang_amd/`` imports this module; only ``tests/``,
``__graft_entry__.smoke()`` and the ``cpu_baseline`` leg of ``bench.py`` do,
as the checker and never as the thing measured or shipped.

Two restatements of the reference algorithm, both plain PyTorch on the CPU:

* ``*_ref``   follow the reference step by step in the INPUT dtype -- per request:
  page-table slice -> K/V gather -> GQA head repeat -> torch SDPA
  (attn_backend.py:34-110 prefill, :112-149 decode; KV write
  memory_pool.py:152-171).  This is what "the reference's torch-CPU backend"
  costs and rounds like; it is pinned against the golden vectors captured from
  the reference itself (tests/golden/, generated by tests/golden/gen_golden.py)
  and is the ``cpu_baseline`` ("port") of bench.py.
* ``*_exact`` evaluate the same mathematical definition
  ``softmax(q K^T / sqrt(D) + mask) V`` in float64 on the same (already rounded)
  inputs, vectorised per request.  GPU kernels are compared with this one, so
  the tolerance measures the kernel's own rounding and not the reference's.

The third-party arithmetic on the path is torch's
``scaled_dot_product_attention`` (call sites attn_backend.py:94, :141;
torch>=2.0 per the reference's requirements.txt:1; installed here 2.10.0).
The reference holds no tests or vectors for it, so parity is pinned by the
goldens captured from the reference run in this build's container.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.nn.functional as F


# --------------------------------------------------------------------------- KV write
def kv_scatter_ref(
    k_slab: torch.Tensor,
    v_slab: torch.Tensor,
    loc: torch.Tensor,
    k_new: torch.Tensor,
    v_new: torch.Tensor,
) -> None:
    """In place ``slab[loc] = new`` with the reference's dtype handling
    (memory_pool.py:159-171): int32 loc widened, new rows cast to the slab dtype."""
    rows = loc.long()
    if k_new.dtype != k_slab.dtype:
        k_new = k_new.to(k_slab.dtype)
        v_new = v_new.to(v_slab.dtype)
    k_slab[rows] = k_new
    v_slab[rows] = v_new


# --------------------------------------------------------------------------- gather
def gather_request_kv(
    k_slab: torch.Tensor,
    v_slab: torch.Tensor,
    req_to_token: torch.Tensor,
    req_pool_idx: int,
    length: int,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Slots, K rows and V rows of one request's first ``length`` tokens
    (attn_backend.py:55-59, :123-128).  The slot vector is the bit-exact part."""
    slots = req_to_token[req_pool_idx, :length].long()
    return slots, k_slab[slots], v_slab[slots]


def _expand_kv_heads(x: torch.Tensor, n_q_heads: int) -> torch.Tensor:
    """[len, Hkv, D] -> [len, Hq, D]; q head h reads kv head h // (Hq // Hkv)."""
    n_kv = x.shape[1]
    if n_kv < n_q_heads:
        x = x.repeat_interleave(n_q_heads // n_kv, dim=1)
    return x


# --------------------------------------------------------------------------- reference-dtype path
def decode_ref(
    q: torch.Tensor,
    k_slab: torch.Tensor,
    v_slab: torch.Tensor,
    req_to_token: torch.Tensor,
    req_pool_indices: torch.Tensor,
    seq_lens: torch.Tensor,
) -> torch.Tensor:
    """One query row per request, no mask, SDPA default scale 1/sqrt(D)."""
    n_q_heads = q.shape[1]
    rows = []
    for i in range(len(seq_lens)):
        _, k_i, v_i = gather_request_kv(
            k_slab, v_slab, req_to_token, int(req_pool_indices[i]), int(seq_lens[i])
        )
        k_i = _expand_kv_heads(k_i, n_q_heads).transpose(0, 1).unsqueeze(0)
        v_i = _expand_kv_heads(v_i, n_q_heads).transpose(0, 1).unsqueeze(0)
        q_i = q[i : i + 1].transpose(0, 1).unsqueeze(0)  # [1, Hq, 1, D]
        o_i = F.scaled_dot_product_attention(q_i, k_i, v_i)
        rows.append(o_i.squeeze(0).transpose(0, 1).flatten(-2))
    return torch.cat(rows, dim=0)


def prefill_ref(
    q: torch.Tensor,
    k_slab: torch.Tensor,
    v_slab: torch.Tensor,
    req_to_token: torch.Tensor,
    req_pool_indices: torch.Tensor,
    seq_lens: torch.Tensor,
    prefix_lens: torch.Tensor,
    extended_lens: torch.Tensor,
) -> torch.Tensor:
    """Extend rows over the full sequence with an additive -inf bias in q's dtype
    where ``col > prefix + row`` (attn_backend.py:74-101)."""
    n_q_heads = q.shape[1]
    rows = []
    q_off = 0
    for i in range(len(seq_lens)):
        ext = int(extended_lens[i])
        if ext == 0:
            continue
        prefix, full = int(prefix_lens[i]), int(seq_lens[i])
        _, k_i, v_i = gather_request_kv(
            k_slab, v_slab, req_to_token, int(req_pool_indices[i]), full
        )
        k_i = _expand_kv_heads(k_i, n_q_heads).transpose(0, 1).unsqueeze(0)
        v_i = _expand_kv_heads(v_i, n_q_heads).transpose(0, 1).unsqueeze(0)
        q_i = q[q_off : q_off + ext].transpose(0, 1).unsqueeze(0)  # [1, Hq, ext, D]
        q_off += ext
        hidden = torch.arange(full).unsqueeze(0) > torch.arange(
            prefix, prefix + ext
        ).unsqueeze(1)
        bias = torch.zeros((1, 1, ext, full), dtype=q.dtype).masked_fill(
            hidden, float("-inf")
        )
        o_i = F.scaled_dot_product_attention(q_i, k_i, v_i, attn_mask=bias)
        rows.append(o_i.squeeze(0).transpose(0, 1).flatten(-2))
    if not rows:
        return q.new_zeros((0, q.shape[1] * q.shape[2]))
    return torch.cat(rows, dim=0)


def forward_ref(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    v: Optional[torch.Tensor],
    k_slab: torch.Tensor,
    v_slab: torch.Tensor,
    req_to_token: torch.Tensor,
    req_pool_indices: torch.Tensor,
    seq_lens: torch.Tensor,
    out_cache_loc: torch.Tensor,
    is_prefill: bool,
    prefix_lens: Optional[torch.Tensor] = None,
    extended_lens: Optional[torch.Tensor] = None,
    save_kv_cache: bool = True,
) -> torch.Tensor:
    """The backend entry (attn_backend.py:9-32) on raw tensors: write the new
    rows first, then attend.  Mutates the slabs like the reference does."""
    if save_kv_cache and k is not None and v is not None:
        kv_scatter_ref(k_slab, v_slab, out_cache_loc, k, v)
    if is_prefill:
        return prefill_ref(
            q, k_slab, v_slab, req_to_token, req_pool_indices, seq_lens,
            prefix_lens, extended_lens,
        )  # fmt: skip
    return decode_ref(q, k_slab, v_slab, req_to_token, req_pool_indices, seq_lens)


# --------------------------------------------------------------------------- float64 definition
def _attend_exact(
    q_i: torch.Tensor, k_i: torch.Tensor, v_i: torch.Tensor, first_visible_len: int
) -> Tuple[torch.Tensor, torch.Tensor]:
    """q_i [R, Hq, D], k_i/v_i [L, Hkv, D]; row r sees keys 0 .. first_visible_len-1+r.
    Returns (out [R, Hq*D], lse [R, Hq]) in float64."""
    n_rows, n_q_heads, dim = q_i.shape
    group = n_q_heads // k_i.shape[1]
    qd = q_i.double().view(n_rows, k_i.shape[1], group, dim)
    kd, vd = k_i.double(), v_i.double()
    scores = torch.einsum("rhgd,lhd->rhgl", qd, kd) / math.sqrt(dim)
    visible = torch.arange(k_i.shape[0]).unsqueeze(0) < (
        first_visible_len + torch.arange(n_rows)
    ).unsqueeze(1)
    scores = scores.masked_fill(~visible.view(n_rows, 1, 1, -1), float("-inf"))
    lse = torch.logsumexp(scores, dim=-1)
    probs = torch.exp(scores - lse.unsqueeze(-1))
    out = torch.einsum("rhgl,lhd->rhgd", probs, vd)
    return out.reshape(n_rows, n_q_heads * dim), lse.reshape(n_rows, n_q_heads)


def decode_exact(
    q, k_slab, v_slab, req_to_token, req_pool_indices, seq_lens, return_lse=False
):
    outs, lses = [], []
    for i in range(len(seq_lens)):
        n = int(seq_lens[i])
        if n <= 0:
            outs.append(torch.zeros((1, q.shape[1] * q.shape[2]), dtype=torch.float64))
            lses.append(torch.full((1, q.shape[1]), float("-inf"), dtype=torch.float64))
            continue
        _, k_i, v_i = gather_request_kv(
            k_slab, v_slab, req_to_token, int(req_pool_indices[i]), n
        )
        o, lse = _attend_exact(q[i : i + 1], k_i, v_i, n)
        outs.append(o)
        lses.append(lse)
    out = torch.cat(outs, dim=0)
    return (out, torch.cat(lses, dim=0)) if return_lse else out


def prefill_exact(
    q, k_slab, v_slab, req_to_token, req_pool_indices, seq_lens, prefix_lens, extended_lens
):
    outs = []
    q_off = 0
    for i in range(len(seq_lens)):
        ext = int(extended_lens[i])
        if ext == 0:
            continue
        _, k_i, v_i = gather_request_kv(
            k_slab, v_slab, req_to_token, int(req_pool_indices[i]), int(seq_lens[i])
        )
        o, _ = _attend_exact(q[q_off : q_off + ext], k_i, v_i, int(prefix_lens[i]) + 1)
        q_off += ext
        outs.append(o)
    if not outs:
        return torch.zeros((0, q.shape[1] * q.shape[2]), dtype=torch.float64)
    return torch.cat(outs, dim=0)


def merge_states_exact(parts_o: torch.Tensor, parts_lse: torch.Tensor):
    """[P, R, H, D], [P, R, H] -> merged ([R, H*D], [R, H]) in float64."""
    lse = parts_lse.double()
    mx = lse.max(dim=0).values
    safe = torch.where(torch.isinf(mx), torch.zeros_like(mx), mx)
    w = torch.exp(lse - safe)
    tot = w.sum(dim=0)
    out = (w.unsqueeze(-1) * parts_o.double()).sum(dim=0) / torch.where(
        tot > 0, tot, torch.ones_like(tot)
    ).unsqueeze(-1)
    merged_lse = torch.where(tot > 0, safe + torch.log(tot), torch.full_like(tot, float("-inf")))
    return out.reshape(out.shape[0], -1), merged_lse


# --------------------------------------------------------------------------- scored attention
def scored_exact(q, k_slab, v_slab, table_rows, seq_lens, row_req, row_pos, scale, cap=0.0, slopes=None, start=None, stop=None):
    """Scored attention in float64, query row by query row (no counterpart in the reference).

    ``q`` [R, Hq, D]; query row r belongs to request ``row_req[r]`` (whose slots are ``table_rows[req][: seq_lens[req]]``)
    at position ``row_pos[r]``; it sees ``[start[r], stop[r])`` of it (None: 0 and its own position + 1).
    Returns ``out`` [R, Hq, D], ``mass`` = sum p |v| of the same shape (what relative errors of the probabilities are
    weighted with), ``lse`` [R, Hq], ``received``: per row the probability of every position of its request summed over heads,
    and ``top`` [R, Hq]: the largest sum |q_d k_d| * scale of a visible token (what the error of a score is proportional to)."""
    n_rows, hq, dim = q.shape
    hkv = k_slab.shape[1]
    out = torch.zeros(n_rows, hq, dim, dtype=torch.float64)
    mass = torch.zeros_like(out)
    lse = torch.full((n_rows, hq), float("-inf"), dtype=torch.float64)
    top = torch.zeros(n_rows, hq, dtype=torch.float64)
    received = []
    for r in range(n_rows):
        req, pos = int(row_req[r]), int(row_pos[r])
        n = int(seq_lens[req])
        lo = 0 if start is None else int(start[r])
        hi = pos + 1 if stop is None else int(stop[r])
        lo = max(0, min(lo, n))
        hi = max(lo, min(hi, n))
        got = torch.zeros(n, dtype=torch.float64)
        if hi > lo:
            slots = table_rows[req][lo:hi].long()
            k = k_slab[slots].double().repeat_interleave(hq // hkv, dim=1)  # [n, Hq, D]
            v = v_slab[slots].double().repeat_interleave(hq // hkv, dim=1)
            prod = q[r].double()[None] * k
            s = prod.sum(-1) * scale
            top[r] = prod.abs().sum(-1).amax(0) * scale
            if cap > 0:
                s = cap * torch.tanh(s / cap)
            if slopes is not None:
                s = s - slopes.double()[None, :] * (torch.arange(lo, hi, dtype=torch.float64) - pos).abs()[:, None]
            lse[r] = torch.logsumexp(s, 0)
            p = torch.exp(s - lse[r])
            out[r] = (p[:, :, None] * v).sum(0)
            mass[r] = (p[:, :, None] * v.abs()).sum(0)
            got[lo:hi] = p.sum(1)
        received.append(got)
    return out, mass, lse, received, top
