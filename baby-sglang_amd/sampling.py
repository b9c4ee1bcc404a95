"""Next-token selection on the device, for whole batches at once.

Counterpart of the reference's ``sample.py`` (reference: sample.py:8-17 ``SamplingParams``,
:19-37 repetition penalty, :40-90 ``sample_next_ids``).  The reference is called once per
request with a ``[1, vocab]`` row; here every function takes the ``[batch, vocab]`` logits of a
step and stays on the device (no per-request loop, no host read).  The filtered distribution
is the reference's bit for bit -- temperature, then top-k (ties with the k-th value kept),
then nucleus filtering over the survivors (the first token always kept), then softmax -- but
top-k and top-p share ONE descending sort: masking the values below the k-th only turns the
tail of the sorted row into -inf, which is exactly the sorted row of the masked logits.
The random draw itself (``torch.multinomial``) depends on the generator state and is not
comparable across implementations.

Not in the reference: presence and frequency penalties, sparse biases and token masks
(``SamplingParams``, ``LogitControls``), applied to the logits ahead of all that by one HIP launch
(``_hip.logit_controls``); the tokens a request has produced then live in a table on the device, so a step
moves none of them.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, Optional, Sequence

import torch


@dataclass
class SamplingParams:
    """Fields of the reference's ``SamplingParams`` (sample.py:8-17; ``json_schema`` belongs to
    constrained decoding, which is not part of this build)."""

    max_new_tokens: int = 64
    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    eos_id: int = -1
    do_sample: bool = False
    repetition_penalty: float = 1.0
    # not in the reference: over the tokens a request has produced, x - frequency * count - presence
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0
    logit_bias: Optional[Dict[int, float]] = None  # token id -> what is added to its logit
    allowed_token_ids: Optional[Sequence[int]] = None  # every other token is left out

    def needs_controls(self) -> bool:
        return bool(self.presence_penalty or self.frequency_penalty or self.logit_bias or self.allowed_token_ids is not None)


def pack_token_mask(allowed: torch.Tensor) -> torch.Tensor:
    """``allowed`` (bool [..., vocab]) as the int32 words ``_hip.logit_controls`` takes: bit t % 32 of word t / 32."""
    vocab = allowed.shape[-1]
    padded = torch.nn.functional.pad(allowed.to(torch.int64), (0, -vocab % 32))
    words = (padded.view(*allowed.shape[:-1], -1, 32) << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


class LogitControls:
    """What ``SamplingParams`` asks of the logits of a serving loop's steps, and the tokens its requests have produced:
    an int32 table ``[rows, columns]`` on the GPU, row r belonging to whoever owns page-table row r.  ``note``
    appends a step's ids, ``apply`` gives the controlled logits; neither reads anything back."""

    def __init__(self, params: SamplingParams, rows: int, columns: int, vocab: int, device: torch.device):
        if torch.device(device).type != "cuda":
            raise NotImplementedError("presence / frequency penalties, logit biases and token masks run on the GPU only")
        from . import _hip

        if columns > _hip.LOGIT_MAX_HISTORY and (params.presence_penalty or params.frequency_penalty or (params.repetition_penalty or 1.0) > 1.0):
            raise NotImplementedError(f"penalties over more than {_hip.LOGIT_MAX_HISTORY} tokens of a request (max_new_tokens is {columns})")
        if params.logit_bias and len(params.logit_bias) > _hip.LOGIT_MAX_BIAS:
            raise NotImplementedError(f"{len(params.logit_bias)} logit biases, up to {_hip.LOGIT_MAX_BIAS} are taken")
        self.params = params
        self.vocab = vocab
        self.history = torch.zeros((rows, columns), dtype=torch.int32, device=device)
        fill = lambda x: torch.full((rows,), float(x), dtype=torch.float32, device=device)  # noqa: E731
        self.repetition = fill(params.repetition_penalty) if (params.repetition_penalty or 1.0) > 1.0 else None
        self.presence = fill(params.presence_penalty) if params.presence_penalty else None
        self.frequency = fill(params.frequency_penalty) if params.frequency_penalty else None
        self.bias_ids = self.bias_values = self.token_mask = None
        if params.logit_bias:
            ids, values = zip(*sorted(params.logit_bias.items()))
            if min(ids) < 0 or max(ids) >= vocab:
                raise ValueError(f"logit_bias names a token outside the vocabulary of {vocab}")
            self.bias_ids = torch.tensor([ids], dtype=torch.int32, device=device).repeat(rows, 1)
            self.bias_values = torch.tensor([values], dtype=torch.float32, device=device).repeat(rows, 1)
        if params.allowed_token_ids is not None:
            allowed = torch.zeros(vocab, dtype=torch.bool)
            ids = torch.as_tensor(list(params.allowed_token_ids), dtype=torch.long)
            if ids.numel() == 0 or int(ids.min()) < 0 or int(ids.max()) >= vocab:
                raise ValueError(f"allowed_token_ids must name at least one token, all of them inside the vocabulary of {vocab}")
            allowed[ids] = True
            self.token_mask = pack_token_mask(allowed)[None].to(device)
            self._first = torch.zeros(rows, dtype=torch.int32, device=device)

        # (without a mask or a bias of -inf every token keeps a chance)
        self._can_empty = params.allowed_token_ids is not None or bool(params.logit_bias and min(params.logit_bias.values()) == float("-inf"))

    def note(self, rows: torch.Tensor, counts: torch.Tensor, ids: torch.Tensor) -> None:
        """Token ``ids[i]`` is number ``counts[i]`` (from 0) that row ``rows[i]``'s request produced."""
        self.history[rows, counts] = ids.to(torch.int32)

    def apply(self, logits: torch.Tensor, rows: torch.Tensor, counts: torch.Tensor, token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The logits of requests on ``rows`` that have produced ``counts`` tokens each.  ``token_mask`` (int32 words, one row
        per request) narrows the parameters' own.  Controls that leave a request no token raise (a draw from nothing
        ends the process); telling takes a read of the device, made only where masks or infinite biases are in play."""
        from . import _hip

        n, words = logits.shape[0], (self.vocab + 31) // 32
        kw = {}
        if self.repetition is not None or self.presence is not None or self.frequency is not None:
            cut = lambda t: None if t is None else t[:n]  # noqa: E731
            kw = dict(history=self.history, history_rows=rows, history_lens=counts, repetition=cut(self.repetition), presence=cut(self.presence),
                      frequency=cut(self.frequency))
        if self.bias_ids is not None:
            kw.update(bias_ids=self.bias_ids[:n], bias_values=self.bias_values[:n])
        if token_mask is not None:
            if token_mask.dtype != torch.int32 or token_mask.dim() != 2 or token_mask.shape[0] != n or token_mask.shape[1] < words:
                raise ValueError(f"token_mask must be int32 [{n}, {words}] (pack_token_mask), got {token_mask.dtype} {tuple(token_mask.shape)}")
            token_mask = token_mask.to(logits.device).contiguous()
            kw["token_mask"] = token_mask if self.token_mask is None else token_mask[:, :words] & self.token_mask
        elif self.token_mask is not None:
            kw.update(token_mask=self.token_mask, mask_rows=self._first[:n])
        controlled = _hip.logit_controls(logits, **kw)
        if self._can_empty or token_mask is not None:
            empty = (controlled.amax(-1) == float("-inf")).tolist()
            if any(empty):
                raise ValueError(f"masks and biases leave no token to pick for request {empty.index(True)} of the batch")
        return controlled


def apply_repetition_penalty_(logits: torch.Tensor, prev_ids: Sequence[Sequence[int]], penalty: float) -> torch.Tensor:
    """In place: logits of tokens a request has already produced or been given are divided by
    ``penalty`` when positive and multiplied by it otherwise (sample.py:19-37), for all rows
    with one indexed update.  ``prev_ids[i]`` are row i's tokens (duplicates count once)."""
    if penalty is None or penalty <= 1.0:
        return logits
    rows, cols = [], []
    for i, ids in enumerate(prev_ids):
        uniq = set(int(t) for t in ids)
        rows.extend([i] * len(uniq))
        cols.extend(uniq)
    if not rows:
        return logits
    r = torch.tensor(rows, dtype=torch.long, device=logits.device)
    c = torch.tensor(cols, dtype=torch.long, device=logits.device)
    val = logits[r, c]
    logits[r, c] = torch.where(val > 0, val / penalty, val * penalty)
    return logits


def next_token_probs(logits: torch.Tensor, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0) -> torch.Tensor:
    """The distribution the reference draws from (sample.py:59-89), ``[batch, vocab]``."""
    if temperature is None or temperature <= 0:
        temperature = 1.0
    scaled = logits / temperature
    vocab = scaled.shape[-1]
    use_k = bool(top_k) and top_k > 0
    use_p = bool(top_p) and top_p < 1.0
    if not use_k and not use_p:
        return torch.softmax(scaled, dim=-1)
    minus_inf = torch.full((), float("-inf"), dtype=scaled.dtype, device=scaled.device)
    if not use_p:
        kth = torch.topk(scaled, k=min(top_k, vocab), dim=-1).values[..., -1:]
        return torch.softmax(torch.where(scaled < kth, minus_inf, scaled), dim=-1)
    ordered, order = torch.sort(scaled, descending=True, dim=-1)
    if use_k:
        kth = ordered[..., min(top_k, vocab) - 1 : min(top_k, vocab)]
        ordered = torch.where(ordered < kth, minus_inf, ordered)
    mass = torch.cumsum(torch.softmax(ordered, dim=-1), dim=-1)
    drop = mass > top_p
    drop[..., 0] = False
    ordered = torch.where(drop, minus_inf, ordered)
    kept = torch.full_like(scaled, float("-inf")).scatter_(-1, order, ordered)
    return torch.softmax(kept, dim=-1)


def sample_next_ids(
    logits: torch.Tensor,
    do_sample: bool = False,
    temperature: float = 1.0,
    top_k: int = 0,
    top_p: float = 1.0,
    prev_ids: Optional[Sequence[Sequence[int]]] = None,
    repetition_penalty: float = 1.0,
    generator: Optional[torch.Generator] = None,
) -> torch.Tensor:
    """One id per row of ``logits`` (a copy is penalised, never the caller's tensor)."""
    if prev_ids is not None and repetition_penalty is not None and repetition_penalty > 1.0:
        logits = apply_repetition_penalty_(logits.clone(), prev_ids, repetition_penalty)
    if not do_sample:
        return torch.argmax(logits, dim=-1)
    probs = next_token_probs(logits, temperature, top_k, top_p)
    return torch.multinomial(probs, num_samples=1, generator=generator).squeeze(-1)
