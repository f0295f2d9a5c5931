"""Chunked prefill and decode drivers (the callers of the hot path, after lazykv/generate.py:97-184)."""

from __future__ import annotations

import time
from collections.abc import Iterator
from dataclasses import dataclass, field

import torch
from transformers import PreTrainedModel
from transformers.cache_utils import Cache


def cache_model_kwargs(cache: Cache) -> dict[str, object]:
    fn = getattr(cache, "model_kwargs", None)
    return fn() if fn is not None else {}


@dataclass
class PrefillResult:
    last_logits: torch.Tensor  # [vocab] float32
    wall_s: float  # host clock around the prefill, synchronised on both sides
    event_s: float  # device time between CUDA events (0.0 on a CPU model)
    chunks: int


class _Clock:
    """Wall time and, for a CUDA model, event time of one region (both synchronised)."""

    def __init__(self, device: torch.device) -> None:
        self.cuda = device.type == "cuda"

    def __enter__(self) -> _Clock:
        if self.cuda:
            self.a, self.b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda.synchronize()
            self.a.record()
        self.t0 = time.perf_counter()
        return self

    def stop(self) -> tuple[float, float]:
        if self.cuda:
            self.b.record()
            torch.cuda.synchronize()
        wall = time.perf_counter() - self.t0
        return wall, (self.a.elapsed_time(self.b) / 1e3 if self.cuda else 0.0)

    def __exit__(self, *exc: object) -> None:
        return None


@torch.inference_mode()
def prefill(model: PreTrainedModel, cache: Cache, input_ids: torch.Tensor, chunk_size: int, observer: object | None = None) -> PrefillResult:
    """Chunked prefill keeping only the last position's logits (lazykv/generate.py:97-125)."""
    if observer is not None:
        raise ValueError("attention observers (prefill scoring) are not built")
    ids = input_ids.to(model.device).view(1, -1)
    logits, chunks = None, 0
    with _Clock(model.device) as clock:
        for s in range(0, ids.shape[1], chunk_size):
            out = model(input_ids=ids[:, s : s + chunk_size], past_key_values=cache, use_cache=True, logits_to_keep=1)
            logits, chunks = out.logits, chunks + 1
        assert logits is not None
        last = logits[0, -1].float()
        wall, ev = clock.stop()
    return PrefillResult(last, wall, ev, chunks)


@dataclass
class DecodeResult:
    tokens: list[int]
    wall_s: list[float] = field(default_factory=list)  # per token, host sync included
    event_s: list[float] = field(default_factory=list)  # per token, CUDA events (0.0 on a CPU model)


@torch.inference_mode()
def teacher_forced_decode(model: PreTrainedModel, cache: Cache, first_logits: torch.Tensor, continuation_ids: torch.Tensor) -> Iterator[torch.Tensor]:
    """Log-probs at each forced continuation position, one single-token decode step each."""
    yield torch.log_softmax(first_logits.float(), dim=-1)
    ids = torch.empty((1, 1), dtype=torch.long, device=model.device)
    extra = cache_model_kwargs(cache)
    for tok in continuation_ids.view(-1).tolist()[:-1]:
        ids.fill_(tok)
        out = model(input_ids=ids, past_key_values=cache, use_cache=True, logits_to_keep=1, **extra)
        yield torch.log_softmax(out.logits[0, -1].float(), dim=-1)


@torch.inference_mode()
def greedy_decode(model: PreTrainedModel, cache: Cache, first_logits: torch.Tensor, n_tokens: int) -> DecodeResult:
    """Greedy decode (lazykv/generate.py:134-154): token 0 from the prefill logits, then n_tokens
    single-token steps, each timed; the token reaches the host every step, as in generation."""
    tok = int(torch.argmax(first_logits).item())
    res = DecodeResult(tokens=[tok])
    ids = torch.empty((1, 1), dtype=torch.long, device=model.device)
    extra = cache_model_kwargs(cache)
    for _ in range(n_tokens):
        ids.fill_(tok)
        with _Clock(model.device) as clock:
            out = model(input_ids=ids, past_key_values=cache, use_cache=True, logits_to_keep=1, **extra)
            nxt = torch.argmax(out.logits[0, -1])
            wall, ev = clock.stop()
        tok = int(nxt.item())
        res.wall_s.append(wall)
        res.event_s.append(ev)
        res.tokens.append(tok)
    return res


def teacher_forced_steps(model: PreTrainedModel, cache: Cache, context_ids: torch.Tensor, continuation_ids: torch.Tensor,
                         chunk_size: int) -> Iterator[torch.Tensor]:
    """Log-probs (float32) at each continuation position: row i is the distribution over
    continuation token i given the context and continuation[:i], scored through single-token
    decode steps after a chunked prefill of the context (lazykv/generate.py:157-168)."""
    pre = prefill(model, cache, context_ids, chunk_size)
    yield from teacher_forced_decode(model, cache, pre.last_logits, continuation_ids)


def teacher_forced_logprobs(model: PreTrainedModel, cache: Cache, context_ids: torch.Tensor, continuation_ids: torch.Tensor,
                            chunk_size: int) -> torch.Tensor:
    """Every row of teacher_forced_steps as one float32 CPU tensor [positions, vocab], filled in
    place (lazykv/generate.py:186-197)."""
    rows: torch.Tensor | None = None
    for i, row in enumerate(teacher_forced_steps(model, cache, context_ids, continuation_ids, chunk_size)):
        if rows is None:
            rows = torch.empty((continuation_ids.numel(), row.numel()), dtype=torch.float32)
        rows[i].copy_(row)
    assert rows is not None
    return rows


@dataclass
class SpeculativeResult:
    tokens: list[int]
    drafted: int = 0  # tokens that the draft proposed
    kept: int = 0  # of them, tokens that the target kept


@torch.inference_mode()
def speculative_decode(model: PreTrainedModel, cache: Cache, draft_model: PreTrainedModel, draft_cache: Cache, first_token: int, n_tokens: int,
                       n_draft: int, temperature: float = 1.0, generator: torch.Generator | None = None) -> SpeculativeResult:
    """n_tokens tokens after `first_token`, sampled from `model` at `temperature`, with `draft_model` proposing
    n_draft tokens at a time (no reference counterpart: the reference decodes token by token).

    Both caches hold the same context, up to but without first_token, and are left holding it with
    first_token and every returned token but the last, so a call can go on from there. A round feeds the target the last token and the drafted ones in
    one forward pass, and kernels.verify_drafts decides how many of them are kept and which token follows;
    the caches forget the others, so they need truncate() (FullGPUCache) and, for a while, room for one token
    more than they are left with. Where the call fails they are left as they were. `generator` (on the model's
    device) draws the proposals and the uniforms.
    """
    for name, c in (("cache", cache), ("draft_cache", draft_cache)):
        if not hasattr(c, "truncate"):
            raise ValueError(f"speculative decoding takes rejected tokens back: {name} ({type(c).__name__}) has no truncate()")
    if n_draft < 1 or n_tokens < 0 or temperature <= 0:
        raise ValueError(f"n_draft {n_draft} is at least 1, n_tokens {n_tokens} at least 0, temperature {temperature} above 0")
    if cache is draft_cache:
        raise ValueError("the target and the draft need a cache each")
    if cache.get_seq_length() != draft_cache.get_seq_length():
        raise ValueError(f"the caches hold {cache.get_seq_length()} and {draft_cache.get_seq_length()} tokens")
    known = [m.get_input_embeddings().num_embeddings for m in (model, draft_model)]
    drawn = [m.config.get_text_config().vocab_size for m in (model, draft_model)]
    if drawn[0] != drawn[1] or min(known) < drawn[0]:  # a token of one model has to be an index into the other's embedding
        raise ValueError(f"the models' vocabularies differ: embeddings of {known[0]} and {known[1]}, logits of {drawn[0]} and {drawn[1]} tokens")
    if not 0 <= first_token < min(known):
        raise ValueError(f"first_token {first_token} is outside the vocabulary of {min(known)}")
    from lazykv_b200 import kernels

    def probabilities(m: PreTrainedModel, c: Cache, tokens: torch.Tensor, keep: int) -> torch.Tensor:
        logits = m(input_ids=tokens, past_key_values=c, use_cache=True, logits_to_keep=keep, **cache_model_kwargs(c)).logits
        return torch.softmax(logits.float() / temperature, dim=-1)

    res = SpeculativeResult(tokens=[])
    dev, start = model.device, cache.get_seq_length()
    behind = [first_token]  # returned tokens that the draft's cache does not hold yet, the target's but the last
    try:
        while len(res.tokens) < n_tokens:
            held = cache.get_seq_length()
            k = min(n_draft, n_tokens - len(res.tokens))
            fed, rows, drafted = torch.tensor([behind], dtype=torch.long, device=dev), [], []
            for _ in range(k):
                rows.append(probabilities(draft_model, draft_cache, fed, 1)[:, -1])
                fed = torch.multinomial(rows[-1], 1, generator=generator)
                drafted.append(fed)
            tokens = torch.cat(drafted, dim=1)
            target = probabilities(model, cache, torch.cat([torch.tensor([behind[-1:]], dtype=torch.long, device=dev), tokens], dim=1), k + 1)
            uniforms = torch.rand((1, k + 1), device=dev, generator=generator)
            kept, following = kernels.verify_drafts(target, torch.stack(rows, dim=1), tokens, uniforms)
            decided = torch.cat([kept.long(), following, tokens[0]]).tolist()  # one copy to the host per round
            n, nxt = decided[0], decided[1]
            if nxt < 0:
                raise RuntimeError("the target's probabilities have no finite, positive sum")
            res.drafted += k
            res.kept += n
            new = decided[2 : 2 + n] + [nxt]
            cache.truncate(held + 1 + n)  # the last token of the round before, and the drafted tokens that were kept
            draft_cache.truncate(min(held + 1 + n, draft_cache.get_seq_length()))
            # With all k kept the draft has not seen the last of them.
            behind = new[-2:] if n == k else new[-1:]
            res.tokens += new
        if len(res.tokens) > n_tokens:  # the token after n_tokens kept ones
            res.tokens = res.tokens[:n_tokens]
            cache.truncate(cache.get_seq_length() - 1)
            draft_cache.truncate(cache.get_seq_length())
        if draft_cache.get_seq_length() < cache.get_seq_length():
            probabilities(draft_model, draft_cache, torch.tensor([behind[:1]], dtype=torch.long, device=dev), 1)
    except BaseException:
        for c in (cache, draft_cache):
            c.truncate(start)
        raise
    return res
