"""A batch of sequences that share a prompt, decoded together: one layer's KV in pages, the prompt's
held and read once for all.

The reference decodes one sequence at a time; RaggedTier (ragged.py) batches sequences that have
nothing in common. Here every sequence is a fork of one prefix (a system prompt, a document, several
samples of one request). A step takes T new tokens of every sequence (one, or a token and those
drafted after it), writes their keys and values into the sequences' pages (kernels.paged_write),
attends their queries to the prefix and to their own tokens (kernels.prefix_attention), and, where
tokens were drafted, keeps those that the verification accepted (kernels.verify_drafts). A chunk takes any
number of new tokens of each sequence at once (a user's turn, a prompt of its own), straight from the
projections: normalised and rotated into the pages (kernels.paged_write_rotated) and attended
(kernels.chunk_attention).

A batch with track=True keeps to a budget: every step and chunk adds up the weight that each own token
gets from its queries (kernels.attention_sums), and evict() keeps the tokens of most weight of each head
(kernels.paged_evict) and frees the pages behind them.

Layout (one layer): pages [n_pages, h, 2, page, d] in the model dtype, or int8 codes with scales
[n_pages, h, 2, page] float32, one per token, head and key or value; page tables int32, -1 past a
sequence's own pages. The prefix's tokens are positions 0 .. prefix_len - 1 of its own page list and a
sequence's own tokens positions 0 .. of its; rotary positions are the caller's (from next_position() on), or
chunk()'s own. After evict() a sequence's slots are in no order and differ by head; `positions` says which
token is where.
"""

from __future__ import annotations

import itertools
from dataclasses import dataclass

import torch

from lazykv_b200 import kernels as K
from lazykv_b200._lib import require_cuda


@dataclass
class _Call:
    """What a tracked step or chunk added to the sums, as take_back() needs it."""

    sums: torch.Tensor  # [n, heads, slots] before it
    query: torch.Tensor  # the packed rows, and their lse, of sequences with a few new tokens
    lse: torch.Tensor
    scale: float
    cap: float


@dataclass
class _Part:
    """A sequence's part of its last call."""

    call: _Call
    at: int  # its place in call.sums
    row: int  # its first row of call.query, or -1: they are not kept
    held: int  # own tokens in front of the call's


class PagedBatch:
    """One layer's KV for up to `max_seqs` sequences of up to `max_tokens` own tokens behind one prefix.

    `n_pages` pages of `page` tokens hold the prefix and every sequence's own tokens; `quant` is "int8"
    or None (the model dtype). `track` keeps the sums and positions that evict() needs: `sums` [max_seqs,
    heads, slots] float32 and `positions` int32 alike, by sequence id. For take_back(), a tracked batch also holds
    each sequence's sums as they were before its last call, and that call's queries where they are up to MOST_DRAFTED.
    """

    MOST_DRAFTED = 64  # new tokens of a tracked call of which take_back() can take back a part

    def __init__(self, heads: int, group: int, head_dim: int, max_seqs: int, max_tokens: int, n_pages: int, page: int = 16, quant: str | None = "int8",
                 device: torch.device | str = "cuda", dtype: torch.dtype = torch.bfloat16, track: bool = False) -> None:
        if dtype != torch.bfloat16 or head_dim not in (64, 128) or page not in (16, 32, 64, 128):
            raise ValueError("a paged batch is bfloat16 with head_dim 64 or 128 and pages of 16, 32, 64 or 128 tokens")
        if quant not in (None, "int8"):
            raise ValueError(f"quant is 'int8' or None, got {quant!r}")
        if min(heads, group, max_seqs, max_tokens, n_pages) < 1:
            raise ValueError("heads, group, max_seqs, max_tokens and n_pages are at least 1")
        self.h, self.g, self.d, self.page = heads, group, head_dim, page
        dev = torch.device(device)
        if dev.type == "cuda" and dev.index is None:  # the current device now, whichever is current at a later call
            dev = torch.device("cuda", torch.cuda.current_device())
        self.dev, self.dtype = dev, dtype
        self.max_seqs, self.max_tokens = max_seqs, max_tokens
        self.cols = -(-max_tokens // page)
        self.pages = torch.zeros((n_pages, heads, 2, page, head_dim), dtype=torch.int8 if quant else dtype, device=self.dev)
        self.scales = torch.zeros((n_pages, heads, 2, page), device=self.dev) if quant else None
        self.table = torch.full((max_seqs, self.cols), -1, dtype=torch.int32, device=self.dev)
        self.prefix_table = torch.empty(0, dtype=torch.int32, device=self.dev)
        self.prefix_len = 0
        self.sums = torch.zeros((max_seqs, heads, self.cols * page), device=self.dev) if track else None
        self.positions = torch.full((max_seqs, heads, self.cols * page), -1, dtype=torch.int32, device=self.dev) if track else None
        K.status_attach(self.pages.device)
        self._prefix_pages: list[int] = []
        self._free_pages = list(range(n_pages - 1, -1, -1))
        self._free_seqs = list(range(max_seqs - 1, -1, -1))
        self.lengths: dict[int, int] = {}  # own tokens of each live sequence
        self._dropped: dict[int, int] = {}  # tokens that evict() has dropped of it
        self._settled: dict[int, int] = {}  # its tokens that evict() may have moved
        self._pages_of: dict[int, list[int]] = {}
        self._last: dict[int, _Part] = {}  # of a tracked batch

    # -- the prefix and the sequences -------------------------------------------------------------------

    def _take(self, n: int) -> list[int]:
        if n > len(self._free_pages):
            raise RuntimeError(f"cache full: {n} pages wanted, {len(self._free_pages)} free")
        return [self._free_pages.pop() for _ in range(n)]

    def _kv(self, keys: torch.Tensor, values: torch.Tensor) -> None:
        require_cuda(keys, values)
        if keys.dim() != 3 or keys.shape[0] != self.h or keys.shape[2] != self.d or keys.dtype != self.dtype or values.shape != keys.shape:
            raise ValueError(f"expected [{self.h}, L, {self.d}] {self.dtype} keys and values")

    def set_prefix(self, keys: torch.Tensor, values: torch.Tensor) -> None:
        """The prompt's KV [h, L, d] (any L, 0 too), in place of an earlier prompt's; no sequence may be live."""
        self._kv(keys, values)
        if self.lengths:
            raise RuntimeError(f"{len(self.lengths)} sequences were forked from the present prefix")
        n = -(-keys.shape[1] // self.page)
        if n > len(self._free_pages) + len(self._prefix_pages):
            raise RuntimeError(f"cache full: {n} pages wanted, {len(self._free_pages) + len(self._prefix_pages)} free")
        free = list(self._free_pages)
        self._free_pages.extend(reversed(self._prefix_pages))
        try:
            pages = self._take(n)
            table = torch.tensor(pages, dtype=torch.int32, device=self.dev)
            if n:
                self._write(keys, values, table.view(1, n))
        except BaseException:  # refused before anything was written: the earlier prompt stays
            self._free_pages = free
            raise
        self._prefix_pages, self.prefix_table, self.prefix_len = pages, table, keys.shape[1]

    def _write(self, keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor) -> None:
        zero = torch.zeros(1, dtype=torch.int32, device=self.dev)
        K.paged_write(keys.transpose(0, 1).unsqueeze(0), values.transpose(0, 1).unsqueeze(0), self.pages, table, zero, scales=self.scales)

    def fork(self) -> int:
        """A new sequence behind the prefix, without tokens of its own; returns its id."""
        if not self._free_seqs:
            raise RuntimeError(f"all {self.max_seqs} sequences are taken")
        s = self._free_seqs.pop()
        self.lengths[s], self._pages_of[s], self._dropped[s], self._settled[s] = 0, [], 0, 0
        return s

    def drop(self, s: int) -> None:
        """Retire sequence `s`: its pages and its id are free again."""
        del self.lengths[s], self._dropped[s], self._settled[s]
        self._last.pop(s, None)
        self._free_pages.extend(reversed(self._pages_of.pop(s)))
        self.table[s].fill_(-1)
        self._free_seqs.append(s)

    def _reserve(self, seq_ids: list[int], counts: list[int]) -> None:
        """Pages for counts[i] more tokens of every sequence, or of none where they do not suffice."""
        rows, cols, new = [], [], []
        for s, t in zip(seq_ids, counts):
            if self.lengths[s] + t > self.max_tokens:
                raise RuntimeError(f"sequence {s} is at {self.lengths[s]} of its {self.max_tokens} tokens: no room for {t}")
            for c in range(len(self._pages_of[s]), -(-(self.lengths[s] + t) // self.page)):
                rows.append(s)
                cols.append(c)
        if rows:
            new = self._take(len(rows))
            for s, page in zip(rows, new):
                self._pages_of[s].append(page)
            at = self._to_device(torch.tensor([rows, cols, new], pin_memory=True))
            self.table[at[0], at[1]] = at[2].to(torch.int32)

    def _to_device(self, pinned: torch.Tensor) -> torch.Tensor:
        """A copy that the stream orders and the host does not wait for (torch keeps the pinned block until it is done)."""
        return pinned.to(self.dev, non_blocking=True)

    # -- the decode step ----------------------------------------------------------------------------------

    def step(self, seq_ids: list[int], query: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, scale: float,
             out_dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """T new tokens of every sequence: keys / values [n, T, h, d] are written, and query [n, T, h * g, d]
        attends the prefix and the sequences' own tokens, each position those up to itself. Returns
        (out [n, T, h * g, d], lse [n, T, h * g] float32)."""
        K.raise_on_status("PagedBatch.step")  # an earlier step's wait that ran out (not synchronised)
        n = len(seq_ids)
        if len(set(seq_ids)) != n:
            raise ValueError(f"a sequence is named twice in {seq_ids}")
        if keys.dim() != 4 or keys.shape[0] != n or keys.shape[2:] != (self.h, self.d) or values.shape != keys.shape or keys.dtype != self.dtype:
            raise ValueError(f"expected keys and values [{n}, T, {self.h}, {self.d}] {self.dtype}")
        t = keys.shape[1]
        if query.shape != (n, t, self.h * self.g, self.d):
            raise ValueError(f"expected query [{n}, {t}, {self.h * self.g}, {self.d}], got {tuple(query.shape)}")
        require_cuda(query, keys, values)
        self._reserve(seq_ids, [t] * n)
        lens = [self.lengths[s] for s in seq_ids]
        first = [self.next_position(s) for s in seq_ids]
        ints = self._to_device(torch.tensor([seq_ids, lens, [x + t for x in lens], first], dtype=torch.int32, pin_memory=True))
        table = self.table.index_select(0, ints[0])
        K.paged_write(keys, values, self.pages, table, ints[1], scales=self.scales)
        done = K.prefix_attention(query, self.pages, table, ints[2], self.prefix_table, self.prefix_len, scale, scales=self.scales, out_dtype=out_dtype)
        if self.sums is not None and n * t:
            offsets = torch.arange(0, n * t + 1, t, dtype=torch.int32, device=self.dev)
            place = torch.arange(t, dtype=torch.int32, device=self.dev).repeat(n)
            rows = query.reshape(n * t, -1, self.d)
            last = self._track(ints[0], place, ints[1].repeat_interleave(t), ints[3].repeat_interleave(t), t, rows, done[1].view(n * t, -1), table, ints[2], offsets, scale, 0.0)
            self._note(seq_ids, [t] * n, last, rows, done[1].view(n * t, -1), scale, 0.0)
        for s in seq_ids:  # behind the calls: a refused step leaves the sequences as they were
            self.lengths[s] += t
        return done

    def next_position(self, s: int) -> int:
        """The position of sequence `s`'s next token, to which step()'s caller rotates it (chunk() does so itself): behind the
        prefix and all tokens of its own, those that evict() dropped too."""
        return self.prefix_len + self._dropped[s] + self.lengths[s]

    def _track(self, ids: torch.Tensor, place: torch.Tensor, held: torch.Tensor, first: torch.Tensor, counts: int | torch.Tensor, query: torch.Tensor, lse: torch.Tensor,
               table: torch.Tensor, lens: torch.Tensor, offsets: torch.Tensor, scale: float, cap: float) -> torch.Tensor:
        """Adds the weights of packed queries to the sums, and notes the new tokens' positions (row i is token place[i] of a
        chunk behind held[i] others, at position first[i] + place[i]). Returns the sums [n, heads, slots] as they were."""
        owner = ids.repeat_interleave(counts, output_size=place.numel())
        self.positions[owner.long(), :, (held + place).long()] = (first + place)[:, None]
        before = self.sums.index_select(0, ids)
        self.sums.index_copy_(0, ids.long(), K.attention_sums(query, lse, self.pages, table, lens, offsets, scale, sums=before, cap=cap, scales=self.scales))
        return before

    def _note(self, seq_ids: list[int], counts: list[int], before: torch.Tensor, query: torch.Tensor, lse: torch.Tensor, scale: float, cap: float) -> None:
        """Keeps what take_back() needs of a call's packed rows (before the lengths grow)."""
        query, lse, ends = query.detach(), lse.detach(), [0, *itertools.accumulate(counts)]
        few = [i for i, t in enumerate(counts) if 1 < t <= self.MOST_DRAFTED]  # (of one token all or none stays)
        if len(few) == len(counts):  # (copies: the caller has both tensors too)
            query, lse, first = query.clone(), lse.clone(), dict(enumerate(ends))
        else:
            query, lse = (torch.cat([x[:0], *(x[ends[i] : ends[i + 1]] for i in few)]) for x in (query, lse))
            first = dict(zip(few, itertools.accumulate((counts[i] for i in few), initial=0)))
        call = _Call(before, query, lse, scale, cap)
        for i, (s, t) in enumerate(zip(seq_ids, counts)):
            if t:
                self._last[s] = _Part(call, i, first.get(i, -1), self.lengths[s])

    def chunk(self, seq_ids: list[int], counts: list[int], query: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, scale: float,
              frequencies: torch.Tensor | None = None, q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
              interleaved: bool = False, cap: float = 0.0) -> tuple[torch.Tensor, torch.Tensor]:
        """counts[i] new tokens (0 too) of sequence seq_ids[i], packed in this order: query [rows, h * g, d], keys and values
        [rows, h, d] as the projections leave them. Queries and keys are normalised (where weights are given) and rotated
        by `frequencies` (none: not at all) to the sequences' next positions behind the prefix, keys and values written, and
        the queries attend the prefix and their sequences' tokens up to themselves. Returns (out [rows, h * g, d] bfloat16,
        lse [rows, h * g] float32)."""
        K.raise_on_status("PagedBatch.chunk")  # an earlier call's wait that ran out (not synchronised)
        n, rows = len(seq_ids), sum(counts)
        if len(set(seq_ids)) != n or len(counts) != n or min(counts, default=0) < 0:
            raise ValueError(f"expected a count of new tokens for each of the sequences {seq_ids}, each named once; got {counts}")
        if keys.shape != (rows, self.h, self.d) or values.shape != keys.shape or keys.dtype != self.dtype or query.shape != (rows, self.h * self.g, self.d):
            raise ValueError(f"expected query [{rows}, {self.h * self.g}, {self.d}], keys and values [{rows}, {self.h}, {self.d}] {self.dtype}")
        require_cuda(query, keys, values)
        self._reserve(seq_ids, counts)
        held = [self.lengths[s] for s in seq_ids]
        first = [self.next_position(s) for s in seq_ids]
        ends = [sum(counts[:i]) for i in range(n + 1)]
        ints = self._to_device(torch.tensor([seq_ids + [0], held + [0], [x + t for x, t in zip(held, counts)] + [0], first + [0], counts + [0], ends], dtype=torch.int32, pin_memory=True))
        ids, lens, offsets = ints[0, :n], ints[2, :n], ints[5]
        table = self.table.index_select(0, ids)
        place = torch.arange(rows, dtype=torch.int32, device=self.dev) - offsets[:n].repeat_interleave(ints[4, :n], output_size=rows)
        start = ints[3, :n].repeat_interleave(ints[4, :n], output_size=rows)
        if frequencies is None:
            frequencies = torch.empty(0, device=self.dev)
        query = K.paged_write_rotated(query, keys, values, start + place, frequencies, self.pages, table, lens, offsets, scales=self.scales, q_weight=q_weight,
                                      k_weight=k_weight, eps=eps, interleaved=interleaved)
        done = K.chunk_attention(query, self.pages, table, lens, offsets, scale, scales=self.scales, prefix_table=self.prefix_table, prefix_len=self.prefix_len, cap=cap)
        if self.sums is not None and rows:
            before = ints[1, :n].repeat_interleave(ints[4, :n], output_size=rows)
            last = self._track(ids, place, before, start, ints[4, :n], query, done[1], table, lens, offsets, scale, cap)
            self._note(seq_ids, counts, last, query, done[1], scale, cap)
        for s, t in zip(seq_ids, counts):  # behind the calls: a refused chunk leaves the sequences as they were
            self.lengths[s] += t
        return done

    def evict(self, seq_ids: list[int], keep: int, recent: int = 0, sinks: int = 0) -> None:
        """Cuts the own tokens of these sequences down to `keep` a head: the first `sinks` and the last `recent` of the sequence
        (by position) and then those of most weight so far. Pages behind them are free again; shorter sequences stay as they
        are. Needs track=True."""
        if self.sums is None:
            raise RuntimeError("evict() ranks tokens by their weights: the batch was made without track=True")
        if len(set(seq_ids)) != len(seq_ids) or keep < 1 or min(recent, sinks) < 0 or recent + sinks > keep:
            raise ValueError(f"expected sequences named once and a budget that holds the {sinks} first and {recent} last tokens, got {seq_ids} and {keep}")
        long = [s for s in seq_ids if self.lengths[s] > keep]
        if not long:
            return
        ints = self._to_device(torch.tensor([long, [self.lengths[s] for s in long], [self.next_position(s) - recent for s in long]], dtype=torch.int32, pin_memory=True))
        sums, positions = self.sums.index_select(0, ints[0]), self.positions.index_select(0, ints[0])
        K.paged_evict(self.pages, self.table.index_select(0, ints[0]), ints[1], sums, positions, keep, since=ints[2], sinks=self.prefix_len + sinks, scales=self.scales,
                      out=(sums, positions))
        at = ints[0].long()
        self.sums.index_copy_(0, at, sums)
        self.positions.index_copy_(0, at, positions)
        cols = -(-keep // self.page)
        self.table[:, cols:].index_fill_(0, at, -1)
        for s in long:
            self._free_pages.extend(reversed(self._pages_of[s][cols:]))
            del self._pages_of[s][cols:]
            self._dropped[s] += self.lengths[s] - keep
            self.lengths[s] = self._settled[s] = keep
            self._last.pop(s, None)

    def take_back(self, s: int | list[int], tokens: int | list[int]) -> None:
        """Forget the last `tokens` own tokens of sequence `s` (drafted ones that were rejected), or tokens[i] of each
        sequence s[i] of a list; their pages stay the sequences' and are written again. What evict() has moved cannot be taken back.

        With track=True the weights that the forgotten tokens' queries gave to the others leave the sums: these are as if
        only the tokens that stay had come. That holds for tokens of the sequence's last step or chunk, all of them or, of
        a call of up to MOST_DRAFTED of its tokens, a part; others are refused."""
        ids = list(s) if isinstance(s, (list, tuple)) else [s]
        counts = list(tokens) if isinstance(tokens, (list, tuple)) else [tokens]
        if len(set(ids)) != len(ids) or len(counts) != len(ids):
            raise ValueError(f"expected a count of tokens for each of the sequences {ids}, each named once; got {counts}")
        calls: dict[int, list[tuple[int, int, _Part]]] = {}  # by call: sequence, tokens of it that stay
        for i, n in zip(ids, counts):
            part = self._last.get(i)
            most = self.lengths[i] - (self._settled[i] if self.sums is None else part.held if part is not None else self.lengths[i])
            if not 0 <= n <= most:
                raise ValueError(f"sequence {i} has {most} tokens to take back, not {n}")
            if part is not None and n:
                if n < most and part.row < 0:
                    raise ValueError(f"of a tracked chunk of more than {self.MOST_DRAFTED} tokens all are taken back or none, not {n} of {most}")
                calls.setdefault(id(part.call), []).append((i, most - n, part))
        for parts in calls.values():
            self._add_again(parts[0][2].call, parts)
        for i, n in zip(ids, counts):
            self.lengths[i] -= n

    def _add_again(self, call: _Call, parts: list[tuple[int, int, _Part]]) -> None:
        """Sums of sequences as if only the first so many tokens of their part of `call` had come."""
        n = len(parts)
        kept = [stay for _, stay, _ in parts]
        ends = [0, *itertools.accumulate(kept)]
        rows = [part.row + t for _, stay, part in parts for t in range(stay)]
        flat = [i for i, _, _ in parts] + [part.at for _, _, part in parts] + [part.held + stay for _, stay, part in parts] + ends + rows
        ints = self._to_device(torch.tensor(flat, dtype=torch.int32, pin_memory=True))
        ids, at, lens, offsets, row = ints.split([n, n, n, n + 1, len(rows)])
        sums = call.sums.index_select(0, at)
        if rows:
            K.attention_sums(call.query.index_select(0, row), call.lse.index_select(0, row), self.pages, self.table.index_select(0, ids), lens, offsets, call.scale, sums=sums,
                             cap=call.cap, scales=self.scales, out=sums)
        assert self.sums is not None
        self.sums.index_copy_(0, ids.long(), sums)

    def read(self, s: int, dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The whole sequence, prefix and own tokens, as (keys, values) [h, L, d] in the model dtype (or `dtype`,
        of int8 pages): what a step attends, say for RaggedTier.add (in the slots' order)."""
        dtype = dtype or self.dtype
        zero = torch.zeros(1, dtype=torch.int32, device=self.dev)
        parts = []
        for table, n in ((self.prefix_table.view(1, -1), self.prefix_len), (self.table[s : s + 1], self.lengths[s])):
            parts.append(K.paged_read(self.pages, table, zero, n, scales=self.scales, dtype=dtype))
        return tuple(torch.cat([p[i][0] for p in parts]).transpose(0, 1).contiguous() for i in (0, 1))  # type: ignore[return-value]
