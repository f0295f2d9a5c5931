"""A batch of sequences that share a prompt, decoded together: one layer's KV in pages, the prompt's
held and read once for all.

The reference decodes one sequence at a time; RaggedTier (ragged.py) batches sequences that have
nothing in common. Here every sequence is a fork of one prefix (a system prompt, a document, several
samples of one request). A step takes T new tokens of every sequence (one, or a token and those
drafted after it), writes their keys and values into the sequences' pages (kernels.paged_write),
attends their queries to the prefix and to their own tokens (kernels.prefix_attention), and, where
tokens were drafted, keeps those that the verification accepted (kernels.verify_drafts).

Layout (one layer): pages [n_pages, h, 2, page, d] in the model dtype, or int8 codes with scales
[n_pages, h, 2, page] float32, one per token, head and key or value; page tables int32, -1 past a
sequence's own pages. The prefix's tokens are positions 0 .. prefix_len - 1 of its own page list and a
sequence's own tokens positions 0 .. of its; rotary positions are the caller's (prefix_len + position).
"""

from __future__ import annotations

import torch

from lazykv_b200 import kernels as K
from lazykv_b200._lib import require_cuda


class PagedBatch:
    """One layer's KV for up to `max_seqs` sequences of up to `max_tokens` own tokens behind one prefix.

    `n_pages` pages of `page` tokens hold the prefix and every sequence's own tokens; `quant` is "int8"
    or None (the model dtype).
    """

    def __init__(self, heads: int, group: int, head_dim: int, max_seqs: int, max_tokens: int, n_pages: int, page: int = 16, quant: str | None = "int8",
                 device: torch.device | str = "cuda", dtype: torch.dtype = torch.bfloat16) -> None:
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
        K.status_attach(self.pages.device)
        self._prefix_pages: list[int] = []
        self._free_pages = list(range(n_pages - 1, -1, -1))
        self._free_seqs = list(range(max_seqs - 1, -1, -1))
        self.lengths: dict[int, int] = {}  # own tokens of each live sequence
        self._pages_of: dict[int, list[int]] = {}

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
        self.lengths[s], self._pages_of[s] = 0, []
        return s

    def drop(self, s: int) -> None:
        """Retire sequence `s`: its pages and its id are free again."""
        del self.lengths[s]
        self._free_pages.extend(reversed(self._pages_of.pop(s)))
        self.table[s].fill_(-1)
        self._free_seqs.append(s)

    def _reserve(self, seq_ids: list[int], t: int) -> None:
        """Pages for t more tokens of every sequence, or of none where they do not suffice."""
        rows, cols, new = [], [], []
        for s in seq_ids:
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
        self._reserve(seq_ids, t)
        lens = [self.lengths[s] for s in seq_ids]
        ints = self._to_device(torch.tensor([seq_ids, lens, [x + t for x in lens]], dtype=torch.int32, pin_memory=True))
        table = self.table.index_select(0, ints[0])
        K.paged_write(keys, values, self.pages, table, ints[1], scales=self.scales)
        done = K.prefix_attention(query, self.pages, table, ints[2], self.prefix_table, self.prefix_len, scale, scales=self.scales, out_dtype=out_dtype)
        for s in seq_ids:  # behind the calls: a refused step leaves the sequences as they were
            self.lengths[s] += t
        return done

    def take_back(self, s: int, tokens: int) -> None:
        """Forget the last `tokens` own tokens of sequence `s` (drafted ones that were rejected); their pages stay
        the sequence's and are written again."""
        if not 0 <= tokens <= self.lengths[s]:
            raise ValueError(f"sequence {s} has {self.lengths[s]} tokens, not {tokens} to take back")
        self.lengths[s] -= tokens

    def read(self, s: int, dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The whole sequence, prefix and own tokens, as (keys, values) [h, L, d] in the model dtype (or `dtype`,
        of int8 pages): what a step attends, say for RaggedTier.add."""
        dtype = dtype or self.dtype
        zero = torch.zeros(1, dtype=torch.int32, device=self.dev)
        parts = []
        for table, n in ((self.prefix_table.view(1, -1), self.prefix_len), (self.table[s : s + 1], self.lengths[s])):
            parts.append(K.paged_read(self.pages, table, zero, n, scales=self.scales, dtype=dtype))
        return tuple(torch.cat([p[i][0] for p in parts]).transpose(0, 1).contiguous() for i in (0, 1))  # type: ignore[return-value]
