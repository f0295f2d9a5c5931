"""PagedBatch and speculative decoding around refused calls, and where a step's work is ordered."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

H, G, D = 2, 4, 64


@pytest.mark.parametrize("quant", ["int8", None])
def test_a_refused_prefix_leaves_the_earlier_one(quant: str | None) -> None:
    from lazykv_b200.paged import PagedBatch

    gen = torch.Generator().manual_seed(1)
    rand = lambda *s: torch.randn(s, generator=gen).bfloat16().cuda()  # noqa: E731
    batch = PagedBatch(H, G, D, max_seqs=2, max_tokens=40, n_pages=8, quant=quant)
    batch.set_prefix(rand(H, 50, D), rand(H, 50, D))
    q, k, v = rand(1, 1, H * G, D), rand(1, 1, H, D), rand(1, 1, H, D)

    def step() -> tuple[torch.Tensor, torch.Tensor]:
        s = batch.fork()
        done = batch.step([s], q, k, v, 0.125)
        batch.drop(s)
        return done

    want, table, free = step(), batch.prefix_table.tolist(), sorted(batch._free_pages)
    x = rand(H, 37, D)
    turned = rand(H, D, 37).transpose(1, 2)  # channels that are not contiguous
    for keys, values in ((x, x.float()), (turned, x), (x, turned)):
        with pytest.raises(ValueError):
            batch.set_prefix(keys, values)
        assert batch.prefix_len == 50 and batch.prefix_table.tolist() == table and sorted(batch._free_pages) == free
        got = step()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    batch.set_prefix(x, x)
    assert batch.prefix_len == 37 and len(batch._free_pages) == 5


def test_a_step_does_not_wait_for_the_stream() -> None:
    """Steps that take new pages and steps that do not, behind work that is still running: none synchronises, and each
    result is the one that the same steps give when every one is waited for."""
    from lazykv_b200.paged import PagedBatch

    gen = torch.Generator().manual_seed(2)
    rand = lambda *s: torch.randn(s, generator=gen).bfloat16().cuda()  # noqa: E731
    pk, pv = rand(H, 100, D), rand(H, 100, D)
    steps = [(rand(3, t, H * G, D), rand(3, t, H, D), rand(3, t, H, D)) for t in (1, 15, 1, 4, 30, 1)]
    big = torch.randn((4096, 4096), device="cuda")
    results = []
    for waited in (True, False):
        batch = PagedBatch(H, G, D, max_seqs=3, max_tokens=64, n_pages=30)
        batch.set_prefix(pk, pv)
        ids = [batch.fork() for _ in range(3)]
        got = []
        torch.cuda.synchronize()
        torch.cuda.set_sync_debug_mode("default" if waited else "error")
        try:
            for x in steps:
                if not waited:
                    big = big @ big * 1e-4
                got.append(batch.step(ids, *x, 0.125))
                if waited:
                    torch.cuda.synchronize()
        finally:
            torch.cuda.set_sync_debug_mode("default")
        torch.cuda.synchronize()
        results.append(got)
    for (a, c), (e, f) in zip(*results):
        assert torch.equal(a, e) and torch.equal(c, f)


def test_a_batch_stays_on_the_device_that_was_current_when_it_was_made() -> None:
    from lazykv_b200.paged import PagedBatch

    batch = PagedBatch(H, G, D, max_seqs=1, max_tokens=16, n_pages=2, device="cuda")
    assert batch.dev == batch.pages.device == batch.table.device and batch.dev.index == torch.cuda.current_device()


def test_speculative_decoding_that_fails_leaves_the_caches_as_they_were(monkeypatch) -> None:  # noqa: ANN001
    """A draft of another vocabulary, a cache without room, a verification that finds no weight after some rounds: the
    caches hold the context again, and the call that follows returns what it returns without the failed one."""
    from transformers import LlamaForCausalLM

    from lazykv_b200 import kernels
    from lazykv_b200.cache import FullGPUCache
    from lazykv_b200.generate import prefill, speculative_decode
    from tests.tiny_model import CAP, make_tiny, prefilled

    cfg, model = make_tiny()
    wide = type(cfg)(**{**cfg.to_dict(), "vocab_size": cfg.vocab_size + 8})
    torch.manual_seed(6)
    other = LlamaForCausalLM(wide)
    other.set_attn_implementation(model.config._attn_implementation)
    other = other.to(dtype=torch.bfloat16).cuda().eval()

    def caches(draft, room: int = CAP):  # noqa: ANN001, ANN202
        ids, full, _ = prefilled(model, cfg)
        n = full.get_seq_length()
        cache = FullGPUCache(cfg.num_hidden_layers, room)
        prefill(draft, cache, ids[:, :n], chunk_size=32)
        return int(ids[0, n]), n, full, cache

    def decode(first: int, full, draft, cache):  # noqa: ANN001, ANN202
        return speculative_decode(model, full, draft, cache, first, 9, 3, generator=torch.Generator(device="cuda").manual_seed(1)).tokens

    first, n, full, cache = caches(model)
    want = decode(first, full, model, cache)

    first, n, full, cache = caches(other)
    with pytest.raises(ValueError, match="vocabularies"):  # refused before any token reaches the other's embedding
        decode(first, full, other, cache)
    assert full.get_seq_length() == n and cache.get_seq_length() == n
    own = FullGPUCache(cfg.num_hidden_layers, CAP)
    prefill(model, own, prefilled(model, cfg)[0][:, :n], chunk_size=32)
    assert decode(first, full, model, own) == want

    first, n, full, cache = caches(model, room=prefilled(model, cfg)[1].get_seq_length() + 4)
    with pytest.raises(Exception):  # noqa: B017 - the draft's cache is full after a round or two
        decode(first, full, model, cache)
    assert full.get_seq_length() == n and cache.get_seq_length() == n

    first, n, full, cache = caches(model)
    rounds, real = [], kernels.verify_drafts

    def runs_out(*args):  # noqa: ANN002, ANN202
        rounds.append(1)
        kept, token = real(*args)
        return kept, token if len(rounds) < 2 else torch.full_like(token, -1)

    monkeypatch.setattr(kernels, "verify_drafts", runs_out)
    with pytest.raises(RuntimeError, match="positive sum"):
        decode(first, full, model, cache)
    monkeypatch.undo()
    assert full.get_seq_length() == n and cache.get_seq_length() == n
    assert decode(first, full, model, cache) == want
