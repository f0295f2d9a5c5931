"""The paged batch as it is used: a prompt, forks, steps of one and of several drafted tokens with their
verification, tokens taken back, sequences dropped and replaced, against the definition in 64 bits over a
dense copy of everything that was written; and speculative decoding of a small model."""

from __future__ import annotations

import pytest
import torch

from tests.paged_plain import quantise_rows, verify

pytestmark = pytest.mark.gpu

H, G, D = 2, 4, 64


def _held(x: torch.Tensor, int8: bool) -> torch.Tensor:
    """Rows [..., d] as the cache holds them, float64."""
    if not int8:
        return x.double()
    codes, s = quantise_rows(x)
    return codes.double() * s.double()[..., None]


def _dense(query: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    """One query position [h * g, d] over keys / values [L, h, d] float64: (out, sum p |v|)."""
    s = torch.einsum("hgd,nhd->hgn", query.double().view(H, G, D), keys) * scale
    p = torch.softmax(s, -1)
    return torch.einsum("hgn,nhd->hgd", p, values).reshape(H * G, D), torch.einsum("hgn,nhd->hgd", p, values.abs()).reshape(H * G, D)


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("prefix,page", [(0, 16), (37, 16), (300, 32)])
def test_steps_verify_take_back_and_fork_again(prefix: int, page: int, int8: bool) -> None:
    from lazykv_b200 import kernels as K
    from lazykv_b200.paged import PagedBatch

    gen = torch.Generator().manual_seed(prefix + page)
    batch = PagedBatch(H, G, D, max_seqs=6, max_tokens=80, n_pages=80, page=page, quant="int8" if int8 else None)
    rand = lambda *s: torch.randn(s, generator=gen).bfloat16()  # noqa: E731
    pk, pv = rand(H, prefix, D), rand(H, prefix, D)
    batch.set_prefix(pk.cuda(), pv.cuda())
    free = len(batch._free_pages)
    held = {}  # per sequence: keys, values [L, h, d] as written
    ids = [batch.fork() for _ in range(5)]
    for s in ids:
        held[s] = (rand(0, H, D), rand(0, H, D))
    vocab, scale = 50, D**-0.5
    for t in (1, 4, 1, 7, 3, 5):
        n = len(ids)
        q, k, v = rand(n, t, H * G, D), rand(n, t, H, D), rand(n, t, H, D)
        out, lse = batch.step(ids, q.cuda(), k.cuda(), v.cuda(), scale, out_dtype=torch.float32)
        for i, s in enumerate(ids):
            held[s] = (torch.cat([held[s][0], k[i]]), torch.cat([held[s][1], v[i]]))
            keys = _held(torch.cat([pk.transpose(0, 1), held[s][0]]), int8)
            values = _held(torch.cat([pv.transpose(0, 1), held[s][1]]), int8)
            for step in range(t):
                m = keys.shape[0] - t + 1 + step
                want, mass = _dense(q[i, step], keys[:m], values[:m], scale)
                # weights are rounded once to bfloat16 (2^-8 of the sum p |v|); the scores' float32 rounding is far below
                assert bool(((out[i, step].double().cpu() - want).abs() <= 1.02 * 2.0**-8 * mass + 1e-5).all())
        if t > 1:  # t - 1 drafted tokens: what the verification rejects is taken back
            target = torch.softmax(2 * torch.randn((n, t, vocab), generator=gen), -1)
            draft = torch.softmax(2 * torch.randn((n, t - 1, vocab), generator=gen), -1)
            tokens = torch.multinomial(draft.reshape(-1, vocab), 1, generator=gen).view(n, t - 1)
            u = torch.rand((n, t), generator=gen)
            kept, token = K.verify_drafts(target.cuda(), draft.cuda(), tokens.cuda(), u.cuda())
            want_kept, want_token = verify(target, draft, tokens, u)
            assert kept.tolist() == want_kept and token.tolist() == want_token
            for i, s in enumerate(ids):
                back = t - 1 - want_kept[i]
                batch.take_back(s, back)
                m = held[s][0].shape[0] - back
                held[s] = (held[s][0][:m], held[s][1][:m])
        if t == 7:  # a sequence ends, another takes its place
            batch.drop(ids[2])
            ids[2] = batch.fork()
            held[ids[2]] = (rand(0, H, D), rand(0, H, D))
    for s in ids:
        assert batch.lengths[s] == held[s][0].shape[0]
        k, v = batch.read(s)
        assert k.shape == (H, prefix + batch.lengths[s], D) and k.is_contiguous()
        for got, p, own in ((k, pk, held[s][0]), (v, pv, held[s][1])):
            want = _held(torch.cat([p.transpose(0, 1), own]), int8)
            err = (got.double().cpu().transpose(0, 1) - want).abs()
            assert bool((err <= (1.01 * 2.0**-8 if int8 else 0.0) * want.abs()).all())
        batch.drop(s)
    assert len(batch._free_pages) == free and int((batch.table >= 0).sum()) == 0
    # the prefix can be replaced now, by one that takes other pages
    batch.set_prefix(rand(H, 64, D).cuda(), rand(H, 64, D).cuda())
    assert batch.prefix_len == 64


def test_what_the_paged_batch_refuses() -> None:
    from lazykv_b200.paged import PagedBatch

    for bad in (dict(head_dim=96), dict(page=24), dict(quant="int4"), dict(dtype=torch.float32), dict(max_seqs=0)):
        with pytest.raises(ValueError):
            PagedBatch(**{**dict(heads=H, group=G, head_dim=D, max_seqs=2, max_tokens=32, n_pages=4), **bad})
    batch = PagedBatch(H, G, D, max_seqs=2, max_tokens=40, n_pages=4)
    x = torch.zeros((H, 20, D), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="CUDA"):
        batch.set_prefix(x.cpu(), x.cpu())
    with pytest.raises(RuntimeError, match="cache full"):
        batch.set_prefix(x.repeat(1, 4, 1), x.repeat(1, 4, 1))
    batch.set_prefix(x, x)  # two of the four pages
    a, b = batch.fork(), batch.fork()
    with pytest.raises(RuntimeError, match="taken"):
        batch.fork()
    with pytest.raises(RuntimeError, match="forked"):
        batch.set_prefix(x, x)
    q, kv = torch.zeros((2, 17, H * G, D), dtype=torch.bfloat16, device="cuda"), torch.zeros((2, 17, H, D), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="twice"):
        batch.step([a, a], q, kv, kv, 1.0)
    with pytest.raises(ValueError, match="expected query"):
        batch.step([a, b], q[:, :1], kv, kv, 1.0)
    with pytest.raises(RuntimeError, match="cache full"):  # four pages wanted, two free: nothing is taken
        batch.step([a, b], q, kv, kv, 1.0)
    assert len(batch._free_pages) == 2 and batch.lengths == {a: 0, b: 0}
    batch.step([a], q[:1], kv[:1], kv[:1], 1.0)
    with pytest.raises(ValueError, match="take back"):
        batch.take_back(a, 18)
    with pytest.raises(RuntimeError, match="no room"):
        batch.step([a], q[:1].repeat(1, 2, 1, 1), kv[:1].repeat(1, 2, 1, 1), kv[:1].repeat(1, 2, 1, 1), 1.0)


def test_a_refused_step_leaves_the_sequences_as_they_were() -> None:
    from lazykv_b200.paged import PagedBatch

    batch = PagedBatch(H, G, D, max_seqs=1, max_tokens=40, n_pages=4)
    a = batch.fork()
    q, kv = torch.zeros((1, 2, H * G, D), dtype=torch.bfloat16, device="cuda"), torch.zeros((1, 2, H, D), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="bfloat16"):
        batch.step([a], q.float(), kv, kv, 1.0)
    with pytest.raises((ValueError, TypeError)):
        batch.step([a], q, kv, kv, 1.0, out_dtype=torch.int8)
    assert batch.lengths == {a: 0}
    batch.step([a], q, kv, kv, 1.0)
    assert batch.lengths == {a: 2}


def test_the_wrappers_refuse_what_does_not_fit() -> None:
    from lazykv_b200 import kernels as K

    dev = "cuda"
    pages, scales = torch.zeros((4, H, 2, 16, D), dtype=torch.int8, device=dev), torch.zeros((4, H, 2, 16), device=dev)
    table, ints = torch.zeros((2, 3), dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    kv, q = torch.zeros((2, 1, H, D), dtype=torch.bfloat16, device=dev), torch.zeros((2, 1, H * G, D), dtype=torch.bfloat16, device=dev)
    bad_writes = [dict(values=kv[:, :, :1]), dict(keys=kv[0], values=kv[0]), dict(pages=pages.transpose(0, 1)), dict(scales=None), dict(scales=scales.half()),
                  dict(table=table.long()), dict(table=table[:1]), dict(table=table.t().contiguous().t()), dict(starts=ints.long()), dict(starts=ints[:1]),
                  dict(pages=pages.bfloat16()), dict(pages=pages.float(), scales=None), dict(keys=kv.transpose(2, 3).contiguous().transpose(2, 3)),
                  dict(starts=ints.cpu())]
    for bad in bad_writes:
        with pytest.raises(ValueError):
            K.paged_write(**{**dict(keys=kv, values=kv, pages=pages, table=table, starts=ints, scales=scales), **bad})
    out = torch.zeros((2, 1, H, D), dtype=torch.bfloat16, device=dev)
    bad_reads = [dict(n_tokens=-1), dict(dtype=torch.float16), dict(lens=ints.long()), dict(out=(out, out.float())), dict(out=(out, out[:1])),
                 dict(pages=pages.bfloat16(), scales=None, dtype=torch.float32)]
    for bad in bad_reads:
        with pytest.raises(ValueError):
            K.paged_read(**{**dict(pages=pages, table=table, starts=ints, n_tokens=1, scales=scales), **bad})
    bad_attends = [dict(query=q.float()), dict(query=q[0]), dict(query=q[:, :, :3]), dict(query=q[:1]), dict(lens=ints.float()), dict(prefix_table=table),
                   dict(prefix_len=49), dict(prefix_len=-1), dict(out=q.float(), out_dtype=torch.bfloat16), dict(out=q[:1]), dict(lse=torch.zeros(3, device=dev)),
                   dict(pages=pages.float(), scales=None), dict(out_dtype=torch.float16)]
    for bad in bad_attends:
        with pytest.raises(ValueError):
            K.prefix_attention(**{**dict(query=q, pages=pages, table=table, lens=ints, prefix_table=table[0], prefix_len=40, scale=1.0, scales=scales), **bad})
    p, tok, u = torch.zeros((2, 4, 9), device=dev), torch.zeros((2, 3), dtype=torch.int64, device=dev), torch.zeros((2, 4), device=dev)
    bad_verifies = [dict(target=p.half()), dict(target=p[:, :3]), dict(draft=p), dict(tokens=tok.int()), dict(uniforms=u[:, :3]), dict(uniforms=u.double()),
                    dict(target=p.transpose(1, 2).contiguous().transpose(1, 2))]
    for bad in bad_verifies:
        with pytest.raises(ValueError):
            K.verify_drafts(**{**dict(target=p, draft=p[:, :3], tokens=tok, uniforms=u), **bad})


# -- speculative decoding --------------------------------------------------------------------------------


@pytest.fixture(scope="module")
def tiny():  # noqa: ANN201
    from tests.tiny_model import make_tiny

    return make_tiny()


@pytest.mark.parametrize("n_draft,n_tokens", [(1, 9), (3, 10), (5, 1), (4, 0), (6, 23)])
@pytest.mark.parametrize("same", [True, False], ids=["own draft", "other draft"])
def test_speculative_decoding_takes_what_the_plain_verification_takes(tiny, monkeypatch, same: bool, n_draft: int, n_tokens: int) -> None:  # noqa: ANN001
    """The same tokens as with the verification's definition in its place (the generator draws the same numbers),
    the caches left with every token but the last, and holding what a prefill of those tokens holds."""
    from lazykv_b200 import kernels
    from lazykv_b200.cache import FullGPUCache
    from lazykv_b200.generate import prefill, speculative_decode
    from tests.tiny_model import CAP, prefilled

    cfg, model = tiny
    draft_model = model
    if not same:
        from transformers import LlamaForCausalLM

        torch.manual_seed(5)
        draft_model = LlamaForCausalLM(cfg)
        draft_model.set_attn_implementation(model.config._attn_implementation)
        draft_model = draft_model.to(dtype=torch.bfloat16).cuda().eval()

    def plain(target, draft, tokens, uniforms):  # noqa: ANN001, ANN202
        kept, token = verify(target.cpu(), draft.cpu(), tokens.cpu(), uniforms.cpu())
        return torch.tensor(kept, dtype=torch.int32, device="cuda"), torch.tensor(token, device="cuda")

    results = []
    for check in (None, plain):
        if check is not None:
            monkeypatch.setattr(kernels, "verify_drafts", check)
        ids, full, _ = prefilled(model, cfg)
        n = full.get_seq_length()
        draft_cache = FullGPUCache(cfg.num_hidden_layers, CAP)
        prefill(draft_model, draft_cache, ids[:, :n], chunk_size=32)
        gen = torch.Generator(device="cuda").manual_seed(n_draft)
        first = int(ids[0, n])
        res = speculative_decode(model, full, draft_model, draft_cache, first, n_tokens, n_draft, temperature=0.7, generator=gen)
        assert len(res.tokens) == n_tokens and 0 <= res.kept <= res.drafted
        assert full.get_seq_length() == n + n_tokens and draft_cache.get_seq_length() == full.get_seq_length()
        results.append((res.tokens, res.kept, res.drafted))
    monkeypatch.undo()
    assert results[0] == results[1]
    if n_tokens == 0:
        return
    # the cache holds the context, the first token and all but the last: one more forward pass from it and from a prefill
    context = torch.cat([ids[0, : n + 1], torch.tensor(results[0][0][:-1], dtype=torch.long, device="cuda")])[None]
    assert context.shape[1] == full.get_seq_length()
    fresh = FullGPUCache(cfg.num_hidden_layers, CAP)
    prefill(model, fresh, context, chunk_size=32)
    for a, b in zip(full.layers, fresh.layers):
        x, y = a.keys[:, :, : n + n_tokens].float(), b.keys[:, :, : n + n_tokens].float()
        # bfloat16 layers computed in other chunk sizes: a few roundings (2^-8 each) through four layers
        assert bool(((x - y).abs() <= 16 * 2.0**-8 * y.abs().amax()).all())


def test_speculative_decoding_refuses_caches_that_cannot_forget(tiny) -> None:  # noqa: ANN001
    from transformers.cache_utils import Cache

    from lazykv_b200.cache import FullGPUCache
    from lazykv_b200.generate import speculative_decode

    cfg, model = tiny
    full = FullGPUCache(cfg.num_hidden_layers, 64)

    class Fixed(Cache):
        def __init__(self) -> None:
            super().__init__(layers=[])

    with pytest.raises(ValueError, match="truncate"):
        speculative_decode(model, Fixed(), model, full, 1, 4, 2)
    for bad in (dict(n_draft=0), dict(n_tokens=-1), dict(temperature=0.0)):
        with pytest.raises(ValueError, match="at least"):
            speculative_decode(model, full, model, FullGPUCache(cfg.num_hidden_layers, 64), **{**dict(first_token=1, n_tokens=4, n_draft=2), **bad})
