"""The operators of a paged cache that takes prompts in chunks and keeps to a budget, as they are measured.

New tokens come packed, [rows, heads, dim]: sequence b's are rows offsets[b] .. offsets[b + 1] - 1 and the
last of its lens[b] tokens in the cache. Four kinds of case:

  rotate  paged_write_rotated: queries and keys normalised per head and rotated, keys and values written into
          the pages (and, of int8 pages, the new tokens read back as the values that their codes stand for)
  attend  chunk_attention: the chunks' queries over what their sequences hold, and over a shared prefix
  sums    attention_sums: the weight that every cached token got from the chunks' queries
  evict   paged_evict: each head keeps the tokens of most weight (of int8 pages, what is kept is read back)

`own` selects the framework's kernels; otherwise `run` computes the plain form in elementary torch
operations.
"""

import torch

own = False

FLT_MIN = 1.1754943508222875e-38  # the least normal float32: the floor of a quantisation scale
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # One decode step of a batch of 64: the smallest call, launch latency counts.
        {"name": "rotate decode 64 int8", "op": "rotate", "batch": 64, "chunk": 1, "held": 9000, "heads": 8, "group": 4, "dim": 128, "page": 16, "cache": "int8", "input": "bf16",
         "rotated": 128, "interleaved": False, "norm": True},
        # Ragged chunks of a float32 model, half of a head rotated in neighbouring pairs, no norms.
        {"name": "rotate 5 x 700 f32", "op": "rotate", "batch": 5, "chunk": 701, "held": 3001, "heads": 4, "group": 3, "dim": 64, "page": 32, "cache": "model", "input": "f32",
         "rotated": 32, "interleaved": True, "norm": False},
        # A whole prompt into int8 pages.
        {"name": "rotate prompt 32K int8", "op": "rotate", "batch": 1, "chunk": 32768, "held": 0, "heads": 8, "group": 4, "dim": 128, "page": 64, "cache": "int8", "input": "bf16",
         "rotated": 128, "interleaved": False, "norm": True},
        # A short turn of one conversation.
        {"name": "attend 17 on 300", "op": "attend", "batch": 1, "chunk": 17, "context": 300, "prefix": 0, "heads": 8, "group": 4, "dim": 64, "page": 16, "cache": "bf16", "cap": 0.0},
        # A mixed batch of chunks of 0 to 96 tokens behind a shared prompt, capped scores.
        {"name": "attend 24 mixed on 8191", "op": "attend", "batch": 24, "chunk": 96, "context": 500, "prefix": 8191, "heads": 8, "group": 4, "dim": 64, "page": 32, "cache": "bf16", "cap": 50.0},
        # A chunk of a long prompt in int8 pages.
        {"name": "attend 2048 on 16K int8", "op": "attend", "batch": 1, "chunk": 2048, "context": 16384, "prefix": 0, "heads": 8, "group": 4, "dim": 128, "page": 64, "cache": "int8", "cap": 0.0},
        # The largest: a chunk of 4,096 tokens at the end of 36K.
        {"name": "attend 4096 on 32K", "op": "attend", "batch": 1, "chunk": 4096, "context": 32768, "prefix": 0, "heads": 8, "group": 4, "dim": 128, "page": 16, "cache": "bf16", "cap": 0.0},
        # One decode step of 48 sequences, weights added to what was summed before: the keys' bytes bound it.
        {"name": "sums decode 48 int8", "op": "sums", "batch": 48, "chunk": 1, "context": 6000, "heads": 8, "group": 4, "dim": 128, "page": 16, "cache": "int8", "cap": 0.0},
        # The last queries of a prompt look back at all of it.
        {"name": "sums window 32 on 40K", "op": "sums", "batch": 1, "chunk": 32, "context": 40000, "heads": 8, "group": 4, "dim": 128, "page": 64, "cache": "bf16", "cap": 0.0},
        # Every query of ragged chunks counts, capped scores, seven query heads to a KV head.
        {"name": "sums 3 x 999 on 9K", "op": "sums", "batch": 3, "chunk": 999, "context": 9001, "heads": 4, "group": 7, "dim": 64, "page": 32, "cache": "bf16", "cap": 30.0},
        # A decoding batch a few tokens above its budget: few tokens move.
        {"name": "evict 64 at 1040", "op": "evict", "batch": 64, "held": 1040, "keep": 1024, "recent": 64, "heads": 8, "dim": 128, "page": 16, "cache": "bf16"},
        # A prompt cut down to its budget.
        {"name": "evict 40K to 5000 int8", "op": "evict", "batch": 1, "held": 40001, "keep": 5000, "recent": 256, "heads": 8, "dim": 128, "page": 64, "cache": "int8"},
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over its logarithm."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["rotate", "attend", "attend", "sums", "evict"])
    case = {"op": op, "heads": rng.choice([1, 2, 4, 8]), "dim": rng.choice([64, 128]), "page": rng.choice([16, 32, 64])}
    if op == "rotate":
        batch = _log(rng, 1, 128)
        rotated = rng.choice([case["dim"], case["dim"], case["dim"] // 2, 24])
        return {**case, "batch": batch, "chunk": _log(rng, 1, max(2, 32768 // batch)), "held": _log(rng, 1, max(2, 200000 // batch)), "group": rng.choice([1, 2, 4, 7]), "cache": rng.choice(["int8", "int8", "model"]),
                "input": rng.choice(["bf16", "bf16", "f32"]), "rotated": rotated, "interleaved": rng.random() < 0.4, "norm": rng.random() < 0.6}
    if op == "evict":
        batch = _log(rng, 1, 64)
        held = _log(rng, 20, max(40, min(60000, 131072 // batch)))
        keep = max(1, int(held * rng.uniform(0.05, 1.05)))
        return {**case, "batch": batch, "held": held, "keep": keep, "recent": int(keep * rng.uniform(0, 0.5)), "cache": rng.choice(["int8", "bf16"])}
    case |= {"batch": _log(rng, 1, 64), "group": rng.choice([1, 2, 4, 7, 8]), "cache": rng.choice(["bf16", "int8"]), "cap": rng.choice([0.0, 0.0, 30.0])}
    chunk = rng.choice([1, _log(rng, 1, 16), _log(rng, 1, max(2, 4096 // case["batch"]))])
    most = 2**31 // (case["batch"] * chunk * case["heads"] * case["group"])  # what the plain form holds of scores
    case |= {"chunk": chunk, "context": _log(rng, 1, max(2, min(40000, most, 524288 // case["batch"])))}
    return case | {"prefix": rng.choice([0, _log(rng, 1, max(2, min(16384, most)))])} if op == "attend" else case


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _spread(n, most):
    """n whole numbers from 0 (where there are several) to `most`, evenly."""
    return [most] if n == 1 else [round(most * i / (n - 1)) for i in range(n)]


def _lengths(case):
    """Each sequence's new tokens, and the tokens it held before them: the case's, whatever the seed."""
    b = case["batch"]
    new = [1] * b if case["chunk"] == 1 else _spread(b, case["chunk"])
    before = _spread(b, case.get("context", case.get("held")))
    return new, [before[(7 * i + b // 2) % b] if b % 7 else before[b - 1 - i] for i in range(b)]


def _quantise(x):
    """int8 codes and the float32 scale of each row of the last dimension; quotients in 64 bits, since many lie next to the border of two codes."""
    scale = (x.abs().amax(-1).double() / 127.0).float().clamp_min(FLT_MIN)
    return torch.round(x.double() / scale.double()[..., None]).clamp(-127, 127).to(torch.int8), scale


def _tables(g, lengths, page, spare=0):
    """Pages for sequences of these lengths in shuffled order, -1 past each sequence's own: [n, most] int32, and the pages' number."""
    need = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(need) + spare, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lengths), max(1, max(need))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at : at + n]
        at += n
    return table, order[at:], sum(need) + spare


def _pages(g, n, case):
    """A cache of n filled pages: keys with a bias of each channel as models have them, and values."""
    h, bs, d = case["heads"], case["page"], case["dim"]
    bias = _randn(g, 1, h, 1, d)
    full = torch.empty((n, h, 2, bs, d), dtype=torch.int8 if case["cache"] == "int8" else torch.bfloat16, device="cuda")
    scales = torch.empty((n, h, 2, bs), device="cuda") if case["cache"] == "int8" else None
    for i in range(0, n, 1024):
        x = _randn(g, min(1024, n - i), h, 2, bs, d)
        x[:, :, 0] += bias
        if scales is None:
            full[i : i + 1024] = x.to(torch.bfloat16)
        else:
            full[i : i + 1024], scales[i : i + 1024] = _quantise(x.to(torch.bfloat16))
    return full, scales


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g, s = _gen(seed), {"case": dict(case)}
    h, d, page, b = case["heads"], case["dim"], case["page"], case["batch"]
    if case["op"] == "evict":
        lens = [case["held"] - x for x in _spread(b, case["held"] // 8)]
        s["table"], _, n = _tables(g, lens, page)
        s["pages"], s["scales"] = _pages(g, n, case)
        s["lens"], cap = _ints(lens), s["table"].shape[1] * page
        # A few tokens have most of the weight, and a tenth none: ties.
        s["sums"] = torch.exp(2.0 * _randn(g, b, h, cap)) * (torch.rand((b, h, cap), generator=g, device="cuda") > 0.1)
        s["positions"] = torch.arange(cap, dtype=torch.int32, device="cuda").expand(b, h, cap).contiguous()
        s["since"] = s["lens"] - case["recent"]
        s["zeros"] = torch.zeros_like(s["lens"])
        return s
    new, before = _lengths(case)
    s["offsets"] = _ints([sum(new[:i]) for i in range(b + 1)])
    s["lens"] = _ints([x + y for x, y in zip(new, before)])
    rows, hq = sum(new), h * case["group"]
    if case["op"] == "rotate":
        dtype = TYPES[case["input"]]
        qkv = _randn(g, rows, hq + 2 * h, d).to(dtype)  # one projection's output
        s["query"], s["keys"], s["values"] = qkv[:, :hq], qkv[:, hq : hq + h], qkv[:, hq + h :]
        s["q_weight"], s["k_weight"] = ((1 + 0.2 * _randn(g, 2, d)).to(dtype).unbind() if case["norm"] else (None, None))
        s["positions"] = _ints([y + t for x, y in zip(new, before) for t in range(x)])
        pairs = torch.arange(case["rotated"] // 2, dtype=torch.float64, device="cuda")
        s["frequencies"] = (500000.0 ** (-2 * pairs / case["rotated"])).float()
        s["table"], _, n = _tables(g, [x + y for x, y in zip(new, before)], page)
        s["pages"] = torch.zeros((n, h, 2, page, d), dtype=torch.int8 if case["cache"] == "int8" else dtype, device="cuda")
        s["scales"] = torch.zeros((n, h, 2, page), device="cuda") if case["cache"] == "int8" else None
        s["starts"] = _ints(before)
        return s
    prefix = case.get("prefix", 0)
    s["table"], s["prefix_table"], n = _tables(g, [x + y for x, y in zip(new, before)], page, -(-prefix // page))
    s["pages"], s["scales"] = _pages(g, n, case)
    s["query"] = (1.5 * _randn(g, rows, hq, d)).to(torch.bfloat16)
    if case["op"] == "sums":  # the attention came before it
        s["lse"] = _plain_attend(s)[1]
        s["sums"] = torch.exp(_randn(g, b, h, s["table"].shape[1] * page))
    return s


def _owners(s):
    """Sequence and place in its chunk of every packed row."""
    row = torch.arange(s["query"].shape[0], device="cuda")
    owner = torch.searchsorted(s["offsets"][1:].long(), row, right=True)
    return owner, row - s["offsets"].long()[owner]


def _plain_rotate(s):
    case = s["case"]
    owner, place = _owners(s)
    angle = s["positions"].double()[:, None] * s["frequencies"].double()
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    n = case["rotated"] // 2
    # Where codes are made of float32 values, those have to be the right ones to the last bit: many lie next to a border.
    wide = torch.float64 if case["input"] == "f32" else torch.float32
    cos, sin = cos.to(wide), sin.to(wide)

    def turn(x, w):
        x = x.to(wide)
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.to(wide)
        a, b = (x[..., 0 : 2 * n : 2], x[..., 1 : 2 * n : 2]) if case["interleaved"] else (x[..., :n], x[..., n : 2 * n])
        a, b = a * cos - b * sin, b * cos + a * sin
        both = torch.stack([a, b], dim=-1).flatten(-2) if case["interleaved"] else torch.cat([a, b], dim=-1)
        return torch.cat([both, x[..., 2 * n :]], dim=-1).float()

    query, keys = turn(s["query"], s["q_weight"]).to(s["query"].dtype), turn(s["keys"], s["k_weight"])
    at = s["lens"].long()[owner] - (s["offsets"][1:] - s["offsets"][:-1]).long()[owner] + place
    ids, at = s["table"].long()[owner, at // case["page"]], at % case["page"]
    x = torch.stack([keys, s["values"].float()], dim=2)  # [rows, h, 2, d]
    if s["scales"] is None:
        s["pages"][ids, :, :, at] = x.to(s["pages"].dtype)
        return query, s["pages"]
    s["pages"][ids, :, :, at], s["scales"][ids, :, :, at] = _quantise(x)
    return query, *_plain_read(s, s["starts"], s["lens"], case["chunk"], s["query"].dtype)


def _plain_read(s, starts, lens, n, dtype):
    """n tokens of each sequence from starts on, zeros past lens: keys and values [b, n, h, d]."""
    page, wide = s["case"]["page"], s["table"].shape[1]
    at = starts.long()[:, None] + torch.arange(n, device="cuda")
    ids = s["table"].long().gather(1, (at // page).clamp(max=wide - 1))
    x = s["pages"][ids.clamp(min=0), :, :, at % page].float() * s["scales"][ids.clamp(min=0), :, :, at % page][..., None]
    x = torch.where(((at < lens[:, None]) & (ids >= 0))[..., None, None, None], x, 0.0).to(dtype)
    return x[:, :, :, 0].contiguous(), x[:, :, :, 1].contiguous()


def _held(s, table):
    """Keys and values of the pages of `table` [..., columns] in 32 bits: [2, h, ..., columns * page, d]."""
    ids = table.long().clamp(min=0)
    x = s["pages"][ids].float()
    if s["scales"] is not None:
        x *= s["scales"][ids][..., None]
    n = ids.dim() - 1  # [..., columns, h, 2, page, d]
    return x.permute(n + 2, n + 1, *range(n), n, n + 3, n + 4).flatten(-3, -2)


def _capped(x, cap):
    return x.div_(cap).tanh_().mul_(cap) if cap else x


def _plain_scores(s):
    """The chunks' queries as padded rows [h, b, T * group, d], the own keys' scores [h, b, T, group, tokens] (minus
    infinity where a query does not see a token), and the own values."""
    case, q = s["case"], s["query"]
    b, t, h, d = case["batch"], case["chunk"], case["heads"], case["dim"]
    first, last = s["offsets"][:-1].long(), s["offsets"][1:].long()
    step = torch.arange(t, device="cuda")
    row = (first[:, None] + step).clamp(max=q.shape[0] - 1)
    rows = q[row].float().reshape(b, t, h, -1, d).permute(2, 0, 1, 3, 4).reshape(h, b, -1, d) * d**-0.5
    k, v = _held(s, s["table"])
    z = _capped(rows @ k.transpose(2, 3), case["cap"]).reshape(h, b, t, case["group"], -1)
    upto = s["lens"].long()[:, None] - (last - first)[:, None] + step  # the last token that query t sees
    seen = (torch.arange(z.shape[-1], device="cuda") <= upto[..., None]) & (step[None, :] < (last - first)[:, None])[..., None]
    return rows, z.masked_fill_(~seen[None, :, :, None], -torch.inf), v


def _plain_attend(s):
    case = s["case"]
    b, t, h, d = case["batch"], case["chunk"], case["heads"], case["dim"]
    rows, z, v = _plain_scores(s)
    z = z.reshape(h, b, -1, z.shape[-1])
    top = z.amax(-1, keepdim=True)
    shared = None
    if case.get("prefix", 0):
        kp, vp = _held(s, s["prefix_table"])[:, :, : case["prefix"]]
        shared = _capped((rows.reshape(h, -1, d) @ kp.transpose(1, 2)).reshape(h, b, -1, case["prefix"]), case["cap"])
        top = torch.maximum(top, shared.amax(-1, keepdim=True))
    top = top.clamp_min(-1e30)  # padded rows see nothing
    z = z.sub_(top).exp_()
    total, out = z.sum(-1), z @ v
    if shared is not None:
        shared = shared.sub_(top).exp_()
        total = total + shared.sum(-1)
        out = out + (shared.reshape(h, -1, case["prefix"]) @ vp).reshape(out.shape)
    out, lse = out / total[..., None], top[..., 0] + total.log()
    owner, place = _owners(s)
    out = out.reshape(h, b, t, case["group"], d)[:, owner, place].permute(1, 0, 2, 3).reshape(s["query"].shape)
    return out.to(torch.bfloat16), lse.reshape(h, b, t, case["group"])[:, owner, place].permute(1, 0, 2).reshape(out.shape[:2])


def _plain_sums(s):
    case = s["case"]
    b, t, h = case["batch"], case["chunk"], case["heads"]
    z = _plain_scores(s)[1]
    first = s["offsets"][:-1].long()
    row = (first[:, None] + torch.arange(t, device="cuda")).clamp(max=s["lse"].shape[0] - 1)
    lse = s["lse"][row].reshape(b, t, h, -1).permute(2, 0, 1, 3)  # [h, b, t, group]
    got = z.sub_(lse[..., None]).exp_().sum((2, 3)).transpose(0, 1)
    at, lens = torch.arange(got.shape[-1], device="cuda"), s["lens"][:, None]
    old = at < lens - (s["offsets"][1:] - s["offsets"][:-1])[:, None]  # new tokens' sums begin here
    return torch.where(old[:, None], s["sums"], 0.0) + got


def _plain_evict(s):
    case, lens = s["case"], s["lens"][:, None, None]
    keep, page = case["keep"], case["page"]
    slot = torch.arange(s["sums"].shape[-1], device="cuda")
    there, safe = slot < lens, s["positions"] >= s["since"][:, None, None]
    safe |= s["positions"] < 4
    rank = torch.where(there, torch.where(safe, torch.inf, s["sums"]), -torch.inf).argsort(dim=-1, descending=True, stable=True).argsort(dim=-1)
    kept = there & (rank < keep)
    b, j, to = (~kept & (slot < keep) & there).nonzero(as_tuple=True)  # holes, and as many kept tokens behind them
    _, _, of = (kept & (slot >= keep)).nonzero(as_tuple=True)
    src = s["table"].long()[b, of // page], j, slice(None), of % page
    dst = s["table"].long()[b, to // page], j, slice(None), to % page
    s["pages"][dst] = s["pages"][src]
    if s["scales"] is not None:
        s["scales"][dst] = s["scales"][src]
    sums, positions, left = s["sums"].clone(), s["positions"].clone(), s["lens"].clamp(max=keep)
    sums[b, j, to], positions[b, j, to] = s["sums"][b, j, of], s["positions"][b, j, of]
    gone = slot >= left[:, None, None]
    sums, positions = sums.masked_fill_(gone, 0.0), positions.masked_fill_(gone, -1)
    if s["scales"] is None:
        return left, sums, positions, s["pages"]
    return left, sums, positions, *_plain_read(s, s["zeros"], left, keep, torch.bfloat16)


def run(s):
    case = s["case"]
    if case["op"] == "rotate":
        if not own:
            return _plain_rotate(s)
        from lazykv_b200 import kernels

        query = kernels.paged_write_rotated(s["query"], s["keys"], s["values"], s["positions"], s["frequencies"], s["pages"], s["table"], s["lens"], s["offsets"],
                                            scales=s["scales"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=1e-6, interleaved=case["interleaved"])
        if s["scales"] is None:
            return query, s["pages"]
        return query, *kernels.paged_read(s["pages"], s["table"], s["starts"], case["chunk"], lens=s["lens"], scales=s["scales"], dtype=s["query"].dtype)
    if case["op"] == "attend":
        if not own:
            return _plain_attend(s)
        from lazykv_b200 import kernels

        return kernels.chunk_attention(s["query"], s["pages"], s["table"], s["lens"], s["offsets"], case["dim"] ** -0.5, scales=s["scales"],
                                       prefix_table=s["prefix_table"], prefix_len=case["prefix"], cap=case["cap"])
    if case["op"] == "sums":
        if not own:
            return _plain_sums(s)
        from lazykv_b200 import kernels

        return kernels.attention_sums(s["query"], s["lse"], s["pages"], s["table"], s["lens"], s["offsets"], case["dim"] ** -0.5, sums=s["sums"], scales=s["scales"],
                                      cap=case["cap"])
    if not own:
        return _plain_evict(s)
    from lazykv_b200 import kernels

    left, sums, positions = kernels.paged_evict(s["pages"], s["table"], s["lens"], s["sums"], s["positions"], case["keep"], since=s["since"], sinks=4, scales=s["scales"])
    if s["scales"] is None:
        return left, sums, positions, s["pages"]
    return left, sums, positions, *kernels.paged_read(s["pages"], s["table"], s["zeros"], case["keep"], lens=left, scales=s["scales"])


def _seen(case):
    """Pairs of a query token and an own token that it sees."""
    new, before = _lengths(case)
    return sum(n * m + n * (n + 1) // 2 for n, m in zip(new, before))


def work(case):
    h, d, b = case["heads"], case["dim"], case["batch"]
    size = 1 if case["cache"] == "int8" else 4 if case.get("input") == "f32" else 2
    held = h * (d * size + (4 if case["cache"] == "int8" else 0))  # a token's keys, or its values, in the cache
    if case["op"] == "evict":
        lens = [case["held"] - x for x in _spread(b, case["held"] // 8)]
        cap = -(-max(lens) // case["page"]) * case["page"]
        # Sums and positions read and written, and a kept token in the tail for every hole before it, here of even weights.
        moved = sum(case["keep"] * (n - case["keep"]) // n for n in lens if n > case["keep"])
        read = 2 * min(case["keep"], max(lens)) * b * h * d * 2 + 2 * held * sum(min(n, case["keep"]) for n in lens) if case["cache"] == "int8" else 0
        return {"bytes": 8 * h * sum(lens) + 8 * h * b * cap + 4 * held * moved + read, "flops": 8 * h * sum(lens)}
    new, before = _lengths(case)
    rows, hq, keys = sum(new), h * case["group"], sum(new) + sum(before)
    if case["op"] == "rotate":
        e = 4 if case["input"] == "f32" else 2
        read = 2 * held * rows + 2 * b * case["chunk"] * h * d * e if case["cache"] == "int8" else 0
        return {"bytes": rows * ((2 * hq + 2 * h) * d * e + 2 * held + 4) + read, "flops": rows * (10 * (hq + h) * d + 6 * h * d)}
    if case["op"] == "attend":
        pairs = _seen(case) + rows * case["prefix"]
        return {"bytes": 2 * held * (keys + case["prefix"]) + rows * hq * (4 * d + 4), "flops": 4 * d * hq * pairs}
    return {"bytes": held * keys + rows * hq * (2 * d + 4) + 4 * h * (sum(before) + b * -(-max(x + y for x, y in zip(new, before)) // case["page"]) * case["page"]),
            "flops": 2 * d * hq * _seen(case)}


# -- the definitions in 64 bits, a sequence and a head at a time --


def _codes_of(x):
    """What int8 pages hold of float32 rows: whole multiples of the row's scale."""
    scale = (x.abs().amax(-1, keepdim=True).double() / 127).float().double().clamp_min(FLT_MIN)
    return (x.double() / scale).round() * scale


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "attend": _exact_attend, "sums": _exact_sums, "evict": _exact_evict}[case["op"]](s)


def _exact_rotate(s):
    case, n = s["case"], s["case"]["rotated"] // 2
    turns = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double()[:, None, None] * s["frequencies"].double())

    def of(x, w):
        x = x.double()
        if w is not None:
            x = w.double() * x / ((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt()
        first = slice(0, 2 * n, 2) if case["interleaved"] else slice(0, n)
        second = slice(1, 2 * n, 2) if case["interleaved"] else slice(n, 2 * n)
        y, z = x.clone(), torch.complex(x[..., first], x[..., second]) * turns
        y[..., first], y[..., second] = z.real, z.imag
        return y

    query, keys, values = of(s["query"], s["q_weight"]), of(s["keys"], s["k_weight"]), s["values"].double()
    new, before = _lengths(case)
    if case["cache"] == "int8":
        kv = torch.stack([_codes_of(keys.float()), _codes_of(s["values"].float())])
        out = torch.zeros((2, case["batch"], case["chunk"], case["heads"], case["dim"]), dtype=torch.float64, device="cuda")
        at = 0
        for i, m in enumerate(new):
            out[:, i, :m] = kv[:, at : at + m]
            at += m
        return query, out[0], out[1]
    pages, at = s["pages"].double(), 0
    for i, (m, held) in enumerate(zip(new, before)):
        pos = held + torch.arange(m, device="cuda")
        ids = s["table"][i].long()[pos // case["page"]]
        for kv, x in enumerate((keys, values)):
            pages[ids, :, kv, pos % case["page"]] = x[at : at + m]
        at += m
    return query, pages


def _exact_tokens(s, ids, n, j):
    """Keys and values of head j of the first n tokens in these pages, [n, d] each."""
    x = s["pages"][ids.long(), j].double()
    if s["scales"] is not None:
        x = x * s["scales"][ids.long(), j].double()[..., None]
    x = x.transpose(0, 1).reshape(2, -1, x.shape[-1])[:, :n]
    return x[0], x[1]


def _exact_rows(s, prefix):
    """(sequence, KV head, query rows, their scores in 64 bits [tokens * group, keys], values) piece by piece; own tokens first."""
    case, at = s["case"], 0
    new, before = _lengths(case)
    grp, page = case["group"], case["page"]
    for i, (m, held) in enumerate(zip(new, before)):
        for j in range(case["heads"] if m else 0):
            k, v = _exact_tokens(s, s["table"][i, : -(-(m + held) // page)], m + held, j)
            if prefix:
                more = _exact_tokens(s, s["prefix_table"], prefix, j)
                k, v = torch.cat([k, more[0]]), torch.cat([v, more[1]])
            for t in range(0, m, 512):
                some = slice(at + t, at + min(m, t + 512))
                q = s["query"][some, j * grp : (j + 1) * grp].double()
                z = torch.einsum("tgd,nd->tgn", q, k) / case["dim"] ** 0.5
                if case["cap"]:
                    z = case["cap"] * torch.tanh(z / case["cap"])
                limit = held + t + torch.arange(z.shape[0], device="cuda")
                z[:, :, : m + held].masked_fill_((torch.arange(m + held, device="cuda") > limit[:, None])[:, None], -torch.inf)
                yield i, j, some, z, v
        at += m


def _exact_attend(s):
    grp = s["case"]["group"]
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["query"].shape[:2], dtype=torch.float64, device="cuda")
    for _, j, some, z, v in _exact_rows(s, s["case"]["prefix"]):
        lse[some, j * grp : (j + 1) * grp] = torch.logsumexp(z, -1)
        out[some, j * grp : (j + 1) * grp] = torch.softmax(z, -1) @ v
    return out, lse


def _exact_sums(s):
    new, before = _lengths(s["case"])
    grp = s["case"]["group"]
    out = s["sums"].double()
    for i, m in enumerate(before):
        out[i, :, m:] = 0
    for i, j, some, z, _ in _exact_rows(s, 0):
        out[i, j, : z.shape[-1]] += torch.exp(z - s["lse"][some, j * grp : (j + 1) * grp].double()[..., None]).sum((0, 1))
    return out


def _exact_evict(s):
    case = s["case"]
    keep, page, n = case["keep"], case["page"], s["sums"].shape[-1]
    sums, lens = s["sums"].double().cpu(), s["lens"].tolist()
    out_sums, out_pos = torch.zeros_like(sums), torch.full(sums.shape, -1, dtype=torch.int32)
    pages = s["pages"].double()
    if s["scales"] is not None:
        pages = pages * s["scales"].double()[..., None]
    moved = pages.clone()
    for i, m in enumerate(lens):
        for j in range(case["heads"]):
            w = sums[i, j, :m].clone()
            w[max(0, m - case["recent"]) :] = torch.inf
            w[:4] = torch.inf
            kept = torch.sort(torch.sort(w, descending=True, stable=True).indices[:keep]).values
            slots, late = torch.arange(n)[: min(m, keep)].clone(), kept[kept >= keep]
            holes = slots[~torch.isin(slots, kept)]
            slots[holes] = late
            out_sums[i, j, : len(slots)], out_pos[i, j, : len(slots)] = sums[i, j, slots], slots.int()
            to, of = holes.cuda(), late.cuda()
            ids = s["table"][i].long()
            moved[ids[to // page], j, :, to % page] = pages[ids[of // page], j, :, of % page]
    left = torch.tensor([min(m, keep) for m in lens], dtype=torch.int32)
    if s["scales"] is None:
        return left, out_sums, out_pos, moved
    out = torch.zeros((2, case["batch"], keep, case["heads"], case["dim"]), dtype=torch.float64, device="cuda")
    for i, m in enumerate(left.tolist()):
        x = torch.cat(list(moved[s["table"][i, : -(-m // page)].long()]), dim=2)[:, :, :m]  # [h, 2, m, d]
        out[:, i, :m] = x.permute(1, 2, 0, 3)
    return left, out_sums, out_pos, out[0], out[1]
