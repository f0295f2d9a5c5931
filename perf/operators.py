"""The operators of a decode step for a batch of sequences that share a prompt, as they are measured.

A batch forked from one long prompt keeps the prompt's KV once, in pages of a paged cache, and every
sequence's own tokens in further pages. A step writes the new tokens' KV into the pages (quantised to
int8 with a scale per token and head, or in the model's type), attends every sequence's queries to the
shared prompt and to its own tokens, and, where tokens were drafted, verifies them against the model's
probabilities. Four kinds of case:

  write   paged_write of new tokens, and paged_read of them back (the values that the codes stand for)
  read    paged_read of whole sequences
  attend  prefix_attention over the shared pages and the sequences' own
  verify  verify_drafts

`own` selects the framework's kernels; otherwise `run` computes the plain form in elementary torch
operations.
"""

import torch

own = False

FLT_MIN = 1.1754943508222875e-38  # the least normal float32: the floor of a quantisation scale
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # One decode step's KV of a batch of 64, 8 KV heads: the smallest write, launch latency counts.
        {"name": "write decode 64 int8", "op": "write", "batch": 64, "tokens": 1, "heads": 8, "dim": 128, "page": 16, "held": 4000, "cache": "int8", "input": "bf16", "fused": False},
        # Five drafted tokens for 48 sequences, keys and values as slices of one packed projection, float32 model, small heads.
        {"name": "write drafts packed f32", "op": "write", "batch": 48, "tokens": 5, "heads": 4, "dim": 64, "page": 16, "held": 1003, "cache": "int8", "input": "f32", "fused": True},
        # A prefilled prompt of 64K tokens quantised into the cache.
        {"name": "write prompt 64K int8", "op": "write", "batch": 1, "tokens": 65536, "heads": 8, "dim": 128, "page": 64, "held": 0, "cache": "int8", "input": "bf16", "fused": False},
        # A few sequences of odd length handed on in the model's type (a fork, a move to another tier).
        {"name": "read 3 x 1001 bf16", "op": "read", "batch": 3, "tokens": 1001, "heads": 8, "dim": 64, "page": 16, "cache": "bf16", "output": "bf16"},
        # Ragged sequences of up to 16K tokens dequantised.
        {"name": "read 12 x 16K int8", "op": "read", "batch": 12, "tokens": 16000, "heads": 8, "dim": 128, "page": 32, "cache": "int8", "output": "bf16"},
        # Two sequences on a short prompt: every launch counts.
        {"name": "attend 2 on 1000", "op": "attend", "batch": 2, "tokens": 1, "heads": 8, "group": 4, "dim": 64, "page": 16, "prefix": 1000, "suffix": 90, "cache": "bf16"},
        # An ordinary chat batch: 32 sequences on a prompt of 16K, int8 pages.
        {"name": "attend 32 on 16K int8", "op": "attend", "batch": 32, "tokens": 1, "heads": 8, "group": 4, "dim": 128, "page": 16, "prefix": 16384, "suffix": 777, "cache": "int8"},
        # Five positions a sequence (four drafted tokens), odd lengths, the model's type, small heads.
        {"name": "attend 24x5 on 8191", "op": "attend", "batch": 24, "tokens": 5, "heads": 8, "group": 4, "dim": 64, "page": 16, "prefix": 8191, "suffix": 1203, "cache": "bf16"},
        # One KV head per query head, a long prompt and few sequences: the pages' bytes bound it.
        {"name": "attend 6 mha on 32K", "op": "attend", "batch": 6, "tokens": 1, "heads": 16, "group": 1, "dim": 128, "page": 64, "prefix": 32768, "suffix": 300, "cache": "bf16"},
        # The largest: 128 sequences on a prompt of 128K, int8 pages.
        {"name": "attend 128 on 128K int8", "op": "attend", "batch": 128, "tokens": 1, "heads": 8, "group": 4, "dim": 128, "page": 64, "prefix": 131072, "suffix": 2000, "cache": "int8"},
        # One sequence with four drafted tokens.
        {"name": "verify 1x4", "op": "verify", "batch": 1, "drafted": 4, "vocab": 32000, "greedy": False},
        # A batch with seven drafted tokens each over a large vocabulary.
        {"name": "verify 64x7", "op": "verify", "batch": 64, "drafted": 7, "vocab": 128256, "greedy": False},
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over its logarithm."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "verify"])
    dim, page, heads = rng.choice([64, 128]), rng.choice([16, 32, 64]), rng.choice([1, 2, 4, 8])
    if op == "write":
        batch = _log(rng, 1, 128)
        return {"op": op, "batch": batch, "tokens": _log(rng, 1, max(2, 32768 // batch)), "heads": heads, "dim": dim, "page": page, "held": rng.randrange(0, 2000),
                "cache": rng.choice(["int8", "int8", "model"]), "input": rng.choice(["bf16", "bf16", "f32"]), "fused": rng.random() < 0.5}
    if op == "read":
        batch, cache = _log(rng, 1, 32), rng.choice(["int8", "bf16"])
        return {"op": op, "batch": batch, "tokens": _log(rng, 1, max(2, 131072 // batch)), "heads": heads, "dim": dim, "page": page, "cache": cache,
                "output": rng.choice(["bf16", "f32"]) if cache == "int8" else "bf16"}
    if op == "attend":
        batch, tokens, group = _log(rng, 1, 128), rng.choice([1, 1, 1, 2, 4, 7]), rng.choice([1, 2, 4, 7, 8])
        rows = batch * tokens * group
        return {"op": op, "batch": batch, "tokens": tokens, "heads": heads, "group": group, "dim": dim, "page": page, "prefix": _log(rng, 1, min(131072, max(64, 2**26 // rows))),
                "suffix": _log(rng, tokens, 2000), "cache": rng.choice(["bf16", "int8"])}
    return {"op": op, "batch": _log(rng, 1, 96), "drafted": rng.randrange(1, 9), "vocab": _log(rng, 500, 160000), "greedy": rng.random() < 0.3}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _spread(n, most):
    """n whole numbers from 0 (where there are several) to `most`, evenly: the sequences' lengths, whatever the seed."""
    return [most] if n == 1 else [round(most * i / (n - 1)) for i in range(n)]


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


def _pages(g, n, case, dtype):
    """A cache of n filled pages: keys with a bias of each channel as models have them, and values."""
    h, bs, d = case["heads"], case["page"], case["dim"]
    bias = _randn(g, 1, h, 1, d)
    full = torch.empty((n, h, 2, bs, d), dtype=torch.int8 if case["cache"] == "int8" else dtype, device="cuda")
    scales = torch.empty((n, h, 2, bs), device="cuda") if case["cache"] == "int8" else None
    for i in range(0, n, 1024):
        x = _randn(g, min(1024, n - i), h, 2, bs, d)
        x[:, :, 0] += bias
        if scales is None:
            full[i : i + 1024] = x.to(dtype)
        else:
            full[i : i + 1024], scales[i : i + 1024] = _quantise(x.to(torch.bfloat16))
    return full, scales


def prepare(case, seed):
    g, s = _gen(seed), {"case": dict(case)}
    if case["op"] == "verify":
        b, k, v = case["batch"], case["drafted"], case["vocab"]
        logits = _randn(g, b, k + 1, v) * 2.5
        s["target"] = torch.softmax(logits, -1)
        draft = torch.softmax(logits[:, :k] + 0.5 * _randn(g, b, k, v), -1)
        s["tokens"] = torch.multinomial(draft.reshape(b * k, v), 1, generator=g).reshape(b, k)
        s["draft"] = None if case["greedy"] else draft
        s["uniforms"] = torch.rand((b, k + 1), generator=g, device="cuda")
        return s
    h, d, page, b = case["heads"], case["dim"], case["page"], case["batch"]
    if case["op"] == "write":
        t, dtype = case["tokens"], TYPES[case["input"]]
        if case["fused"]:  # slices of one projection's output, query heads first
            qkv = _randn(g, b, t, 4 * h, d).to(dtype)
            s["keys"], s["values"] = qkv[:, :, 2 * h : 3 * h], qkv[:, :, 3 * h :]
        else:
            s["keys"], s["values"] = _randn(g, b, t, h, d).to(dtype), _randn(g, b, t, h, d).to(dtype)
        held = _spread(b, case["held"])
        s["table"], _, n = _tables(g, [x + t for x in held], page)
        s["starts"] = torch.tensor(held, dtype=torch.int32, device="cuda")
        s["pages"] = torch.zeros((n, h, 2, page, d), dtype=torch.int8 if case["cache"] == "int8" else dtype, device="cuda")
        s["scales"] = torch.zeros((n, h, 2, page), device="cuda") if case["cache"] == "int8" else None
        return s
    if case["op"] == "read":
        lens = _spread(b, case["tokens"])
        s["table"], _, n = _tables(g, lens, page)
        s["pages"], s["scales"] = _pages(g, n, case, torch.bfloat16)
        s["starts"] = torch.zeros(b, dtype=torch.int32, device="cuda")
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        return s
    lens = _spread(b, case["suffix"])
    prefix_pages = -(-case["prefix"] // page)
    s["table"], s["prefix_table"], n = _tables(g, lens, page, prefix_pages)
    order = torch.randperm(b, generator=g, device="cuda")
    s["table"] = s["table"][order].contiguous()
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")[order].contiguous()
    s["pages"], s["scales"] = _pages(g, n, case, torch.bfloat16)
    s["query"] = (1.5 * _randn(g, b, case["tokens"], h * case["group"], d)).to(torch.bfloat16)
    return s


def _values(codes, scales):
    return codes.float() if scales is None else codes.float() * scales[..., None]


def _rows(s, first, n):
    """Page and place in it of tokens first_b .. first_b + n - 1 of each sequence: [b, n] each, the page -1 where the table has none."""
    page, wide = s["pages"].shape[3], s["table"].shape[1]
    at = first.long()[:, None] + torch.arange(n, device="cuda")
    where = at // page
    ids = s["table"].long().gather(1, where.clamp(max=wide - 1))
    return torch.where(where < wide, ids, -1), at % page, at


def _plain_write(s):
    ids, place, _ = _rows(s, s["starts"], s["keys"].shape[1])
    x = torch.stack([s["keys"], s["values"]], dim=3)  # [b, t, h, 2, d]
    if s["scales"] is None:
        s["pages"][ids, :, :, place] = x
        return
    codes, scales = _quantise(x)
    s["pages"][ids, :, :, place] = codes
    s["scales"][ids, :, :, place] = scales


def _plain_read(s, first, n, lens, dtype):
    ids, place, at = _rows(s, first, n)
    take = ids.clamp(min=0)
    x = s["pages"][take, :, :, place].float()  # [b, n, h, 2, d]
    if s["scales"] is not None:
        x = x * s["scales"][take, :, :, place][..., None]
    there = ids >= 0
    if lens is not None:
        there = there & (at < lens[:, None])
    x = torch.where(there[:, :, None, None, None], x, 0.0).to(dtype)
    return x[:, :, :, 0].contiguous(), x[:, :, :, 1].contiguous()


def _plain_attend(s):
    case, q = s["case"], s["query"]
    b, t, hq, d = q.shape
    h, scale = case["heads"], case["dim"] ** -0.5
    grp = hq // h
    pick = s["prefix_table"].long()
    shared = _values(s["pages"][pick], None if s["scales"] is None else s["scales"][pick])  # [n, h, 2, page, d]
    shared = shared.permute(2, 1, 0, 3, 4).reshape(2, h, -1, d)[:, :, : case["prefix"]]
    pick = s["table"].long().clamp(min=0)
    mine = _values(s["pages"][pick], None if s["scales"] is None else s["scales"][pick])  # [b, n, h, 2, page, d]
    mine = mine.permute(3, 2, 0, 1, 4, 5).reshape(2, h, b, -1, d)
    rows = q.float().reshape(b, t, h, grp, d).permute(2, 0, 1, 3, 4).reshape(h, b, t * grp, d) * scale
    s1 = rows.reshape(h, b * t * grp, d) @ shared[0].transpose(1, 2)
    s2 = (rows @ mine[0].transpose(2, 3)).reshape(h, b, t, grp, -1)
    last = s["lens"].long()[:, None] - t + torch.arange(t, device="cuda")  # the last own token that query t sees
    seen = torch.arange(s2.shape[-1], device="cuda") <= last[..., None]
    s2 = torch.where(seen[None, :, :, None], s2, -torch.inf).reshape(h, b * t * grp, -1)
    top = torch.maximum(s1.amax(-1), s2.amax(-1))[..., None]
    s1, s2 = (s1 - top).exp_(), (s2 - top).exp_()
    total = s1.sum(-1) + s2.sum(-1)
    out = s1 @ shared[1] + (s2.reshape(h, b, t * grp, -1) @ mine[1]).reshape(h, -1, d)
    out, lse = out / total[..., None], top[..., 0] + total.log()
    out = out.reshape(h, b, t, grp, d).permute(1, 2, 0, 3, 4).reshape(b, t, hq, d)
    return out.to(torch.bfloat16), lse.reshape(h, b, t, grp).permute(1, 2, 0, 3).reshape(b, t, hq)


def _plain_verify(s):
    p, q, tokens, u = s["target"], s["draft"], s["tokens"], s["uniforms"].double()
    b, k = tokens.shape
    px = p[:, :k].gather(2, tokens[..., None])[..., 0].double()
    qx = torch.ones_like(px) if q is None else q.gather(2, tokens[..., None])[..., 0].double()
    kept = (u[:, :k] * qx < px).long().cumprod(1).sum(1)
    row = torch.arange(b, device="cuda")
    at = kept.clamp(max=k - 1)
    w = p[row, kept].double()
    if q is None:
        less = torch.zeros_like(w).scatter_(1, tokens[row, at][:, None], torch.inf)
    else:
        less = q[row, at].double()
    rest = torch.where((kept < k)[:, None], (w - less).clamp_min(0.0), w)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, w)
    run_up = rest.cumsum(1)
    token = (run_up <= u[:, k:] * run_up[:, -1:]).sum(1)
    return kept.to(torch.int32), token


def run(s):
    case = s["case"]
    if case["op"] == "verify":
        if own:
            from lazykv_b200 import kernels

            return kernels.verify_drafts(s["target"], s["draft"], s["tokens"], s["uniforms"])
        return _plain_verify(s)
    if case["op"] == "write":
        t, dtype = case["tokens"], TYPES[case["input"]]
        if own:
            from lazykv_b200 import kernels

            kernels.paged_write(s["keys"], s["values"], s["pages"], s["table"], s["starts"], scales=s["scales"])
            return kernels.paged_read(s["pages"], s["table"], s["starts"], t, scales=s["scales"], dtype=dtype)
        _plain_write(s)
        return _plain_read(s, s["starts"], t, None, dtype)
    if case["op"] == "read":
        if own:
            from lazykv_b200 import kernels

            return kernels.paged_read(s["pages"], s["table"], s["starts"], case["tokens"], lens=s["lens"], scales=s["scales"], dtype=TYPES[case["output"]])
        return _plain_read(s, s["starts"], case["tokens"], s["lens"], TYPES[case["output"]])
    if own:
        from lazykv_b200 import kernels

        return kernels.prefix_attention(s["query"], s["pages"], s["table"], s["lens"], s["prefix_table"], case["prefix"], case["dim"] ** -0.5, scales=s["scales"])
    return _plain_attend(s)


def work(case):
    if case["op"] == "verify":
        b, k, v = case["batch"], case["drafted"], case["vocab"]
        # the probabilities of the drafted tokens, and one row (or pair of rows) of each sequence
        return {"bytes": b * (v * 4 * (1 if case["greedy"] else 2) + 20 * k + 16), "flops": 3 * b * v}
    h, d = case["heads"], case["dim"]
    if case["op"] == "attend":
        b, t, hq = case["batch"], case["tokens"], h * case["group"]
        keys = case["prefix"] + sum(_spread(b, case["suffix"]))
        held = h * 2 * (d + 4 if case["cache"] == "int8" else 2 * d)
        return {"bytes": keys * held + b * t * hq * (4 * d + 4), "flops": 4 * d * hq * t * (b * case["prefix"] + sum(_spread(b, case["suffix"])))}
    size = 4 if case.get("input", case.get("output")) == "f32" else 2
    held = 2 * h * (d + 4 if case["cache"] == "int8" else d * size)
    if case["op"] == "write":  # the tokens in, what the pages hold of them, their values out
        n = case["batch"] * case["tokens"]
        return {"bytes": n * (held + 2 * h * d * size * 2), "flops": 6 * n * h * d}
    n, out = sum(_spread(case["batch"], case["tokens"])), case["batch"] * case["tokens"]
    return {"bytes": n * held + out * 2 * h * d * size, "flops": 2 * n * h * d}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "verify":
        return _exact_verify(s)
    if case["op"] == "attend":
        return _exact_attend(s)
    # Values as the cache holds them: whole multiples of the row's scale, which it holds in 32 bits.
    page, table = case["page"], s["table"].tolist()
    b, n = case["batch"], case["tokens"]
    first = s["starts"].tolist()
    if case["op"] == "write":
        def of(x):
            x = x.double()
            if s["scales"] is None:
                return x
            scale = (x.abs().amax(-1, keepdim=True) / 127).float().double().clamp_min(FLT_MIN)
            return (x / scale).round() * scale

        return of(s["keys"]), of(s["values"])
    out = torch.zeros((2, b, n, case["heads"], case["dim"]), dtype=torch.float64, device="cuda")
    for i in range(b):
        ids = [x for x in table[i] if x >= 0]
        if ids:
            x = s["pages"][ids].double()
            if s["scales"] is not None:
                x = x * s["scales"][ids].double().unsqueeze(-1)
            x = torch.cat(list(x), dim=2)  # [h, 2, tokens, d]
            m = min(int(s["lens"][i]), x.shape[2])
            out[:, i, :m] = x[:, :, first[i] : first[i] + m].permute(1, 2, 0, 3)
    return out[0], out[1]


def _exact_attend(s):
    case, q = s["case"], s["query"].double()
    b, t, hq, d = q.shape
    h, page = case["heads"], case["page"]
    grp = hq // h
    out = torch.zeros((b, t, hq, d), dtype=torch.float64, device="cuda")
    lse = torch.zeros((b, t, hq), dtype=torch.float64, device="cuda")

    def tokens(ids, n, j):  # keys and values of head j in 64 bits, [n, d] each
        x = s["pages"][ids, j].double()
        if s["scales"] is not None:
            x = x * s["scales"][ids, j].double()[..., None]
        x = x.transpose(0, 1).reshape(2, -1, d)[:, :n]
        return x[0], x[1]

    lens, table = s["lens"].tolist(), s["table"].long()
    for j in range(h):
        kp, vp = tokens(s["prefix_table"].long(), case["prefix"], j)
        for at in range(0, b, 16):  # sequences a few at a time: their scores over the prompt fit the card
            some = range(at, min(b, at + 16))
            shared = torch.einsum("btgd,nd->btgn", q[at : at + 16, :, j * grp : (j + 1) * grp], kp) / d**0.5
            for i in some:
                n = lens[i]
                ki, vi = tokens(table[i, : -(-n // page)], n, j)
                for step in range(t):
                    m = max(0, n - t + step + 1)
                    rows = slice(j * grp, (j + 1) * grp)
                    z = torch.cat([shared[i - at, step], q[i, step, rows] @ ki[:m].T / d**0.5], dim=-1)
                    lse[i, step, rows] = torch.logsumexp(z, -1)
                    w = torch.softmax(z, -1)
                    out[i, step, rows] = w[:, : case["prefix"]] @ vp + w[:, case["prefix"] :] @ vi[:m]
    return out, lse


def _exact_verify(s):
    tokens, u = s["tokens"].tolist(), s["uniforms"].double().tolist()
    k, kept, chosen = len(tokens[0]), [], []
    for i, drafted in enumerate(tokens):
        n = 0
        while n < k:
            p = float(s["target"][i, n, drafted[n]])
            q = 1.0 if s["draft"] is None else float(s["draft"][i, n, drafted[n]])
            if not u[i][n] * q < p:
                break
            n += 1
        w = s["target"][i, n].double()
        if n < k:
            left = w.clone()
            if s["draft"] is None:
                left[drafted[n]] = 0
            else:
                left = torch.relu(left - s["draft"][i, n].double())
            w = left if float(left.sum()) > 0 else w
        edges = torch.cumsum(w, 0)
        kept.append(n)
        chosen.append(int(torch.searchsorted(edges, u[i][k] * edges[-1], right=True)))
    return torch.tensor(kept, dtype=torch.int32), torch.tensor(chosen)
