"""Operators of a decoding step that are timed: appending to a paged key-value cache, attention of one new token over it, and
low-rank adapters beside a shared projection.

Sizes are those of this repository's own workloads (BERT-base heads 12 x 64, the 8192 x 28672 feed-forward products with 64
heads of 128 over 8192 features, 768-wide projections) and generic ones around them: one token to long prompts and caches,
odd sizes, pages that do not divide a tile, both layouts of a page, every type of input and cache.
"""
import ctypes as C
import math

import torch

own = False


def listed():
    return [
        # one new token of one sequence: latency
        {"name": "append_1", "kind": "append", "sequences": 1, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "cache": "f16",
         "page": 16, "order": "hnd", "in": "f32", "style": "half", "rotary": 128, "filled": 1000, "pad": 0},
        # one new token each of 64 sequences, binary16 in, interleaved pairs, the rest of a head not rotated
        {"name": "append_64", "kind": "append", "sequences": 64, "tokens": 1, "heads": 64, "kv_heads": 8, "dim": 128, "cache": "f16",
         "page": 32, "order": "nhd", "in": "f16", "style": "interleaved", "rotary": 64, "filled": 333, "pad": 0},
        # prompts of five requests at once behind each other, padded to a common length, into a cache of signed bytes
        {"name": "append_prompts_i8", "kind": "append", "sequences": 5, "tokens": 801, "heads": 64, "kv_heads": 8, "dim": 128, "cache": "i8",
         "page": 16, "order": "hnd", "in": "f32", "style": "half", "rotary": 128, "filled": 0, "pad": 37},
        # one sequence, a moderate context: latency, and the join of its parts
        {"name": "attention_1x4000", "kind": "attention", "sequences": 1, "longest": 4000, "shortest": 4000, "heads": 32, "kv_heads": 8, "dim": 128,
         "cache": "f16", "page": 16, "order": "hnd", "q": "f32", "out": "f32", "window": 0, "empty": 0},
        # BERT-base heads (one query head per key head), short and uneven contexts, pages of 24 tokens, two idle rows of the batch
        {"name": "attention_32x12x64", "kind": "attention", "sequences": 32, "longest": 512, "shortest": 1, "heads": 12, "kv_heads": 12, "dim": 64,
         "cache": "f16", "page": 24, "order": "nhd", "q": "f16", "out": "f16", "window": 0, "empty": 2},
        # a serving batch: 64 sequences of uneven length up to 8192, cache of signed bytes
        {"name": "attention_64x8192_i8", "kind": "attention", "sequences": 64, "longest": 8192, "shortest": 700, "heads": 64, "kv_heads": 8, "dim": 128,
         "cache": "i8", "page": 64, "order": "hnd", "q": "f32", "out": "f32", "window": 0, "empty": 0},
        # one long document: the cache's length is all there is to split
        {"name": "attention_1x131072", "kind": "attention", "sequences": 1, "longest": 131072, "shortest": 131072, "heads": 64, "kv_heads": 8, "dim": 128,
         "cache": "f16", "page": 16, "order": "nhd", "q": "f32", "out": "f32", "window": 0, "empty": 0},
        # one row through a 768-wide projection with an adapter: latency
        {"name": "lora_1x768x768", "kind": "lora", "rows": 1, "segments": 1, "adapters": 1, "k": 768, "n": 768, "rank": 8, "x": "f32", "idle": 0},
        # sizes that are no multiple of anything
        {"name": "lora_ragged", "kind": "lora", "rows": 333, "segments": 5, "adapters": 4, "k": 515, "n": 1001, "rank": 24, "x": "f32", "idle": 17},
        # 16 sequences decoded at once, each with an adapter of its own
        {"name": "lora_16x8192x28672", "kind": "lora", "rows": 16, "segments": 16, "adapters": 16, "k": 8192, "n": 28672, "rank": 16, "x": "u8", "idle": 0},
        # prompts of six requests through the same projection
        {"name": "lora_2048x8192x28672", "kind": "lora", "rows": 2048, "segments": 6, "adapters": 6, "k": 8192, "n": 28672, "rank": 16, "x": "u8", "idle": 100},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


_HEADS = ((12, 12, 64), (32, 8, 128), (64, 8, 128), (16, 16, 80), (24, 8, 96), (8, 1, 256), (40, 2, 128), (20, 4, 64), (6, 6, 48), (16, 4, 192))


def draw(rng):
    kind = rng.choice(("append", "attention", "attention", "lora"))
    if kind == "lora":
        k, n, rows = _log(rng, 64, 8192), _log(rng, 16, 28672), _log(rng, 1, 2048)
        segments = rng.randint(1, min(rows, 32))
        return {"kind": kind, "rows": rows, "segments": segments, "adapters": rng.randint(1, segments), "k": k, "n": n,
                "rank": 8 * rng.choice((1, 2, 2, 3, 4, 6, 8)), "x": rng.choice(("f32", "u8")), "idle": rng.choice((0, 0, rng.randint(0, rows // 4)))}
    heads, kv_heads, dim = rng.choice(_HEADS)
    c = {"kind": kind, "sequences": _log(rng, 1, 64), "heads": heads, "kv_heads": kv_heads, "dim": dim, "cache": rng.choice(("f16", "i8")),
         "page": rng.choice((1, 7, 16, 16, 24, 32, 64, 100)), "order": rng.choice(("hnd", "nhd"))}
    if kind == "append":
        tokens = 1 if rng.random() < 0.4 else _log(rng, 2, 1024)
        while tokens * c["sequences"] * (heads + 2 * kv_heads) * dim > 4005 * 80 * 128:
            tokens = (tokens + 1) // 2
            c["sequences"] = (c["sequences"] + 1) // 2
        c |= {"tokens": tokens, "in": rng.choice(("f32", "f16")), "style": rng.choice(("half", "interleaved", "none")),
              "rotary": rng.choice((dim, dim, dim // 2)), "filled": rng.randint(0, 300), "pad": rng.choice((0, rng.randint(0, tokens - 1)))}
        return c
    longest = _log(rng, 1, 131072)
    while longest * c["sequences"] * kv_heads * dim > 131072 * 8 * 128:
        longest, c["sequences"] = (longest + 1) // 2, (c["sequences"] * 3 + 3) // 4
    c |= {"longest": longest, "shortest": rng.randint(1, longest), "q": rng.choice(("f32", "f16")), "out": rng.choice(("f32", "f16")),
          "window": rng.choice((0, 0, 0, rng.randint(1, longest))), "empty": rng.choice((0, 0, 1))}
    return c


_T = {"f32": torch.float32, "f16": torch.float16, "i8": torch.int8, "u8": torch.uint8}


def _cache(c, g, pages):
    """K and V pages of whatever earlier steps left in them; i8: with their scales [page][head][token]"""
    shape = (pages, c["kv_heads"], c["page"], c["dim"]) if c["order"] == "hnd" else (pages, c["page"], c["kv_heads"], c["dim"])
    s = {}
    for x in "kv":
        if c["cache"] == "f16":
            s[x + "_cache"] = torch.randn(shape, device="cuda", generator=g, dtype=torch.float16)
        else:
            s[x + "_cache"] = torch.randint(-127, 128, shape, device="cuda", generator=g, dtype=torch.int8)
            s[x + "_scale"] = 127.0 / (2.0 + 2.0 * torch.rand((pages, c["kv_heads"], c["page"]), device="cuda", generator=g))
    return s


def _prepare_append(c, g):
    b, t, ps, dim = c["sequences"], c["tokens"], c["page"], c["dim"]
    ctx = c["filled"] + t                                   # sequence i has filled - i tokens (at least none) in the cache
    tp = -(-ctx // ps)
    s = _cache(c, g, b * tp)
    start = (c["filled"] - torch.arange(b, device="cuda")).clamp(min=0)
    pos = start[:, None] + torch.arange(t, device="cuda")[None, :]
    if c["pad"]:                                            # the later a request, the shorter: its last rows are padding
        short = (torch.arange(b, device="cuda") * c["pad"]).clamp(max=t - 1)
        pos = torch.where(torch.arange(t, device="cuda")[None, :] < t - short[:, None], pos, -1)
    qkv = torch.randn((b * t, (c["heads"] + 2 * c["kv_heads"]) * dim), device="cuda", generator=g).to(_T[c["in"]])
    s |= {"c": c, "qkv": qkv, "q_out": torch.zeros((b * t, c["heads"], dim), dtype=_T[c["in"]], device="cuda"),
          "position": pos.reshape(-1).int(), "sequence": torch.arange(b, device="cuda", dtype=torch.int32).repeat_interleave(t),
          "table": torch.randperm(b * tp, device="cuda", generator=g).int().view(b, tp)}
    rotary = 0 if c["style"] == "none" else c["rotary"]
    s["rotary"] = rotary
    if rotary:
        angle = torch.arange(ctx, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary)[None, :]
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    return s


def _prepare_attention(c, g):
    b, ps = c["sequences"], c["page"]
    lens = torch.randint(c["shortest"], c["longest"] + 1, (b,), device="cuda", generator=g)
    lens[-1] = c["longest"]
    if c["empty"]:
        lens[: min(c["empty"], b)] = 0
    tp = -(-c["longest"] // ps)
    # as many pages as sequences of these lengths hold, in the order in which a server came to hand them out
    live = torch.arange(tp, device="cuda")[None, :] * ps < lens[:, None]
    pages = max(1, int(live.sum()))
    s = _cache(c, g, pages)
    table = torch.full((b, tp), -1, dtype=torch.int32, device="cuda")
    table[live] = torch.randperm(pages, device="cuda", generator=g).int()[: int(live.sum())]
    s |= {"c": c, "table": table, "length": lens.int(), "q": (2 * torch.randn((b, c["heads"], c["dim"]), device="cuda", generator=g)).to(_T[c["q"]]),
          "out": torch.empty((b, c["heads"], c["dim"]), dtype=_T[c["out"]], device="cuda"), "lse": torch.empty((b, c["heads"]), device="cuda"),
          "tmp": torch.empty(32 << 20, dtype=torch.uint8, device="cuda")}
    return s


def _prepare_lora(c, g):
    m, k, n, r, seg, ad = c["rows"], c["k"], c["n"], c["rank"], c["segments"], c["adapters"]
    used = m - c["idle"]                                    # rows behind the last segment have no adapter
    cut = torch.randperm(max(used - 1, 0), device="cuda", generator=g)[: seg - 1].sort().values + 1
    first = torch.zeros(seg + 1, dtype=torch.int32, device="cuda")
    first[1: 1 + cut.numel()] = cut.int()
    first[1 + cut.numel():] = used
    adapter = torch.arange(seg, device="cuda", dtype=torch.int32) % ad
    adapter = adapter[torch.randperm(seg, device="cuda", generator=g)].contiguous()
    if seg > 4:
        adapter[seg // 2] = -1                              # one request without an adapter
    ka = (k + 7) // 8 * 8
    s = {"c": c, "first_row": first, "adapter": adapter,
         "a": (torch.randn((ad, r, ka), device="cuda", generator=g) / math.sqrt(k)).half(),
         "b": (torch.randn((ad, n, r), device="cuda", generator=g) / math.sqrt(r)).half(),
         "scale": 0.5 + torch.rand(ad, device="cuda", generator=g), "y": torch.randn((m, n), device="cuda", generator=g),
         "tmp": torch.empty(32 << 20, dtype=torch.uint8, device="cuda")}
    if c["x"] == "f32":
        s["x"] = torch.randn((m, k), device="cuda", generator=g)
    else:
        s["x"] = (128 + 30 * torch.randn((m, k), device="cuda", generator=g)).round().clamp(0, 255).to(torch.uint8)
        s["row_scale"] = 20.0 + 20.0 * torch.rand(m, device="cuda", generator=g)
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"append": _prepare_append, "attention": _prepare_attention, "lora": _prepare_lora}[case["kind"]](case, g)


# ---- the framework's calls ---------------------------------------------------------------------------------------
def _p(t):
    return None if t is None else t.data_ptr()


def _own_cache(B, s):
    c, k = s["c"], s["k_cache"]
    st = k.stride()
    token, head = (st[2], st[1]) if c["order"] == "hnd" else (st[1], st[2])
    return B.KvCache(B.DT_F16 if c["cache"] == "f16" else B.DT_I8, k.shape[0], c["page"], c["kv_heads"], c["dim"], st[0], token, head,
                     k.data_ptr(), s["v_cache"].data_ptr(), _p(s.get("k_scale")), _p(s.get("v_scale")))


def _own_append(s):
    import bolt_b200 as B

    c, qkv, q_out, table = s["c"], s["qkv"], s["q_out"], s["table"]
    dt, at, row = (B.DT_F32, 4, qkv.shape[1]) if c["in"] == "f32" else (B.DT_F16, 2, qkv.shape[1])
    q = qkv.data_ptr()
    k = q + c["heads"] * c["dim"] * at
    v = k + c["kv_heads"] * c["dim"] * at
    rotary = s["rotary"]
    B.kv_append(_own_cache(B, s), B.KvAppend(
        qkv.shape[0], c["heads"], dt, dt, q, k, v, q_out.data_ptr(), row, row, row, c["heads"] * c["dim"], s["sequence"].data_ptr(),
        s["position"].data_ptr(), table.data_ptr(), table.shape[0], table.shape[1], rotary, c["style"] == "interleaved",
        s["cos"].shape[0] if rotary else 0, _p(s.get("cos")), _p(s.get("sin"))))


def _own_attention(s):
    import bolt_b200 as B

    c, table = s["c"], s["table"]
    dt = {"f32": B.DT_F32, "f16": B.DT_F16}
    row = c["heads"] * c["dim"]
    cache = _own_cache(B, s)
    call = B.PagedAttention(c["sequences"], c["heads"], dt[c["q"]], dt[c["out"]], s["q"].data_ptr(), s["out"].data_ptr(), s["lse"].data_ptr(), row, row,
                            table.data_ptr(), s["length"].data_ptr(), table.shape[1], c["window"], 1.0 / math.sqrt(c["dim"]), 0.0)
    B.paged_attention(cache, call, s["tmp"].numel(), s["tmp"].data_ptr())
    return {"out": s["out"], "lse": s["lse"]}


def _own_lora(s):
    import bolt_b200 as B

    c, x, y = s["c"], s["x"], s["y"]
    call = B.Lora(c["rows"], c["n"], c["k"], c["rank"], c["adapters"], c["segments"], B.DT_F32 if c["x"] == "f32" else B.DT_U8_Q, x.data_ptr(),
                  y.data_ptr(), x.shape[1], y.shape[1], s["a"].data_ptr(), s["b"].data_ptr(), s["a"].shape[2], s["scale"].data_ptr(),
                  s["first_row"].data_ptr(), s["adapter"].data_ptr(), 1.0, None, _p(s.get("row_scale")))
    B.lora(call, s["tmp"].numel(), s["tmp"].data_ptr())
    return {"y": y}


# ---- the plain forms -----------------------------------------------------------------------------------------------
def _rotate(x, s):
    r = s["rotary"]
    if r == 0:
        return x
    p = s["position"].clamp(min=0).long()
    cos, sin = s["cos"][p][:, None, :], s["sin"][p][:, None, :]
    if s["c"]["style"] == "half":
        a, b = x[..., : r // 2], x[..., r // 2: r]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., r:]), -1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    return torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2), x[..., r:]), -1)


def _plain_append(s):
    c, dim, t = s["c"], s["c"]["dim"], s["qkv"].shape[0]
    q, k, v = (x.reshape(t, -1, dim).float() for x in s["qkv"].split((c["heads"] * dim, c["kv_heads"] * dim, c["kv_heads"] * dim), 1))
    live = s["position"] >= 0
    s["q_out"][live] = _rotate(q, s).to(s["q_out"].dtype)[live]
    p = s["position"][live].long()
    page, at = s["table"][s["sequence"][live].long(), p // c["page"]].long(), p % c["page"]

    def keep(cache, scales, rows):
        rows = rows[live]
        if scales is not None:
            top = rows.abs().amax(-1)
            # (a quotient of two tensors is rounded once; torch multiplies by a reciprocal for a plain number)
            scale = torch.where(top == 0, torch.ones_like(top), torch.full_like(top, 127.0) / top)
            scales[page, :, at] = scale
            rows = (rows * scale[..., None]).round().clamp(-127, 127)
        if c["order"] == "hnd":
            cache[page, :, at] = rows.to(cache.dtype)
        else:
            cache[page, at] = rows.to(cache.dtype)

    keep(s["k_cache"], s.get("k_scale"), _rotate(k, s))
    keep(s["v_cache"], s.get("v_scale"), v)


def _values(s, x):
    """a cache as the numbers it stands for"""
    if s["c"]["cache"] == "f16":
        return s[x + "_cache"]
    scale = s[x + "_scale"][..., None]
    return s[x + "_cache"] / (scale if s["c"]["order"] == "hnd" else scale.transpose(1, 2))


def _append_outputs(s):
    return {"q": s["q_out"], "k": _values(s, "k"), "v": _values(s, "v")}


def _plain_attention(s):
    c = s["c"]
    b, h, hk, d = c["sequences"], c["heads"], c["kv_heads"], c["dim"]
    table = s["table"].clamp(min=0).long()
    length = table.shape[1] * c["page"]

    def rows(x):
        pages = s[x + "_cache"][table].float()              # [b, pages, ...]
        if c["order"] == "nhd":
            pages = pages.transpose(2, 3)
        if c["cache"] == "i8":
            pages = pages / s[x + "_scale"][table][..., None]
        return pages.transpose(1, 2).reshape(b, hk, length, d)

    at = torch.arange(length, device="cuda")[None, :]
    end = s["length"][:, None].long()
    live = (at < end) & (at >= end - c["window"]) if c["window"] else at < end
    q = s["q"].float().view(b, hk, h // hk, d)
    scores = (q @ rows("k").transpose(-1, -2)) * (1.0 / math.sqrt(d))
    scores = torch.where(live[:, None, None, :], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = (scores - torch.where(top == -math.inf, 0.0, top)).exp()
    total = weights.sum(-1, keepdim=True)
    out = (weights @ rows("v")) / torch.where(total == 0, 1.0, total)
    lse = (top + total.log()).view(b, h)
    s["out"].copy_(out.view(b, h, d))
    s["lse"].copy_(lse)
    return {"out": s["out"], "lse": s["lse"]}


def _plain_lora(s):
    c = s["c"]
    row = torch.arange(c["rows"], device="cuda")[:, None]
    inside = (row >= s["first_row"][None, :-1]) & (row < s["first_row"][None, 1:])                 # [rows, segments]
    which = s["adapter"][:, None] == torch.arange(c["adapters"], device="cuda")[None, :]           # [segments, adapters]
    mine = inside.float() @ which.float()
    x = s["x"].float()
    if c["x"] == "u8":
        x = (x - 128.0) / s["row_scale"][:, None]
    a, b = s["a"][:, :, : c["k"]].float().reshape(-1, c["k"]), s["b"].float().transpose(1, 2).reshape(-1, c["n"])
    t = (x @ a.T).view(c["rows"], c["adapters"], c["rank"]) * (mine * s["scale"][None, :])[:, :, None]
    s["y"] += t.view(c["rows"], -1) @ b
    return {"y": s["y"]}


def run(state):
    kind = state["c"]["kind"]
    if kind == "append":
        if own:
            _own_append(state)
        else:
            _plain_append(state)
        return _append_outputs(state)
    if own:
        return _own_attention(state) if kind == "attention" else _own_lora(state)
    return _plain_attention(state) if kind == "attention" else _plain_lora(state)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------
def _exact_append(s):
    """Products and sums of binary32 numbers in 64 bits, rounded where the operator's definition rounds; a row at a time."""
    c, d, r = s["c"], s["c"]["dim"], s["rotary"]
    f32 = lambda x: x.float().double()  # noqa: E731
    live = [i for i, p in enumerate(s["position"].tolist()) if p >= 0]
    pos = s["position"].tolist()
    idx = torch.tensor(live, device="cuda")
    x = s["qkv"].double()[idx].view(len(live), -1, d)
    turned = x.clone()
    if r:
        angles = [pos[i] for i in live]
        cos, sin = s["cos"].double()[angles].unsqueeze(1), s["sin"].double()[angles].unsqueeze(1)
        first = torch.arange(r // 2, device="cuda") * (1 if c["style"] == "half" else 2)
        second = first + (r // 2 if c["style"] == "half" else 1)
        turned[..., first] = f32(f32(x[..., first] * cos) - f32(x[..., second] * sin))
        turned[..., second] = f32(f32(x[..., second] * cos) + f32(x[..., first] * sin))
    h, hk = c["heads"], c["kv_heads"]
    q = s["q_out"].double()
    q[idx] = turned[:, :h]
    out = {"q": q}
    seq, table = s["sequence"].tolist(), s["table"].tolist()
    page = torch.tensor([table[seq[i]][pos[i] // c["page"]] for i in live], device="cuda")
    at = torch.tensor([pos[i] % c["page"] for i in live], device="cuda")
    for name, rows in (("k", turned[:, h: h + hk]), ("v", x[:, h + hk:])):
        cache = s[name + "_cache"].double()
        if c["order"] == "nhd":
            cache = cache.transpose(1, 2)
        if c["cache"] == "i8":
            scale = s[name + "_scale"].double()
            top = rows.abs().max(-1).values
            new = torch.where(top > 0, f32(127.0 / top), 1.0)
            scale[page, :, at] = new
            cache = cache.clone()
            cache[page, :, at] = torch.round(f32(rows * new[..., None])).clamp(-127, 127)
            cache = cache / scale[..., None]
        else:
            cache = cache.clone()
            cache[page, :, at] = rows
        out[name] = cache.transpose(1, 2) if c["order"] == "nhd" else cache
    return out


def _exact_attention(s):
    c = s["c"]
    h, hk, d, ps = c["heads"], c["kv_heads"], c["dim"], c["page"]
    out = torch.zeros((c["sequences"], h, d), dtype=torch.float64, device="cuda")
    lse = torch.full((c["sequences"], h), -math.inf, dtype=torch.float64, device="cuda")
    for i, end in enumerate(s["length"].tolist()):
        begin = max(0, end - c["window"]) if c["window"] else 0
        if end == 0:
            continue
        t = torch.arange(begin, end, device="cuda")
        page, at = s["table"][i][t // ps].long(), t % ps
        kv = []
        for x in "kv":
            cache = s[x + "_cache"]
            rows = (cache[page, :, at] if c["order"] == "hnd" else cache[page, at]).double()       # [tokens, heads, dim]
            if c["cache"] == "i8":
                rows = rows / s[x + "_scale"][page, :, at].double()[..., None]
            kv.append(rows.repeat_interleave(h // hk, 1))
        z = torch.einsum("hd,thd->ht", s["q"][i].double(), kv[0]) / math.sqrt(d)
        lse[i] = torch.logsumexp(z, -1)
        out[i] = torch.einsum("ht,thd->hd", torch.exp(z - lse[i][:, None]), kv[1])
    return {"out": out, "lse": lse}


def _exact_lora(s):
    c = s["c"]
    y = s["y"].double()
    first, adapter = s["first_row"].tolist(), s["adapter"].tolist()
    for i, a in enumerate(adapter):
        if a < 0:
            continue
        rows = slice(first[i], first[i + 1])
        x = s["x"][rows].double()
        if c["x"] == "u8":
            x = (x - 128.0) / s["row_scale"][rows].double()[:, None]
        y[rows] += s["scale"][a].double() * ((x @ s["a"][a][:, : c["k"]].double().T) @ s["b"][a].double().T)
    return {"y": y}


def exact(case, seed):
    return {"append": _exact_append, "attention": _exact_attention, "lora": _exact_lora}[case["kind"]](prepare(case, seed))


def work(case):
    c, size = case, {"f32": 4, "f16": 2, "i8": 1, "u8": 1}
    if c["kind"] == "lora":
        rows = c["rows"] - c["idle"]
        return {"bytes": rows * c["k"] * size[c["x"]] + 8 * rows * c["n"] + 2 * c["adapters"] * c["rank"] * (c["k"] + c["n"]),
                "flops": 2 * rows * c["rank"] * (c["k"] + c["n"])}
    h, hk, d = c["heads"], c["kv_heads"], c["dim"]
    row = d * size[c["cache"]] + (4 if c["cache"] == "i8" else 0)
    if c["kind"] == "append":
        t = c["sequences"] * c["tokens"] - sum(min(i * c["pad"], c["tokens"] - 1) for i in range(c["sequences"]))
        rotary = 0 if c["style"] == "none" else c["rotary"]
        return {"bytes": t * ((2 * h + 2 * hk) * d * size[c["in"]] + 2 * hk * row + 4 * rotary), "flops": 3 * t * (h + hk) * rotary}
    tokens = sum((c["shortest"] + c["longest"]) / 2 if i < c["sequences"] - 1 else c["longest"] for i in range(min(c["empty"], c["sequences"]), c["sequences"]))
    if c["window"]:
        tokens = min(tokens, c["window"] * c["sequences"])
    return {"bytes": 2 * tokens * hk * row + c["sequences"] * h * (d * (size[c["q"]] + size[c["out"]]) + 4), "flops": 4 * tokens * h * d}
