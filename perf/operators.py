"""What the paged key / value cache and its attention are timed on.

A server that decodes many conversations keeps their keys and values in pages of one pool (a page table per conversation) and may keep them
in eight bits. Three operators work on such a cache; a case's ``"kind"`` says which it takes:

``write``   the new tokens' heads are normalised, rotated and appended to the cache (``append``), then the rows just written are read back (``read``)
``read``    whole conversations are read back as dense rows (moved to another pool, written to disk)
``attend``  the new tokens' queries over everything that is cached, single tokens and chunks of a prompt

Head counts and sizes are those of the repository's model shapes: 12 query heads on 4 key heads of 256, 20 on 5 of 128, 32 on 4 of 128, and
8 on 2 of 64 for small models. ``cache`` is the stored type: f16, bf16, or q8 (8-bit codes and one 32-bit scale per row and head).
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
MOST_FLOPS, MOST_BYTES = 3.2e11, 4.0e8  # no drawn case costs more than the largest listed ones


def _case(name, kind, heads, cache, seqs, new, cached, **more):
    """`new`: tokens of the longest chunk; `cached`: tokens of the longest conversation, the new ones included; `mix` says how the others differ."""
    qh, kvh, hd = heads
    c = dict(kind=kind, q_heads=qh, kv_heads=kvh, head_dim=hd, cache=cache, type="bf16" if cache == "bf16" else "f16", seqs=seqs, new=new, cached=cached, page=64, mix="ragged",
             cap=0.0, window=0, norm=False, neox=False, rope=hd)
    c.update(more)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # One conversation's next token: a layer's cache write, where latency is all there is.
        _case("write_one", "write", (20, 5, 128), "f16", 1, 1, 1536),
        # 32 conversations, a token each: what a batched decode step writes per layer.
        _case("write_step", "write", (12, 4, 256), "q8", 32, 1, 2048),
        # A long prompt in one pass, with norms of queries and keys, into an eight-bit cache.
        _case("write_prompt", "write", (32, 4, 128), "q8", 1, 4096, 4096, type="bf16", norm=True, neox=True),
        # A short conversation is read back.
        _case("read_one", "read", (20, 5, 128), "bf16", 1, 513, 513, page=16),
        # Sixteen long conversations leave an eight-bit pool at once.
        _case("read_all", "read", (12, 4, 256), "q8", 16, 7000, 7000),
        # The next token of a conversation that has just begun: the smallest call.
        _case("attend_first", "attend", (20, 5, 128), "f16", 1, 1, 97, page=16),
        # A batched decode step: 32 conversations of different lengths, a token each, eight-bit cache.
        _case("attend_step", "attend", (12, 4, 256), "q8", 32, 1, 4096),
        # A single very long conversation: all of the device on one row of queries per head.
        _case("attend_long", "attend", (20, 5, 128), "f16", 1, 1, 65431, page=128),
        # Drafted tokens are checked: five per conversation at once, eight-bit cache.
        _case("attend_draft", "attend", (20, 5, 128), "q8", 16, 5, 3001, page=32, type="bf16"),
        # The first pass of a prompt: as many tokens as a pass takes, nothing cached before them.
        _case("attend_prompt", "attend", (12, 4, 256), "f16", 1, 1024, 1024),
        # A later pass of a very long prompt: the largest call.
        _case("attend_chunk", "attend", (20, 5, 128), "q8", 1, 2048, 16384),
        # A step that carries one chunk of a prompt and the next tokens of others, with capped scores and a window.
        _case("attend_mixed", "attend", (32, 4, 128), "bf16", 8, 257, 3500, mix="one", cap=30.0, window=1024),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    while True:
        kind = rng.choice(["write", "read", "attend", "attend", "attend"])
        heads = rng.choice([(12, 4, 256), (20, 5, 128), (32, 4, 128), (8, 2, 64)])
        cache = rng.choice(["f16", "bf16", "q8", "q8"])
        more = dict(page=rng.choice([16, 32, 64, 128]), type=rng.choice(["f16", "bf16"]) if cache == "q8" else cache)
        if kind == "attend":
            form = rng.choice(["step", "step", "draft", "chunk", "chunk", "mixed"])
            if form == "step":
                seqs, new, cached = _log(rng, 1, 64), 1, _log(rng, 2, 65536)
            elif form == "draft":
                seqs, new, cached = _log(rng, 1, 32), rng.randint(2, 9), _log(rng, 16, 8192)
            elif form == "chunk":
                seqs, new, cached = 1, _log(rng, 16, 2048), _log(rng, 16, 16384)
            else:
                seqs, new, cached = rng.randint(2, 12), _log(rng, 16, 400), _log(rng, 64, 4096)
                more["mix"] = "one"
            more.update(cap=rng.choice([0.0, 0.0, 30.0, 50.0]), window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]))
        elif kind == "write":
            seqs, new = rng.choice([(_log(rng, 1, 128), 1), (_log(rng, 1, 8), _log(rng, 2, 700)), (1, _log(rng, 16, 4096))])
            cached = _log(rng, 16, 8192)
            more.update(norm=rng.random() < 0.5, neox=rng.random() < 0.5, rope=rng.choice([heads[2], heads[2] // 2]))
        else:
            seqs, new = _log(rng, 1, 16), _log(rng, 2, 7000)
            cached = new
        c = _case(None, kind, heads, cache, seqs, min(new, max(new, cached)), max(new, cached), **more)
        w = work(c)
        if w["flops"] <= MOST_FLOPS and w["bytes"] <= MOST_BYTES and c["seqs"] * c["new"] * c["q_heads"] * c["cached"] <= 7.0e8:
            return c


def _lengths(c):
    """(new tokens, cached tokens) of every conversation: from the case alone, so that work() knows them. The first is the longest."""
    new, cached = [], []
    for s in range(c["seqs"]):
        f = 1.0 - 0.75 * ((s * 0.618034) % 1.0)  # the others: between a quarter of it and all of it
        n = c["new"] if s == 0 or c["mix"] != "one" else 1
        if c["kind"] == "read":
            n = max(1, int(c["new"] * f))
        elif c["kind"] == "write" and s:
            n = max(1, int(c["new"] * f))
        length = max(n, int(c["cached"] * f))
        new.append(n)
        cached.append(n if c["kind"] == "read" else length)
    return new, cached


def work(case):
    new, cached = _lengths(case)
    qh, kvh, hd, T = case["q_heads"], case["kv_heads"], case["head_dim"], sum(new)
    row = kvh * (hd + 4 if case["cache"] == "q8" else 2 * hd) * 2  # a token's keys and values as they are stored
    if case["kind"] == "read":
        return {"bytes": T * (row + 2 * kvh * hd * 2), "flops": 2 * T * kvh * hd}
    if case["kind"] == "write":  # read the heads, write queries and rows, read the rows again and write them densely
        return {"bytes": T * ((qh + 2 * kvh) * hd * 2 + qh * hd * 2 + 2 * row + 2 * kvh * hd * 2), "flops": T * (qh + 2 * kvh) * hd * 10}
    pairs, rows = 0, 0
    for n, length in zip(new, cached):
        w = case["window"] or length
        a, b = length - n + 1, length  # keys up to its own place, of the first new token and of the last
        cut = max(0, min(b, w) - a + 1)  # tokens that the window does not reach behind
        pairs += (a + a + cut - 1) * cut // 2 + (n - cut) * w
        rows += min(length, n - 1 + w)
    return {"bytes": rows * row + 2 * T * qh * hd * 2, "flops": 4 * hd * qh * pairs}


def _table(c, cached, gen):
    """Pages of the conversations, scattered over a pool that is somewhat larger than they need."""
    per = [-(-n // c["page"]) for n in cached]
    pages = sum(per) + 3
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    table = torch.zeros(c["seqs"], max(per), dtype=torch.int32, device=DEV)
    at = 0
    for s, n in enumerate(per):
        table[s, :n] = order[at:at + n]
        at += n
    return table, pages


def _rows_of(c, tokens, gen, outliers):
    """Keys or values of `tokens` tokens as a cache of this type can hold them exactly: what the cache is filled with before the call.
    Returns (values in 32 bits, codes or None, scales or None)."""
    x = torch.randn(tokens, c["kv_heads"], c["head_dim"], generator=gen, device=DEV)
    if outliers:  # a few channels of keys are much larger than the others
        x = x * (1.0 + 5.0 * (torch.rand(1, c["kv_heads"], c["head_dim"], generator=gen, device=DEV) > 0.97))
    if c["cache"] != "q8":
        x = x.to(TYPES[c["cache"]]).float()
        return x, None, None
    most, where = x.abs().max(-1, keepdim=True)
    scale = (most / 127).to(torch.bfloat16).float()  # so few bits that 127 * scale is exact
    codes = (x / scale).round().clamp_(-127, 127)
    codes.scatter_(-1, where, torch.sign(torch.gather(x, -1, where)) * 127)
    return codes * scale, codes.to(torch.int8), scale


def _angles(positions, dims):
    """cos at 2i and sin at 2i + 1 of every position's row."""
    f = 1000042.0 ** (-torch.arange(0, dims, 2, device=DEV, dtype=torch.float64) / dims)
    a = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * f
    return torch.stack([a.cos(), a.sin()], -1).reshape(positions, dims).float()


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(seed)
    new, cached = _lengths(c)
    qh, kvh, hd, P, T = c["q_heads"], c["kv_heads"], c["head_dim"], c["page"], sum(new)
    dt = TYPES[c["type"]]
    starts = torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32)
    lengths = torch.tensor(cached, dtype=torch.int32, device=DEV)
    table, pages = _table(c, cached, gen)
    st = dict(case=c, starts=starts, lengths=lengths, table=table, pages=pages, tokens=T, most_new=max(new), most=max(cached), scale=hd ** -0.5)
    seq = torch.repeat_interleave(torch.arange(c["seqs"], device=DEV), torch.tensor(new, device=DEV))
    place = torch.arange(T, device=DEV) - starts[seq].long() + (lengths[seq] - (starts[1:] - starts[:-1])[seq]).long()
    if not own:
        st.update(seq=seq, place=place)
    if c["kind"] == "write":
        rows = torch.randn(T, qh + 2 * kvh, hd, generator=gen, device=DEV)
        rows = (rows * torch.exp(0.3 * torch.randn(1, qh + 2 * kvh, hd, generator=gen, device=DEV))).to(dt)  # one product's row: q | k | v
        st.update(q=rows[:, :qh], k=rows[:, qh:qh + kvh], v=rows[:, qh + kvh:], q_norm=None, k_norm=None)
        if c["norm"]:
            st.update(q_norm=1.0 + 0.2 * torch.randn(hd, generator=gen, device=DEV), k_norm=1.0 + 0.2 * torch.randn(hd, generator=gen, device=DEV))
        st["angles"] = _angles(max(cached), c["rope"])
        fill = None
    else:
        total = sum(cached)
        fill = [_rows_of(c, total, gen, outliers) for outliers in (True, False)]
        if c["kind"] == "attend":
            st["q"] = torch.randn(T, qh, hd, generator=gen, device=DEV).to(dt)
    if own:
        import quintrit_b200 as q

        cache = q.PagedCache(1, pages, P, kvh, hd, c["cache"])
        st.update(cache=cache, rows=q.PagedRows(starts, lengths, table, tokens=T, max_new=max(new), max_length=max(cached)))
        if fill is not None:
            all_starts = torch.tensor([0] + cached, device=DEV).cumsum(0).to(torch.int32)
            cache.append(0, q.PagedRows(all_starts, lengths, table, tokens=sum(cached), max_new=max(cached), max_length=max(cached)), None, fill[0][0], fill[1][0])
        if c["kind"] != "attend":
            st.update(k_out=torch.empty(T, kvh, hd, dtype=dt, device=DEV), v_out=torch.empty(T, kvh, hd, dtype=dt, device=DEV))
        if c["kind"] != "read":
            st["q_out"] = torch.empty(T, qh, hd, dtype=dt, device=DEV)
        if c["kind"] == "attend":
            st["workspace"] = cache.attend_workspace(st["rows"], qh)
        return st
    shape = (pages, kvh, P, hd)
    store = torch.int8 if c["cache"] == "q8" else TYPES[c["cache"]]
    st.update(keys=torch.zeros(shape, dtype=store, device=DEV), values=torch.zeros(shape, dtype=store, device=DEV),
              key_scales=torch.zeros(shape[:3], device=DEV), value_scales=torch.zeros(shape[:3], device=DEV))
    if fill is not None:
        n = torch.tensor(cached, device=DEV)
        s = torch.repeat_interleave(torch.arange(c["seqs"], device=DEV), n)
        p = torch.arange(sum(cached), device=DEV) - (n.cumsum(0) - n)[s]
        page, row = table[s, p // P].long(), p % P
        for (x, codes, scale), to, scales in zip(fill, ("keys", "values"), ("key_scales", "value_scales")):
            st[to][page, :, row] = x.to(store) if codes is None else codes
            if codes is not None:
                st[scales][page, :, row] = scale[..., 0]
    return st


def _rotated(x, place, st):
    """The heads [tokens][heads][size] with their first `rope` values rotated by the angles of their places."""
    c, dims = st["case"], st["case"]["rope"]
    cos, sin = (st["angles"][place][:, None, i::2] for i in (0, 1))
    if c["neox"]:
        a, b = x[..., :dims // 2], x[..., dims // 2:dims]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., dims:]], -1)
    a, b = x[..., 0:dims:2], x[..., 1:dims:2]
    return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), x[..., dims:]], -1)


def _normed(x, weights):
    x = x.float()
    return x if weights is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weights


def _stored(st, which, page, row):
    """Rows of the plain cache as 32-bit values: [...][heads][size]."""
    x = st[which][page, :, row].float()
    return x * st["key_scales" if which == "keys" else "value_scales"][page, :, row][..., None] if st["case"]["cache"] == "q8" else x


def _plain_write(st):
    c, place = st["case"], st["place"]
    page, row = st["table"][st["seq"], place // c["page"]].long(), place % c["page"]
    query = _rotated(_normed(st["q"], st["q_norm"]), place, st)
    for x, which, scales in ((_rotated(_normed(st["k"], st["k_norm"]), place, st), "keys", "key_scales"), (st["v"].float(), "values", "value_scales")):
        if c["cache"] == "q8":
            scale = (x.abs().amax(-1, keepdim=True) / 127).clamp_min(2.0 ** -100)
            st[scales][page, :, row] = scale[..., 0]
            x = (x / scale).round().clamp_(-127, 127)
        st[which][page, :, row] = x.to(st[which].dtype)
    dt = st["q"].dtype
    return {"q": query.to(dt), "k": _stored(st, "keys", page, row).to(dt), "v": _stored(st, "values", page, row).to(dt)}


def _plain_read(st):
    c, place, dt = st["case"], st["place"], TYPES[st["case"]["type"]]
    page, row = st["table"][st["seq"], place // c["page"]].long(), place % c["page"]
    return {"k": _stored(st, "keys", page, row).to(dt), "v": _stored(st, "values", page, row).to(dt)}


def _plain_attend(st):
    """All conversations at once, each padded to the longest."""
    c, q = st["case"], st["q"]
    S, N, L, g = c["seqs"], st["most_new"], st["most"], c["q_heads"] // c["kv_heads"]
    j = torch.arange(L, device=DEV)
    page, row = st["table"][:, j // c["page"]].long(), (j % c["page"]).expand(S, L)
    k, v = _stored(st, "keys", page, row), _stored(st, "values", page, row)  # [S][L][heads][size]
    i = st["starts"][:-1, None].long() + torch.arange(N, device=DEV)
    new = (st["starts"][1:] - st["starts"][:-1]).long()
    x = q[i.clamp_max(st["tokens"] - 1)].float() * st["scale"]  # [S][N][q heads][size]
    x = x.reshape(S, N, c["kv_heads"], g, -1).permute(0, 2, 3, 1, 4).reshape(S, c["kv_heads"], g * N, -1)
    z = x @ k.permute(0, 2, 3, 1)
    if c["cap"]:
        z = c["cap"] * torch.tanh(z / c["cap"])
    p = st["lengths"].long()[:, None] - new[:, None] + torch.arange(N, device=DEV)  # the place of every new token
    seen = j <= p[..., None]
    if c["window"]:
        seen &= j > p[..., None] - c["window"]
    z = z.reshape(S, c["kv_heads"], g, N, L).masked_fill_(~seen[:, None, None], -math.inf)
    e = torch.exp(z - z.amax(-1, keepdim=True).clamp_min(-3e38))
    out = (e.reshape(S, c["kv_heads"], g * N, L) @ v.permute(0, 2, 1, 3)).reshape(S, c["kv_heads"], g, N, -1) / e.sum(-1, keepdim=True).clamp_min(1e-38)
    out = out.permute(0, 3, 1, 2, 4).reshape(S, N, c["q_heads"], -1)
    return out[st["seq"], torch.arange(st["tokens"], device=DEV) - st["starts"][st["seq"]].long()].to(q.dtype)


def run(state):
    st, kind = state, state["case"]["kind"]
    if own:
        c, cache = st["case"], st["cache"]
        if kind == "attend":
            return cache.attend(0, st["rows"], st["q"], out=st["q_out"], scale=st["scale"], cap=c["cap"], window=c["window"], workspace=st["workspace"])
        if kind == "write":
            cache.append(0, st["rows"], st["q"], st["k"], st["v"], q_out=st["q_out"], q_norm=st["q_norm"], k_norm=st["k_norm"], cos_sin=st["angles"], neox=c["neox"])
        k, v = cache.read(0, st["rows"], k_out=st["k_out"], v_out=st["v_out"])
        return {"q": st["q_out"], "k": k, "v": v} if kind == "write" else {"k": k, "v": v}
    return _plain_attend(st) if kind == "attend" else _plain_write(st) if kind == "write" else _plain_read(st)


def exact(case, seed):
    """The operators in 64 bits, conversation by conversation, without pages."""
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    new, cached = _lengths(case)
    c, hd, qh, kvh = case, case["head_dim"], case["q_heads"], case["kv_heads"]
    q8 = c["cache"] == "q8"

    def conversation(which, s, length):
        pages = st["table"][s, :-(-length // c["page"])].long()
        x = st[which][pages].double()  # [pages][heads][rows][size]
        if q8:
            x = x * st["key_scales" if which == "keys" else "value_scales"][pages].double()[..., None]
        return x.transpose(1, 2).reshape(-1, kvh, hd)[:length]

    if c["kind"] == "read":
        return {n: torch.cat([conversation(w, s, cached[s]) for s in range(c["seqs"])]) for n, w in (("k", "keys"), ("v", "values"))}
    if c["kind"] == "write":
        place = torch.cat([torch.arange(length - n, length, device=DEV) for n, length in zip(new, cached)])
        half = c["rope"] // 2
        angle = st["angles"].double()[place].reshape(-1, 1, half, 2)
        turn = torch.complex(angle[..., 0], angle[..., 1])

        def heads(x, weights):
            x = x.double()
            if weights is not None:
                x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / hd + 1e-6) * weights.double()
            y = x.clone()
            first, second = (slice(0, half), slice(half, 2 * half)) if c["neox"] else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
            z = torch.complex(x[..., first], x[..., second]) * turn
            y[..., first], y[..., second] = z.real, z.imag
            return y

        def held(x):
            if not q8:
                return x
            d = torch.clamp(x.abs().max(-1, keepdim=True).values / 127.0, min=2.0 ** -100)
            return torch.round(x / d) * d

        return {"q": heads(st["q"], st["q_norm"]), "k": held(heads(st["k"], st["k_norm"])), "v": held(st["v"].double())}
    out = torch.empty(st["tokens"], qh, hd, dtype=torch.float64, device=DEV)
    t0 = 0
    for s in range(c["seqs"]):
        n, length = new[s], cached[s]
        k, v = conversation("keys", s, length), conversation("values", s, length)
        place, j = torch.arange(length - n, length, device=DEV)[:, None], torch.arange(length, device=DEV)[None]
        hidden = (j > place) | ((j <= place - c["window"]) if c["window"] else torch.zeros_like(j > place))
        for h in range(qh):
            z = st["q"][t0:t0 + n, h].double() @ k[:, h // (qh // kvh)].T * st["scale"]
            if c["cap"]:
                z = torch.tanh(z / c["cap"]) * c["cap"]
            out[t0:t0 + n, h] = torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ v[:, h // (qh // kvh)]
        t0 += n
    return out
