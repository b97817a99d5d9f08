"""A batch whose sequences share one cache in pages (quintrit_b200_batch_create_paged): append, attention and read run together in a decoder's passes, next to the batch with a cache per
sequence."""
import numpy as np
import pytest

import oracle
import quintrit_b200 as q
from quintrit_b200 import synth

pytestmark = pytest.mark.gpu

HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _spec(arch, config, ctx=1024, hidden=256, heads=(4, 2, 64), **kw):
    return synth.make_model(arch, True, hidden, 512, 2, *heads, 300, ctx, 500000.0, 1e-5, config=config, random_norms=True, **kw)


def _prompts(lengths, vocab, seed=40):
    return [synth.prompt_tokens(seed + i, n, vocab) for i, n in enumerate(lengths)]


def _run(d, prompts, fed, **kw):
    """Logits of the prompts' ends and of every step with the given tokens, [1 + steps][sequences][vocab], and the batch."""
    b = q.Batch(d, len(prompts), **kw)
    out = [np.stack([b.prefill(s, p)[0] for s, p in enumerate(prompts)])]
    for tokens in fed:
        out.append(b.step(tokens=tokens, want_logits=True)[1])
    return np.stack(out), b


def _round(x, cache, query=False):
    """Queries, and keys and values of a head, as a cache of that type keeps them (queries of Q8: 11 bits of each value)."""
    if cache == "f16" or (cache == "q8" and query):
        return x.astype(np.float16).astype(np.float64)
    if cache == "bf16":
        u = x.astype(np.float32).view(np.uint32)
        return ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32).astype(np.float64)
    d = np.maximum(np.abs(x).max(-1, keepdims=True) / 127, 2.0 ** -100)
    return np.rint(x / d) * d


def _model(spec, tokens, cache):
    """The decoder in 64 bits over one sequence, with the integer products and roundings of the model's definition, queries, keys and values rounded as the paged cache does; logits of every token."""
    H, I, qh, kvh, hd = (spec[k] for k in ("hidden", "inter", "q_heads", "kv_heads", "head_dim"))
    n, qd, kvd = len(tokens), qh * hd, kvh * hd
    shapes = [(qd, H), (kvd, H), (kvd, H), (H, qd), (I, H), (I, H), (H, I)]

    def norm(x, w):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + spec["eps"]) * w

    def project(x, l, *which):
        s = 127 / np.abs(x).max(-1, keepdims=True)
        codes = np.clip(np.sign(x) * np.floor(np.abs(x * s) + 0.5), -128, 127)
        return [codes @ oracle.unpack_planar(spec["weights"][l * 7 + k], *shapes[k]).astype(np.float64).T * spec["scales"][l * 7 + k] / s for k in which]

    half = spec["rope_dims"] // 2
    angle = np.arange(n)[:, None, None] * spec["rope_theta"] ** (-np.arange(half) / half)
    c, sn = np.cos(angle), np.sin(angle)

    def rotate(x):
        first, second = (np.arange(half), np.arange(half) + half) if spec["arch"] != q.ARCH_LLAMA else (2 * np.arange(half), 2 * np.arange(half) + 1)
        out = x.copy()
        out[..., first], out[..., second] = x[..., first] * c - x[..., second] * sn, x[..., first] * sn + x[..., second] * c
        return out

    table = np.asarray(spec["embed"], np.uint16).view(np.float16).reshape(-1, H).astype(np.float64)
    head = table if spec["lm_head"] is None else np.asarray(spec["lm_head"], np.uint16).view(np.float16).reshape(-1, H).astype(np.float64)
    x = table[np.asarray(tokens, np.int64)]
    for l in range(spec["layers"]):
        w = spec["norms"][l * 4:l * 4 + 4]
        a, k, v = (y.reshape(n, -1, hd) for y in project(norm(x, w[0]), l, 0, 1, 2))
        a, k, v = _round(rotate(a), cache, True), _round(rotate(k), cache), _round(v, cache)
        k, v = (np.repeat(y, qh // kvh, axis=1) for y in (k, v))
        z = np.einsum("ihd,jhd->hij", a, k) * hd ** -0.5
        z[:, np.triu(np.ones((n, n), bool), 1)] = -np.inf
        p = np.exp(z - z.max(-1, keepdims=True))
        o = np.einsum("hij,jhd->ihd", p / p.sum(-1, keepdims=True), v).reshape(n, qd)
        x = x + project(norm(o, w[2]) if w[2] is not None else o, l, 3)[0]
        g, u = project(norm(x, w[1]), l, 4, 5)
        y = np.maximum(g, 0) ** 2 * u if spec["arch"] == q.ARCH_BITNET else g / (1 + np.exp(-g)) * u
        x = x + project(norm(y, w[3]) if w[3] is not None else y, l, 6)[0]
    return norm(x, spec["out_norm"]) @ head.T


# How far the logits may lie apart. Against the model in 64 bits the attention differs by the rounding of its weights, 2^-9 relative at most, and by what 32-bit scores of some tens are off; that is less
# than a step of the activations' 8-bit codes (1 / 127 of a row's maximum, 3 to 6 times its root mean square: 2.4 to 4.7% of that). A difference within a step flips a code or not, so that its root
# mean square grows at every quantisation to at most a step: over the four products of two layers sqrt(2 (3 * 2.4^2 + 4.7^2)) = 8.8% of the rows', and as much of the logits', which are linear in
# them. Twice that is allowed; rows of another position or page would be as far off as the logits are large. A batch with a cache per sequence keeps F16 keys and values but F32 queries: a query's
# rounding changes a score by 2^-11 of the sum of its products, hundredths, and is held against the same limit for F16 (BF16 and Q8 move scores of some tens by tenths: there only the model counts).
# Where one value makes most of a row (a product of three normal values, after relu^2) a step is up to 1 / 127 of sqrt(512) root mean squares, 18%, and a flip alone reaches the limit: in the BitNet
# model below, computed in 64 bits over 518 positions, weights off by 2^-11, 2^-9 and 2^-7 at random move the logits of 0.6, 2.1 and 4.2% of the positions by more than it (by 0.6 at most). So one in
# ten may be further off, not more than three of a sequence's ten, and none by 1.
FAR = 0.18


def _far(a, b):
    return float(np.sqrt(np.mean((a - b) ** 2) / np.mean(b ** 2)))


def _near(far):
    far = np.asarray(far)
    assert (far < 1).all() and (far >= FAR).mean() <= 0.1 and ((far >= FAR).sum(axis=0) <= 3).all(), far.round(3)


@pytest.mark.parametrize("cache,page_tokens", [("f16", 16), ("bf16", 64), ("q8", 32)])
@pytest.mark.parametrize("arch,heads", [(q.ARCH_LLAMA, (4, 2, 64)), (q.ARCH_BITNET, (4, 1, 64)), (q.ARCH_LLAMA, (2, 2, 128)), (q.ARCH_LLAMA, (2, 1, 256))])
def test_next_to_a_cache_per_sequence(arch, heads, cache, page_tokens):
    spec = _spec(arch, 191, heads=heads, tied=arch == q.ARCH_BITNET)
    lengths = [1, 3, 250, 41, 509, 17]
    prompts = _prompts(lengths, spec["vocab"])
    fed = [synth.prompt_tokens(70 + k, len(lengths), spec["vocab"]) for k in range(9)]  # more steps than a captured one needs, and pages end among them
    d = q.Decoder(spec)
    got, paged = _run(d, prompts, fed, pages=sum(-(-(n + 9) // page_tokens) for n in lengths), page_tokens=page_tokens, cache=cache)
    assert list(paged.positions()) == [n + 9 for n in lengths]
    assert paged.pages()[1] == 0  # every page is in use
    want = np.stack([_model(spec, list(p) + [t[s] for t in fed], cache)[len(p) - 1:] for s, p in enumerate(prompts)], 1)
    _near([[_far(got[k, s], want[k, s]) for s in range(len(lengths))] for k in range(10)])
    if cache == "f16":
        want, plain = _run(d, prompts, fed)
        assert list(paged.positions()) == list(plain.positions())
        assert np.array_equal(got[0, 0].view(np.uint32), want[0, 0].view(np.uint32))  # one position: its weight is one and its value is the same 16 bits
        _near([[_far(got[k, s], want[k, s]) for s in range(len(lengths))] for k in range(10)])
        plain.free()
    paged.free()
    d.free()


def test_a_prompt_of_several_passes():
    spec = _spec(q.ARCH_LLAMA, 192, ctx=2048)
    prompts = _prompts([1300, 5], spec["vocab"])
    d = q.Decoder(spec)
    want, plain = _run(d, prompts, [[1, 2]])
    got, paged = _run(d, prompts, [[1, 2]], pages=40, page_tokens=64)
    for k in range(2):
        for s in range(2):
            assert _far(got[k, s], want[k, s]) < FAR
    k, v = paged.read_cache(1, 0)
    assert k.shape == (1301, 128) and np.isfinite(k).all() and (np.abs(v).max(axis=1) > 0).all()


@pytest.mark.parametrize("cache", ["f16", "bf16", "q8"])
def test_the_cache_holds_what_was_computed(cache):
    """Keys and values of the first layer depend on the token and the position alone: the value is the same everywhere, the key at p is the key at 0 turned by p's angles."""
    spec = _spec(q.ARCH_LLAMA, 193)
    d = q.Decoder(spec)
    b = q.Batch(d, 3, pages=60, page_tokens=16, cache=cache)
    token, n = 7, 40
    b.prefill(0, np.full(n, token, np.uint32))
    b.prefill(1, [token])
    for _ in range(n - 1):
        b.step(sequences=[1], tokens=[token])
    k, v = b.read_cache(0, 0)
    k1, v1 = b.read_cache(0, 1)
    assert k.shape == v.shape == (n, 128) and b.read_cache(0, 2)[0].shape == (0, 128)
    assert np.array_equal(k, k1) and np.array_equal(v, v1)  # a prompt's pass and single steps
    assert np.array_equal(v, np.tile(v[:1], (n, 1)))
    # pairs (2 i, 2 i + 1) turned by p theta^(-2 i / 64); angles are F32 (off by n half steps at most), three roundings in F32; both keys are rounded to the cache's type: half a step of the
    # larger of a pair, Q8: half of 1 / 127 of the head's maximum, turned by at most the square root of two
    x = k.reshape(n, 2, 32, 2).astype(np.float64)
    angle = np.arange(n)[:, None] * 500000.0 ** (-2.0 * np.arange(32) / 64)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    want = np.stack([x[0, :, :, 0] * c - x[0, :, :, 1] * s, x[0, :, :, 0] * s + x[0, :, :, 1] * c], -1)
    size = np.abs(x[0]).sum(-1)[None, :, :, None]  # at least the length of a pair
    rounding = HALF[cache] * size if cache != "q8" else np.broadcast_to(np.abs(x).max(axis=(2, 3), keepdims=True) * (1 + 2.0 ** -7) / 254, x.shape)
    assert (np.abs(x - want) <= rounding * (1 + 2 ** 0.5) + size * (n + 4) * 2.0 ** -23).all()
    assert all(np.isfinite(x).all() for x in b.read_cache(1, 0))
    b.free()
    d.free()


@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_which_pages_a_sequence_has_makes_no_difference(cache):
    spec = _spec(q.ARCH_LLAMA, 194)
    lengths = [33, 100, 64]
    prompts = _prompts(lengths, spec["vocab"])
    fed = [synth.prompt_tokens(90 + k, 3, spec["vocab"]) for k in range(20)]
    d = q.Decoder(spec)
    want, fresh = _run(d, prompts, fed, pages=24, page_tokens=16, cache=cache)
    b = q.Batch(d, 3, pages=24, page_tokens=16, cache=cache)
    b.prefill(1, prompts[0][:20])  # pages come and go until those of a sequence lie anywhere, with other rows in them
    b.prefill(2, np.tile(prompts[1], 2))
    b.prefill(0, prompts[2])
    b.rewind(2, 17)
    b.prefill(1, prompts[2])
    b.rewind(0, 0)
    b.prefill(0, prompts[1])
    for s in (1, 0, 2):
        b.rewind(s, 0)
    assert b.pages() == (24, 24, 16)
    got = [None] * 3
    for s in (2, 0, 1):
        got[s] = b.prefill(s, prompts[s])[0]
    assert np.array_equal(np.stack(got).view(np.uint32), want[0].view(np.uint32))
    for k, tokens in enumerate(fed):
        assert np.array_equal(b.step(tokens=tokens, want_logits=True)[1].view(np.uint32), want[k + 1].view(np.uint32)), k
    assert b.pages()[1] == 24 - sum(-(-(n + 20) // 16) for n in lengths)
    # back to the prompts' ends and on again
    for s, n in enumerate(lengths):
        b.rewind(s, n)
    assert np.array_equal(b.step(tokens=fed[0], want_logits=True)[1].view(np.uint32), want[1].view(np.uint32))


def test_steps_of_some_sequences():
    spec = _spec(q.ARCH_LLAMA, 195)
    prompts = _prompts([20, 31, 7, 64], spec["vocab"])
    d = q.Decoder(spec)
    plain, paged = q.Batch(d, 4), q.Batch(d, 4, pages=32, page_tokens=16)
    for b in (plain, paged):
        for s in (2, 0, 3, 1):
            b.prefill(s, prompts[s][:5])
            b.prefill(s, prompts[s][5:])
    for k in range(5):
        x, y = (b.step(sequences=[3, 1], tokens=[k + 1, k + 2], want_logits=True)[1] for b in (plain, paged))
        assert _far(y[0], x[0]) < FAR and _far(y[1], x[1]) < FAR
    x, y = (b.step(tokens=[9, 8, 7, 6], want_logits=True)[1] for b in (plain, paged))
    assert all(_far(y[s], x[s]) < FAR for s in range(4))
    toks, lg = paged.step(want_logits=True)  # each its own last choice
    assert np.array_equal(toks, lg.argmax(1))
    assert list(paged.positions()) == [22, 38, 9, 71]


def test_pages_run_out():
    spec = _spec(q.ARCH_LLAMA, 196, ctx=256)
    d = q.Decoder(spec)
    b = q.Batch(d, 3, pages=5, page_tokens=16)
    b.prefill(0, np.arange(32) % 300)
    b.prefill(1, np.arange(31) % 300)
    with pytest.raises(q.QuintritError) as e:
        b.prefill(2, np.arange(17) % 300)
    assert e.value.code == 11 and "2 more pages, 1 are free" in str(e.value)
    assert list(b.positions()) == [32, 31, 0] and b.pages()[1] == 1
    b.prefill(2, np.arange(16) % 300)
    with pytest.raises(q.QuintritError) as e:
        b.step(tokens=[1, 2, 3])
    assert e.value.code == 11 and "2 more pages, 0 are free" in str(e.value)
    assert list(b.positions()) == [32, 31, 16]
    toks, _ = b.step(sequences=[1], tokens=[2])  # has room in its last page
    b.rewind(0, 16)
    assert b.pages()[1] == 1
    b.step(sequences=[2], tokens=[3])
    assert list(b.positions()) == [16, 32, 17] and b.pages()[1] == 0
    with pytest.raises(q.QuintritError) as e:
        b.prefill(0, np.zeros(300, np.uint32))
    assert e.value.code == 11 and "context window" in str(e.value)


def test_refusals():
    spec = _spec(q.ARCH_LLAMA, 197, ctx=256)
    d = q.Decoder(spec)
    for kw, code in ((dict(pages=0), 3), (dict(pages=4, page_tokens=48), 3), (dict(pages=4, page_tokens=8), 3)):
        with pytest.raises(q.QuintritError) as e:
            q.Batch(d, 2, **kw)
        assert e.value.code == code and "must be" in str(e.value)
    with pytest.raises(ValueError):
        q.Batch(d, 2, pages=4, cache="f32")
    for n in (0, 257):
        with pytest.raises(q.QuintritError) as e:
            q.Batch(d, n, pages=4)
        assert e.value.code == 2
    plain = q.Batch(d, 2)
    with pytest.raises(q.QuintritError) as e:
        plain.pages()
    assert e.value.code == 6
    with pytest.raises(q.QuintritError) as e:
        plain.read_cache(0, 0)
    assert e.value.code == 6
    b = q.Batch(d, 2, pages=4)
    b.prefill(0, [1, 2, 3])
    for layer, s in ((2, 0), (0, 2)):
        with pytest.raises(q.QuintritError) as e:
            b.read_cache(layer, s)
        assert e.value.code == 2
    few = np.zeros(128 * 3 - 1, np.float32)
    f32p = few.ctypes.data_as(q.api._f32p)
    lib = q.load_library()
    assert lib.quintrit_b200_batch_read_cache(b._h, 0, 0, f32p, few.size, None, 0) == 4
    assert lib.quintrit_b200_batch_read_cache(b._h, 0, 0, None, 0, None, 0) == 1
    odd = q.Decoder(_spec(q.ARCH_LLAMA, 198, ctx=256, heads=(8, 2, 32)))
    with pytest.raises(q.QuintritError) as e:
        q.Batch(odd, 2, pages=4)
    assert e.value.code == 6
    b.free()
    with pytest.raises(q.QuintritError) as e:
        b.pages()
    assert e.value.code == 14


@pytest.mark.parametrize("heads", [(191, 1, 64), (96, 2, 128), (48, 1, 256), (128, 1, 128)])
def test_long_query_rows(heads):
    """Rows of 12224, 12288 and 16384 values: their codes are made in more shared memory than a kernel has without asking."""
    spec = _spec(q.ARCH_BITNET, 199, ctx=256, heads=heads)
    prompts = _prompts([1, 30], spec["vocab"])
    d = q.Decoder(spec)
    want, plain = _run(d, prompts, [[1, 2], [3, 4]])
    got, paged = _run(d, prompts, [[1, 2], [3, 4]], pages=8, page_tokens=16)
    # (Not bit for bit at one position either: more than 16 heads to a key head take the kernel for many rows, whose exponents are fma(score, scale, -m) with m rounded to 32 bits, so that a sum of one
    # weight is one but for |z| 2^-24, and a code that lies at a half may go the other way, in all heads of the key head at once.)
    _near([[_far(got[k, s], want[k, s]) for s in range(2)] for k in range(3)])
    for x in (plain, paged, d):
        x.free()


class _ByOperators:
    """A decoder's passes over a paged cache put together from the operators, called one by one through ``PagedCache``, and the integer products and 32-bit steps of the model's definition (the
    oracle's) around them: what a batch's passes give, bit for bit."""

    def __init__(self, spec, sequences, cache, page_tokens):
        import torch

        self.t, self.spec, self.kind = torch, spec, cache
        H, I, qh, kvh, hd = (spec[k] for k in ("hidden", "inter", "q_heads", "kv_heads", "head_dim"))
        shapes = [(qh * hd, H), (kvh * hd, H), (kvh * hd, H), (H, qh * hd), (I, H), (I, H), (H, I)]
        self.weights = [oracle.unpack_planar(w, *shapes[i % 7]).astype(np.float64).T for i, w in enumerate(spec["weights"])]
        per = -(-spec["ctx"] // page_tokens)
        self.cache = q.PagedCache(spec["layers"], sequences * per, page_tokens, kvh, hd, cache)
        self.table = torch.randperm(sequences * per, generator=torch.Generator().manual_seed(1)).to(torch.int32).reshape(sequences, per).cuda()
        self.angles = torch.tensor(np.stack([oracle.rope_cache(p, spec["rope_dims"], spec["rope_theta"]) for p in range(spec["ctx"])])).cuda()
        self.embed = np.asarray(spec["embed"], np.uint16).view(np.float16).reshape(-1, H).astype(np.float32)
        self.head = np.asarray(spec["embed"] if spec["lm_head"] is None else spec["lm_head"], np.uint16).reshape(-1, H)

    def rows(self, sequences, new, lengths, longest):
        i32 = lambda v: self.t.tensor(v, dtype=self.t.int32, device="cuda")
        return q.PagedRows(i32([0] + list(np.cumsum(new))), i32(lengths), self.table[i32(sequences).long()], int(sum(new)), max(new), longest)

    def project(self, rows, l, *which):
        """Rows of 32-bit values through projections: [rows][outputs] each."""
        out = [[] for _ in which]
        for x in rows:
            codes, s = oracle.quantize_int8(x)
            for o, k in zip(out, which):
                o.append(oracle.rescale((codes.astype(np.float64) @ self.weights[l * 7 + k]).astype(np.int32), float(self.spec["scales"][l * 7 + k]), float(s)))
        return [np.stack(o) for o in out]

    def forward(self, tokens, rows, wanted):
        """Logits of the packed tokens `wanted`."""
        spec, torch = self.spec, self.t
        qh, kvh, hd = (spec[k] for k in ("q_heads", "kv_heads", "head_dim"))
        norm = lambda x, w: x if w is None else np.stack([oracle.rms_norm(r, w, spec["eps"]) for r in x])
        x = self.embed[np.asarray(tokens, np.int64)]
        n = len(x)
        for l in range(spec["layers"]):
            w = spec["norms"][l * 4:l * 4 + 4]
            heads = [torch.tensor(y).reshape(n, -1, hd).cuda() for y in self.project(norm(x, w[0]), l, 0, 1, 2)]
            q_out = torch.empty(n, qh, hd, dtype={"f16": torch.float16, "bf16": torch.bfloat16, "q8": torch.float32}[self.kind], device="cuda")
            self.cache.append(l, rows, *heads, q_out=q_out, cos_sin=self.angles, neox=spec["arch"] != q.ARCH_LLAMA)
            o = self.cache.attend(l, rows, q_out, out=torch.empty(n, qh, hd, device="cuda"), scale=float(np.float32(1) / np.sqrt(np.float32(hd))))
            x = x + self.project(norm(o.reshape(n, -1).cpu().numpy(), w[2]), l, 3)[0]
            g, u = self.project(norm(x, w[1]), l, 4, 5)
            y = np.stack([(oracle.relu2_mul if spec["arch"] == q.ARCH_BITNET else oracle.swiglu)(a, b) for a, b in zip(g, u)])
            x = x + self.project(norm(y, w[3]), l, 6)[0]
        self.cache.status()
        last = [oracle.f32_to_f16_bits(r) for r in norm(x[wanted], spec["out_norm"])]
        return np.stack([[oracle.vec_dot_f16(row, r) for row in self.head] for r in last])


@pytest.mark.parametrize("cache,page_tokens", [("f16", 16), ("bf16", 64), ("q8", 32)])
@pytest.mark.parametrize("arch,heads", [(q.ARCH_LLAMA, (4, 2, 64)), (q.ARCH_BITNET, (4, 1, 64)), (q.ARCH_LLAMA, (6, 2, 128)), (q.ARCH_BITNET, (3, 1, 256)), (q.ARCH_LLAMA, (40, 1, 64))])
def test_passes_are_the_operators_one_by_one(arch, heads, cache, page_tokens):
    spec = _spec(arch, 200, ctx=512, heads=heads, tied=arch == q.ARCH_BITNET)
    lengths = [1, 3, 150, 41, 333]
    prompts = _prompts(lengths, spec["vocab"])
    fed = [synth.prompt_tokens(70 + k, len(lengths), spec["vocab"]) for k in range(3)]
    d = q.Decoder(spec)
    got, b = _run(d, prompts, fed, pages=sum(-(-(n + 3) // page_tokens) for n in lengths), page_tokens=page_tokens, cache=cache)
    one = _ByOperators(spec, len(lengths), cache, page_tokens)
    want = [np.concatenate([one.forward(p, one.rows([s], [len(p)], [len(p)], len(p)), [len(p) - 1]) for s, p in enumerate(prompts)])]
    every = sorted(range(len(lengths)), key=lambda s: -lengths[s])  # a step takes its longest sequences first; where their tiles are cut into ranges goes by that
    for k, tokens in enumerate(fed):
        out = one.forward([tokens[s] for s in every], one.rows(every, [1] * len(every), [lengths[s] + k + 1 for s in every], spec["ctx"]), list(range(len(every))))
        want.append(out[np.argsort(every)])
    want = np.stack(want).astype(np.float32)
    for s, n in enumerate(lengths):
        whole = one.rows([s], [n + 3], [n + 3], n + 3)
        for l in range(spec["layers"]):
            for x, y in zip(b.read_cache(l, s), one.cache.read(l, whole, dtype=one.t.float32)):
                assert np.array_equal(x, y.reshape(n + 3, -1).cpu().numpy()), (s, l)
    assert np.array_equal(got.view(np.uint32), want.view(np.uint32))
    for x in (b, d):
        x.free()
