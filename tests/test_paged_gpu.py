"""The paged cache on a B200 against the same operators in 64 bits: rows written and read back, attention of single tokens and chunks."""
import itertools

import pytest

torch = pytest.importorskip("torch")
import quintrit_b200 as q
from tests.paged_reference import EPS, attention, attention_bound, make_rows, places, whole, written

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def randn(*shape, seed, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def angles(positions, dims):
    f = 10000.0 ** (-torch.arange(0, dims, 2, device="cuda", dtype=torch.float64) / dims)
    a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * f
    return torch.stack([a.cos(), a.sin()], -1).reshape(positions, dims).float()


def filled(cache_type, kvh, hd, new, lengths, page, seed=1, **more):
    """A cache whose sequences hold random rows, with its rows, what it holds (as stored, 32 bits) and the sequences' first dense rows."""
    rows, pages, _ = make_rows(q, new, lengths, page, seed=seed, **more)
    cache = q.PagedCache(1, pages, page, kvh, hd, cache_type)
    every = whole(q, rows)
    cache.append(0, every, None, randn(every.tokens, kvh, hd, seed=seed), randn(every.tokens, kvh, hd, seed=seed + 1) * 1.5)
    k, v = cache.read(0, every, dtype=torch.float32)
    return cache, rows, k, v, every.starts.tolist()


# ---- rows in and out -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("cache_type,hd,page,in_type", [("f16", 64, 16, "f32"), ("f16", 128, 64, "f16"), ("bf16", 256, 32, "bf16"), ("q8", 64, 256, "f16"), ("q8", 128, 16, "bf16"),
                                                         ("q8", 256, 64, "f32"), ("bf16", 64, 128, "f32")])
@pytest.mark.parametrize("norm,rope,neox", [(False, 0, False), (True, 64, False), (True, 32, True), (False, 64, True), (True, 22, True), (False, 22, False), (False, 2, True), (False, 8, True)])
def test_append_and_read(cache_type, hd, page, in_type, norm, rope, neox):
    new, lengths, qh, kvh = [1, 5, 0, 40, page + 1], [1, 70, 33, 40, 3 * page], 6, 3  # a first token, the middle of a page, no token, a whole sequence, over a page's end
    rows, pages, _ = make_rows(q, new, lengths, page, seed=3)
    cache = q.PagedCache(2, pages, page, kvh, hd, cache_type)
    T, dt = rows.tokens, DT[in_type]
    x = randn(T, qh + 2 * kvh, hd, seed=7, dtype=dt) * 3
    qs, ks, vs = x[:, :qh], x[:, qh:qh + kvh], x[:, qh + kvh:]
    wq, wk = (1 + 0.3 * randn(hd, seed=9), 1 + 0.3 * randn(hd, seed=10)) if norm else (None, None)
    cs = angles(max(lengths), rope * hd // 64 if rope > 22 else rope) if rope else None
    out = cache.append(1, rows, qs, ks, vs, q_norm=wq, k_norm=wk, eps=1e-5, cos_sin=cs, neox=neox)
    pos = torch.tensor([p for _, p in places(rows)], device="cuda")
    # 32-bit arithmetic: a sum of hd squares, a root, a division, four products and a sum: under (hd / 2 + 16) half steps of the pair's magnitude
    for got, want in ((out, written(qs, wq, 1e-5, cs, neox, pos)),):
        assert got.dtype is dt
        bound = want.abs() * EPS[dt] + want.abs().amax(-1, keepdim=True) * (hd / 2 + 16) * 2.0 ** -24
        assert bool(((got.double() - want).abs() <= bound).all())
    k, v = cache.read(1, rows, dtype=torch.float32)
    for got, want in ((k, written(ks, wk, 1e-5, cs, neox, pos)), (v, vs.double())):
        arith = want.abs().amax(-1, keepdim=True) * (hd / 2 + 16) * 2.0 ** -24
        if cache_type == "q8":  # half a step of the code, the scale's own rounding (127 half steps of 2^-24), the product's
            bound = want.abs().amax(-1, keepdim=True) / 127 * 0.5 * (1 + 2.0 ** -10) + arith + want.abs() * 2.0 ** -22
        else:
            bound = want.abs() * EPS[DT[cache_type]] + arith
        assert bool(((got.double() - want).abs() <= bound).all())
    other = cache.read(0, rows, dtype=torch.float32)  # the other layer is as it was
    assert float(other[0].abs().max()) == 0.0 and float(other[1].abs().max()) == 0.0
    cache.status()


@pytest.mark.parametrize("cache_type,out_type", list(itertools.product(["f16", "bf16", "q8"], ["f16", "bf16", "f32"])))
def test_read_rounds_once(cache_type, out_type):
    rows, pages, _ = make_rows(q, [37, 20], [37, 20], 16)
    cache = q.PagedCache(1, pages, 16, 2, 64, cache_type)
    k, v = randn(57, 2, 64, seed=1), randn(57, 2, 64, seed=2)
    cache.append(0, rows, None, k, v)
    k32, v32 = cache.read(0, rows, dtype=torch.float32)
    got = cache.read(0, rows, dtype=DT[out_type])
    assert torch.equal(got[0], k32.to(DT[out_type])) and torch.equal(got[1], v32.to(DT[out_type]))
    if cache_type != "q8":
        assert torch.equal(k32, k.to(DT[cache_type]).float())
    else:  # codes times the row's scale: whole multiples, up to 127
        d = k.abs().amax(-1, keepdim=True) / 127
        assert float(((k32 / d) - (k32 / d).round()).abs().max()) < 1e-4 and float((k32 / d).abs().max()) < 127.01
    only = torch.zeros_like(got[0])
    cache.read(0, rows, k_out=only)
    assert torch.equal(only, got[0])


@pytest.mark.parametrize("cache_type", ["f16", "bf16", "q8"])
def test_values_that_do_not_fit_are_saturated_and_reported(cache_type):
    rows, pages, _ = make_rows(q, [3], [3], 16)
    cache = q.PagedCache(1, pages, 16, 1, 64, cache_type)
    k, v = randn(3, 1, 64, seed=1), randn(3, 1, 64, seed=2)
    v[1, 0, 5], v[1, 0, 6], v[2, 0, 0] = float("inf"), float("nan"), float("-inf")
    cache.append(0, rows, None, k, v)
    _, got = cache.read(0, rows, dtype=torch.float32)
    assert bool(torch.isfinite(got).all())
    assert float(got[1, 0, 5]) > 6e4 and float(got[1, 0, 6]) == 0.0 and float(got[2, 0, 0]) < -6e4
    with pytest.raises(q.QuintritError) as e:
        cache.status()
    assert e.value.code == 5
    cache.status()  # reported once
    # rows of zeros and of the smallest numbers
    cache.append(0, rows, None, torch.zeros_like(k), torch.full_like(v, 1e-40))
    _, got = cache.read(0, rows, dtype=torch.float32)
    assert float(got.abs().max()) <= 1e-38
    cache.status()


def test_queries_in_place_and_rows_behind_the_last_sequence():
    rows, pages, _ = make_rows(q, [4, 3], [9, 3], 16)
    rows = q.PagedRows(rows.starts, rows.lengths, rows.table, 12, 4, 9)  # five rows more than the sequences have
    cache = q.PagedCache(1, pages, 16, 2, 64, "f16")
    x = randn(12, 8, 64, seed=4, dtype=torch.float16)
    qs, k, v = x[:, :4].clone(), x[:, 4:6], x[:, 6:]
    cs = angles(9, 64)
    apart = cache.append(0, rows, qs, k, v, cos_sin=cs, q_out=torch.full_like(qs, 7))
    same = cache.append(0, rows, qs, k, v, cos_sin=cs, q_out=qs)
    assert same is qs and torch.equal(same[:7], apart[:7])
    assert torch.equal(apart[7:], torch.full_like(apart[7:], 7)) and torch.equal(same[7:], x[7:, :4])
    out = cache.attend(0, rows, qs, out=torch.full_like(qs, 5))
    assert torch.equal(out[7:], torch.full_like(out[7:], 5)) and not bool((out[:7] == 5).all())
    ko, vo = torch.full((12, 2, 64), 3.0, device="cuda", dtype=torch.float16), torch.full((12, 2, 64), 3.0, device="cuda", dtype=torch.float16)
    cache.read(0, rows, k_out=ko, v_out=vo)
    assert torch.equal(vo[:7], v[:7]) and bool((vo[7:] == 3).all()) and bool((ko[7:] == 3).all())


# ---- attention -------------------------------------------------------------------------------------------------------------------
def check_attention(cache_type, hd, kvh, group, new, lengths, page, q_type=None, out_type=None, cap=0.0, window=0, scale=None, seed=1, **more):
    cache, rows, k, v, first = filled(cache_type, kvh, hd, new, lengths, page, seed=seed, **more)
    qt = DT[q_type] if q_type else torch.float16 if cache_type == "q8" else DT[cache_type]
    ot = DT[out_type] if out_type else qt
    qs = randn(rows.tokens, kvh * group, hd, seed=seed + 5, dtype=qt)
    scale = hd ** -0.5 if scale is None else scale
    out = cache.attend(0, rows, qs, out=torch.full(qs.shape, 9.0, dtype=ot, device="cuda"), scale=scale, cap=cap, window=window)
    want, mass, size = attention(qs, rows, k, v, first, scale, cap, window)
    wt = torch.bfloat16 if cache_type == "bf16" else torch.float16
    bound = attention_bound(want, mass, size, max(lengths), hd, wt, ot, v, cache_type == "q8", qt, cap)
    off = (out.double() - want).abs()
    assert bool((off <= bound).all()), f"off by {float((off / bound).max()):.2f} bounds"
    cache.status()
    return cache, rows, qs, out


TYPES = ["f16", "bf16", "q8"]


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("hd,kvh,group,page", [(64, 2, 4, 16), (128, 5, 4, 64), (256, 4, 3, 32), (128, 1, 1, 256)])
def test_single_tokens(cache_type, hd, kvh, group, page):
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 200, 333]
    check_attention(cache_type, hd, kvh, group, [1] * len(lengths), lengths, page)


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("hd,group", [(64, 8), (128, 4), (256, 3), (128, 16), (64, 1)])
def test_chunks_of_a_few_tokens(cache_type, hd, group):
    check_attention(cache_type, hd, 2, group, [2, 5, 9, 1, 0, 7], [2, 70, 130, 257, 40, 7], 32)


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("hd,kvh,group", [(64, 2, 4), (128, 1, 5), (256, 1, 3)])
def test_chunks_of_many_tokens(cache_type, hd, kvh, group):
    check_attention(cache_type, hd, kvh, group, [131, 64, 33], [131, 300, 97], 64)


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("new", [1, 6, 150])
@pytest.mark.parametrize("cap,window", [(20.0, 0), (0.0, 1), (0.0, 37), (5.0, 64), (0.0, 1000)])
def test_capped_scores_and_windows(cache_type, new, cap, window):
    check_attention(cache_type, 128, 2, 4, [new, new, new], [new, 400, 257 + new], 16, cap=cap, window=window, scale=0.3)


@pytest.mark.parametrize("q_type,out_type", list(itertools.product(["f16", "bf16", "f32"], ["f16", "bf16", "f32"])))
@pytest.mark.parametrize("new", [1, 70])
def test_query_and_output_types_over_codes(q_type, out_type, new):
    check_attention("q8", 64, 2, 4, [new, 3], [90, 130], 32, q_type=q_type, out_type=out_type)


@pytest.mark.parametrize("cache_type", ["f16", "bf16"])
def test_output_types(cache_type):
    check_attention(cache_type, 64, 2, 4, [1, 3], [90, 130], 32, out_type="f32")


@pytest.mark.parametrize("cache_type", TYPES)
def test_long_sequences_in_ranges(cache_type):
    """One sequence cut into ranges for many blocks, beside short ones; announced too short, it is still served whole."""
    a = check_attention(cache_type, 128, 2, 4, [1, 1, 1], [9001, 100, 1], 64)[3]
    b = check_attention(cache_type, 128, 2, 4, [1, 1, 1], [9001, 100, 1], 64, max_length=200)[3]
    assert float((a.float() - b.float()).abs().max()) < 0.01
    check_attention(cache_type, 64, 1, 2, [3], [20000], 128, window=5000)


def test_scores_far_apart():
    """Scores of hundreds: the maximum grows many times, most weights vanish."""
    for cache_type in TYPES:
        check_attention(cache_type, 128, 2, 4, [1, 20], [500, 300], 64, scale=8.0)


def test_rows_of_zeros_and_of_very_different_sizes():
    for cache_type in ("f16", "q8"):
        rows, pages, _ = make_rows(q, [2, 1], [200, 70], 16, seed=5)
        cache = q.PagedCache(1, pages, 16, 2, 64, cache_type)
        every = whole(q, rows)
        k, v = randn(270, 2, 64, seed=1), randn(270, 2, 64, seed=2)
        v *= torch.exp(4 * randn(270, 2, 1, seed=3)) * 1e-2
        v[10:20], k[30:40], v[200:260] = 0, 0, 0
        if cache_type == "f16":
            v = v.half().float().clamp(-60000, 60000)
        cache.append(0, every, None, k, v)
        k, v = cache.read(0, every, dtype=torch.float32)
        qs = randn(3, 8, 64, seed=8, dtype=torch.float16)
        qs[1] = 0
        out = cache.attend(0, rows, qs, out=torch.empty(3, 8, 64, dtype=torch.float32, device="cuda"))
        want, mass, size = attention(qs, rows, k, v, every.starts.tolist(), 0.125)
        bound = attention_bound(want, mass, size, 200, 64, torch.float16, torch.float32, v, True)
        assert bool(((out.double() - want).abs() <= bound).all())


def test_what_a_mask_hides_has_no_effect():
    """Infinities and NaN written at later positions, or left in a page by a conversation that ended, do not reach a token that does not see them; a query that is no
    number spoils its own outputs only."""
    for cache_type in TYPES:
        rows, pages, _ = make_rows(q, [20], [60], 16, pages_extra=0, seed=2)
        cache = q.PagedCache(1, pages, 16, 1, 64, cache_type)
        bad = torch.full((64, 1, 64), float("nan"), device="cuda")
        bad[::2] = float("inf")
        full = q.PagedRows(torch.tensor([0, 64], dtype=torch.int32, device="cuda"), torch.tensor([64], dtype=torch.int32, device="cuda"), rows.table, 64, 64, 64)
        cache.append(0, full, None, bad, bad)
        every = whole(q, rows)
        k, v = randn(60, 1, 64, seed=1), randn(60, 1, 64, seed=2)
        cache.append(0, every, None, k, v)
        qs = randn(20, 4, 64, seed=3, dtype=torch.bfloat16 if cache_type == "bf16" else torch.float16)
        clean = cache.attend(0, rows, qs).clone()
        assert bool(torch.isfinite(clean).all())
        k[50], v[50] = float("nan"), float("inf")  # position 50 is new token 10
        cache.append(0, every, None, k, v)
        out = cache.attend(0, rows, qs)
        assert torch.equal(out[:10], clean[:10])
        cache.append(0, every, None, randn(60, 1, 64, seed=1), randn(60, 1, 64, seed=2))
        qs[3, 2, 7] = float("nan")
        out = cache.attend(0, rows, qs)
        assert bool(torch.isnan(out[3, 2]).all())
        keep = torch.ones(20, 4, dtype=torch.bool, device="cuda")
        keep[3, 2] = False
        assert torch.equal(out[keep], clean[keep])


def test_bad_tables_and_lengths_are_skipped_and_reported():
    rows, pages, table = make_rows(q, [2, 2, 2], [40, 40, 40], 16, seed=2)
    cache = q.PagedCache(1, pages, 16, 2, 64, "f16")
    every = whole(q, rows)
    x = randn(120, 2, 64, seed=1, dtype=torch.float16)
    cache.append(0, every, None, x, x)
    qs = randn(6, 4, 64, seed=3, dtype=torch.float16)
    clean = cache.attend(0, rows, qs).clone()
    cache.status()

    def raises(rows):
        out = cache.attend(0, rows, qs, out=torch.full_like(qs, 4))
        cache.append(0, rows, None, x[:6], x[:6])
        cache.read(0, rows)
        with pytest.raises(q.QuintritError) as e:
            cache.status()
        assert e.value.code == 5
        cache.append(0, every, None, x, x)
        cache.status()
        return out

    bad = rows.table.clone()
    bad[1, 2], bad[1, 0] = pages, -1
    out = raises(q.PagedRows(rows.starts, rows.lengths, bad, 6, 2, 40))
    assert torch.equal(out[0:2], clean[0:2]) and torch.equal(out[4:6], clean[4:6])
    for lengths in ([40, 49, 40], [40, -3, 40], [40, 1 << 30, 40]):  # the table has room for 48
        out = raises(q.PagedRows(rows.starts, torch.tensor(lengths, dtype=torch.int32, device="cuda"), rows.table, 6, 2, 40))
        assert torch.equal(out[0:2], clean[0:2]) and torch.equal(out[4:6], clean[4:6]) and bool((out[2:4] == 4).all())
    for starts in ([0, 2, 1, 6], [-4, 2, 4, 6], [0, 2, 4, 9], [0, 2, 1 << 30, 6]):
        raises(q.PagedRows(torch.tensor(starts, dtype=torch.int32, device="cuda"), rows.lengths, rows.table, 6, 2, 40))
    # more new tokens than positions: the first ones see nothing
    out = cache.attend(0, q.PagedRows(rows.starts, torch.tensor([40, 1, 0], dtype=torch.int32, device="cuda"), rows.table, 6, 2, 40), qs, out=torch.full_like(qs, 4))
    assert torch.equal(out[0:2], clean[0:2]) and float(out[2].abs().max()) == 0.0 and float(out[3].abs().max()) > 0.0 and float(out[4:6].abs().max()) == 0.0
    # a chunk longer than announced
    with pytest.raises(q.QuintritError):
        cache.attend(0, q.PagedRows(rows.starts, rows.lengths, rows.table, 6, 1, 40), qs)
        cache.status()
    torch.cuda.synchronize()


def test_strided_queries_and_outputs():
    for new in (1, 5, 90):
        cache, rows, k, v, first = filled("f16", 2, 64, [new, new], [100, 150], 16)
        T = rows.tokens
        wide = randn(T, 8 + 3, 2 * 64, seed=3, dtype=torch.float16)
        qs = wide[:, 1:9, 64:]
        out = torch.full((8, T, 64), 2.0, dtype=torch.float16, device="cuda").transpose(0, 1)  # heads apart
        cache.attend(0, rows, qs, out=out)
        want = cache.attend(0, rows, qs.contiguous())
        assert torch.equal(out, want)


def test_captured_calls_follow_their_tensors():
    """A step (append, attend) of two graphs that share nothing but the cache's weights: replayed with other lengths, tables and inputs."""
    lengths = [30, 64, 7]
    rows, pages, _ = make_rows(q, [1, 1, 1], [90, 90, 90], 16, seed=4, max_length=90)
    rows.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
    cache = q.PagedCache(1, pages, 16, 2, 128, "q8")
    cs = angles(96, 128)
    x = randn(3, 12, 128, seed=1, dtype=torch.float16)
    qo, out = torch.empty(3, 8, 128, dtype=torch.float16, device="cuda"), torch.empty(3, 8, 128, dtype=torch.float16, device="cuda")
    ws = cache.attend_workspace(rows, 8)

    def step():
        cache.append(0, rows, x[:, :8], x[:, 8:10], x[:, 10:], q_out=qo, cos_sin=cs, neox=True)
        cache.attend(0, rows, qo, out=out, workspace=ws)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    every = None
    for i in range(4):
        x.copy_(randn(3, 12, 128, seed=10 + i, dtype=torch.float16))
        rows.lengths += 1
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        every = whole(q, rows)
        k, v = cache.read(0, every, dtype=torch.float32)
        want, mass, size = attention(qo, rows, k, v, every.starts.tolist(), 128 ** -0.5)
        assert bool(((got.double() - want).abs() <= attention_bound(want, mass, size, 96, 128, torch.float16, torch.float16, v, True)).all())
        step()
        assert torch.equal(out, got)  # the same calls, not captured
    cache.status()


def test_two_streams_at_once():
    cache, rows, k, v, first = filled("f16", 2, 128, [1] * 4, [3000, 2000, 100, 5], 64)
    qs = [randn(4, 8, 128, seed=i, dtype=torch.float16) for i in range(6)]
    want = [cache.attend(0, rows, x).clone() for x in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for i, x in enumerate(qs):
        with torch.cuda.stream(streams[i % 3]):
            got.append(cache.attend(0, rows, x))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_the_same_call_gives_the_same_bits():
    for cache_type, new in itertools.product(TYPES, (1, 4, 200)):
        cache, rows, _, _, _ = filled(cache_type, 2, 128, [new, new], [5000, 700], 32)
        qs = randn(rows.tokens, 8, 128, seed=1, dtype=torch.bfloat16 if cache_type == "bf16" else torch.float16)
        a = cache.attend(0, rows, qs).clone()
        for _ in range(3):
            assert torch.equal(cache.attend(0, rows, qs), a)


def test_no_tokens():
    rows, pages, _ = make_rows(q, [1], [40], 16)
    none = q.PagedRows(rows.starts * 0, rows.lengths, rows.table, 0, 0, 40)
    cache = q.PagedCache(1, pages, 16, 2, 64, "q8")
    e = torch.empty(0, 2, 64, dtype=torch.float16, device="cuda")
    assert cache.append(0, none, e, e, e).shape == (0, 2, 64)
    assert cache.attend(0, none, e).shape == (0, 2, 64)
    assert cache.read(0, none)[0].shape == (0, 2, 64)


def test_python_refusals():
    cache, rows, _, _, _ = filled("f16", 2, 64, [2], [40], 16)
    good = randn(2, 4, 64, seed=1, dtype=torch.float16)
    for bad in (good[:1], good[:, :3], good[..., :32], good.double(), good.bfloat16(), randn(2, 4, 128, seed=1, dtype=torch.float16)[..., ::2]):
        with pytest.raises((ValueError, q.QuintritError)):
            cache.attend(0, rows, bad)
    with pytest.raises((ValueError, RuntimeError)):
        cache.attend(0, rows, good.cpu())
    with pytest.raises(q.QuintritError):
        cache.attend(1, rows, good)
    with pytest.raises(q.QuintritError):
        cache.attend(0, rows, torch.empty(2 * 4 * 64 + 1, dtype=torch.float16, device="cuda")[1:].view(2, 4, 64))  # not on a 16-byte boundary
    with pytest.raises(q.QuintritError):
        cache.attend(0, rows, good, cap=-1.0)
    with pytest.raises(q.QuintritError):
        cache.attend(0, rows, good, scale=float("nan"))
    with pytest.raises(ValueError):
        q.PagedCache(1, 4, 16, 1, 64, "q4")
    with pytest.raises(ValueError):
        q.PagedRows(rows.starts.long(), rows.lengths, rows.table, 2, 2, 40)
    long_rows, pages, _ = make_rows(q, [1], [30000], 64)
    big = q.PagedCache(1, pages, 64, 1, 64, "f16")
    with pytest.raises(q.QuintritError) as e:
        big.attend(0, long_rows, randn(1, 4, 64, seed=1, dtype=torch.float16), workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    assert e.value.code == 4
    big.free()
    with pytest.raises(q.QuintritError) as e:
        big.status()
    assert e.value.code == 14


def test_windows_and_workspaces_that_are_refused():
    rows, pages, _ = make_rows(q, [1], [1000], 16)
    cache = q.PagedCache(1, pages, 16, 2, 64)
    x = torch.randn(1, 4, 64, device="cuda").half()
    for window in (-1, 2 ** 31):
        with pytest.raises(ValueError):
            cache.attend(0, rows, x, window=window)
    side = torch.cuda.Stream()
    assert cache.attend_workspace(rows, 4).nbytes > 0
    with pytest.raises(ValueError):  # torch would give the memory to others while the call runs
        cache.attend(0, rows, x, stream=side.cuda_stream)
    side.wait_stream(torch.cuda.current_stream())
    out = cache.attend(0, rows, x, stream=side.cuda_stream, workspace=cache.attend_workspace(rows, 4))
    torch.cuda.synchronize()
    assert torch.equal(out, torch.zeros_like(out))  # a new cache holds zeros
    cache.status()


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("hd,kvh,group", [(64, 2, 4), (128, 1, 3), (256, 1, 4)])
def test_many_sequences_with_uneven_chunks(cache_type, hd, kvh, group):
    """More sequences than a warp looks through at once, those with many new tokens among others with a few, one or none."""
    new = [[1, 40, 0, 2, 130, 1, 5, 70, 33, 1, 3][i % 11] for i in range(70)]
    check_attention(cache_type, hd, kvh, group, new, [n + (i * 37) % 400 for i, n in enumerate(new)], 32, max_new=130)


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("sequences", [200, 300])
def test_single_tokens_of_very_many_sequences(cache_type, sequences):
    """As many as share their tiles out, and more."""
    check_attention(cache_type, 64, 2, 4, [1] * sequences, [1 + (i * 113) % 700 for i in range(sequences)], 16)


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("new,group", [(20, 4), (3, 1)])
def test_one_head_in_more_ranges_than_a_warp_has_lanes(cache_type, new, group):
    check_attention(cache_type, 64, 1, group, [new], [20011], 128)
