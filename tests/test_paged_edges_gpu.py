"""The paged cache on a B200 at its edges: sequences shorter than their chunks, segments that follow one another in a block, what tables and lengths may say, the ends of a type's range."""
import pytest

torch = pytest.importorskip("torch")
import quintrit_b200 as q
from tests.paged_reference import EPS, attention, attention_bound, make_rows, places, whole, written
from tests.test_paged_gpu import DT, TYPES, check_attention, filled, randn

pytestmark = pytest.mark.gpu
FEW_MANY = [1, 60]  # new tokens of four heads to a key head: the kernel for few rows, the one for many


def queries(cache_type, *shape, seed):
    return randn(*shape, seed=seed, dtype=torch.bfloat16 if cache_type == "bf16" else torch.float16)


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_chunks_longer_than_their_sequences(cache_type, hd):
    """Whole row blocks before position 0: zeros, whatever the block's warps have just written to shared memory; the last tokens see what there is."""
    new, lengths = [300] * 6, [0, 1, 20, 0, 299, 300]
    cache, _, _, _, _ = filled(cache_type, 2, hd, [1] * 6, [max(n, 1) for n in lengths], 16)
    rows, _, _ = make_rows(q, new, lengths, 16, seed=1)
    qs = queries(cache_type, rows.tokens, 8, hd, seed=6) * 50
    one = None
    for _ in range(50):
        out = cache.attend(0, rows, qs, out=torch.full_like(qs, 4))
        for s, (n, length) in enumerate(zip(new, lengths)):
            first = rows.starts[s] + n - length
            assert int(out[s * n:first].count_nonzero()) == 0 and bool((out[first:(s + 1) * n] != 0).any(-1).all())
        assert one is None or torch.equal(out, one)
        one = out
    cache.status()


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("hd,group,new", [(64, 4, 1), (128, 4, 1), (256, 3, 1), (128, 4, 5)])
def test_segments_that_follow_one_another_in_a_block(cache_type, hd, group, new):
    """Blocks that end one sequence and begin the next: what the warps have written where the first one's results met does not reach the second one's keys and values."""
    lengths = [new + 150 + (i * 211) % 1200 for i in range(120)]
    cache, rows, qs, out = check_attention(cache_type, hd, 4, group, [new] * 120, lengths, 16, q_type="bf16" if cache_type == "bf16" else "f16")
    for _ in range(100):
        assert torch.equal(cache.attend(0, rows, qs), out)
    cache.status()


def reported(cache):
    with pytest.raises(q.QuintritError) as e:
        cache.status()
    return e.value.code, str(e.value)


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("new", [1, 60])
def test_the_longest_sequences(cache_type, new):
    """2^31 - 2^16 positions, all in one page again and again: a window's worth of the last ones is served; longer ones are left out and reported."""
    most, window, P = 2 ** 31 - 2 ** 16, 100, 256
    cache = q.PagedCache(1, 1, P, 1, 64, cache_type)
    table = torch.zeros(1, 1 << 23, dtype=torch.int32, device="cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    k, v = randn(P, 1, 64, seed=1), randn(P, 1, 64, seed=2)
    cache.append(0, q.PagedRows(i32(0, P), i32(most), table, P, P, most), None, k, v)  # position p is row p % 256 (most is a multiple of it)
    k, v = cache.read(0, q.PagedRows(i32(0, P), i32(P), table, P, P, P), dtype=torch.float32)
    kl, vl = cache.read(0, q.PagedRows(i32(0, P), i32(most), table, P, P, most), dtype=torch.float32)
    assert torch.equal(k, kl) and torch.equal(v, vl)
    qs = queries(cache_type, new, 4, 64, seed=3)
    near = cache.attend(0, q.PagedRows(i32(0, new), i32(P), table, new, new, P), qs, window=window)
    far = cache.attend(0, q.PagedRows(i32(0, new), i32(most), table, new, new, most), qs, window=window)
    # the same rows, perhaps in other tiles: weights rounded to the cache's type, results too
    assert float((near.float() - far.float()).abs().max()) <= 4 * EPS[qs.dtype] * float(v.abs().max())
    cache.status()
    for length in (most + 1, 2 ** 31 - 1):
        rows = q.PagedRows(i32(0, new), i32(length), table, new, new, most)
        for kw in (dict(window=window), dict()):
            out = cache.attend(0, rows, qs, out=torch.full_like(qs, 4), **kw)
            assert bool((out == 4).all()) and reported(cache)[0] == 5
        ko, _ = cache.read(0, rows, k_out=torch.full((new, 1, 64), 4.0, device="cuda"))
        assert bool((ko == 4).all()) and reported(cache)[0] == 5


def test_a_table_that_is_a_part_of_another():
    """The rows of a table may lie further apart than they are long; what lies between is not the sequence's, and is not looked at."""
    rows, pages, _ = make_rows(q, [2, 2], [40, 48], 16, seed=2)
    cache = q.PagedCache(1, pages, 16, 2, 64)
    wide = torch.zeros(2, 9, dtype=torch.int32, device="cuda")  # (page 0 beside the rows' own)
    wide[:, 3:6] = rows.table
    part = q.PagedRows(rows.starts, rows.lengths, wide[:, 3:6], 4, 2, 48)
    x = randn(88, 2, 64, seed=1, dtype=torch.float16)
    cache.append(0, whole(q, rows), None, x, x)
    qs = randn(4, 4, 64, seed=3, dtype=torch.float16)
    want = cache.attend(0, rows, qs)
    assert torch.equal(cache.attend(0, part, qs), want)
    assert all(torch.equal(a, b) for a, b in zip(cache.read(0, part), cache.read(0, rows)))
    cache.status()
    for length in (49, 60, 80):
        long = q.PagedRows(rows.starts, torch.tensor([40, length], dtype=torch.int32, device="cuda"), wide[:, 3:6], 4, 2, 80)
        out = cache.attend(0, long, qs, out=torch.full_like(qs, 4))
        assert torch.equal(out[:2], want[:2]) and bool((out[2:] == 4).all()) and reported(cache)[0] == 5
        k, v = cache.read(0, long, k_out=torch.full((4, 2, 64), 4.0, device="cuda"), v_out=torch.full((4, 2, 64), 4.0, device="cuda"))
        assert bool((k[2:] == 4).all()) and bool((v[2:] == 4).all()) and reported(cache)[0] == 5
    with pytest.raises(ValueError):
        q.PagedRows(rows.starts, rows.lengths, wide[:, 3:3], 4, 2, 48)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new", FEW_MANY)
@pytest.mark.parametrize("size", [127 * 2.0 ** -40, 1.0, 127 * 2.0 ** 27, 127 * 2.0 ** 40])
def test_rows_of_zeros_beside_rows_of_any_size_in_eight_bits(hd, new, size):
    """Every position has the same score, every other value row is zeros: it has its part of the sum whatever the others' size."""
    length = 300
    rows, pages, _ = make_rows(q, [new], [length], 64)
    cache = q.PagedCache(1, pages, 64, 1, hd, "q8")
    every = whole(q, rows)
    v = torch.full((length, 1, hd), size, device="cuda")
    v[::2] = 0
    cache.append(0, every, None, randn(length, 1, hd, seed=1), v)
    cache.status()
    out = cache.attend(0, rows, torch.zeros(new, 4, hd, device="cuda"), out=torch.empty(new, 4, hd, device="cuda"))
    p = torch.arange(length - new, length, device="cuda", dtype=torch.float64)
    want = (size * ((p + 1) / 2).floor() / (p + 1))[:, None, None].expand_as(out)  # position 0 is one of zeros
    # a scale, its logarithm, its reciprocal and a weight: 2^-21 of one each at most, logarithms of up to 40 another 2^-18; the codes and F16 weights of one are exact
    assert bool(((out.double() - want).abs() <= want * 2.0 ** -16).all())


def test_the_range_of_eight_bits():
    rows, pages, _ = make_rows(q, [3], [3], 16)
    cache = q.PagedCache(1, pages, 16, 1, 64, "q8")
    most, least = 127 * 2.0 ** 40, 2.0 ** -40
    x = randn(3, 1, 64, seed=1)
    x = x / x.abs().amax(-1, keepdim=True)
    x[0] *= most
    x[1] *= 127 * least
    x[2] *= 20 * least
    cache.append(0, rows, None, x, x)
    cache.status()
    for got in cache.read(0, rows, dtype=torch.float32):
        step = torch.tensor([2.0 ** 40, least, least], device="cuda")[:, None, None]  # half of a step of the codes, and the scale's and the quotient's rounding
        assert bool(((got - x).abs() <= step * (0.5 + 2.0 ** -14)).all())
    for big in (most * 1.01, 3e38):
        y = x.clone()
        y[0, 0, 7], y[2, 0, 9] = big, -big
        cache.append(0, rows, None, x, y)
        got = cache.read(0, rows, dtype=torch.float32)[1]
        assert abs(float(got[0, 0, 7]) / most - 1) < 1e-6 and abs(float(got[2, 0, 9]) / most + 1) < 1e-6
        with pytest.raises(q.QuintritError) as e:
            cache.status()
        assert e.value.code == 5


def test_a_report_names_all_that_was_met():
    rows, pages, _ = make_rows(q, [2, 2], [40, 40], 16)
    cache = q.PagedCache(1, pages, 16, 1, 64)
    table = rows.table.clone()
    table[0, 2] = pages
    x = randn(4, 1, 64, seed=1)
    x[3, 0, 5] = float("nan")
    cache.append(0, q.PagedRows(rows.starts, rows.lengths, table, 4, 2, 40), None, x, x)
    code, said = reported(cache)
    assert code == 5 and "page" in said and "finite" in said
    cache.status()


def test_no_report_is_lost_to_one_that_is_being_read():
    """The word is asked for while calls that set it run: each call's report comes with that answer or the next."""
    rows, pages, _ = make_rows(q, [1], [1], 16)
    cache = q.PagedCache(1, pages, 16, 1, 64)
    bad = torch.full((1, 1, 64), float("nan"), device="cuda")
    side = torch.cuda.Stream()
    lost = 0
    with torch.cuda.stream(side):
        for i in range(2000):
            for _ in range(i % 5):
                cache.append(0, rows, None, bad, bad)
            cache.append(0, rows, None, bad, bad)
            seen = 0
            for wait in (False, True):
                if wait:
                    side.synchronize()
                try:
                    cache.status()
                except q.QuintritError:
                    seen += 1
            lost += seen == 0
    assert lost == 0


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new", [4, 20, 300])
def test_windows_next_to_the_largest_number(cache_type, hd, new):
    cache, _, _, _, _ = filled(cache_type, 2, hd, [1, 1], [new - 3, 30], 16)
    rows, _, _ = make_rows(q, [new, new], [new - 3, 30], 16, seed=1)
    qs = queries(cache_type, 2 * new, 8, hd, seed=3)
    want = cache.attend(0, rows, qs)
    assert int(want[3:new].count_nonzero()) > 0
    for window in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - new, 2 ** 30):
        assert torch.equal(cache.attend(0, rows, qs, window=window), want), window


def test_results_belong_to_the_stream_that_writes_them():
    """Memory that was freed on torch's current stream may still be read there; memory that was freed here may still be written on the call's own."""
    rows, pages, _ = make_rows(q, [64], [64], 16)
    cache = q.PagedCache(1, pages, 16, 2, 64)
    x = randn(64, 8, 64, seed=1, dtype=torch.float16)
    ws = cache.attend_workspace(rows, 4)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    calls = (lambda: [cache.append(0, rows, x[:, :4], x[:, 4:6], x[:, 6:], stream=side.cuda_stream)], lambda: list(cache.read(0, rows, stream=side.cuda_stream)),
             lambda: [cache.attend(0, rows, x[:, :4], workspace=ws, stream=side.cuda_stream)])
    for call in calls:
        shapes = [t.shape for t in call()]
        torch.cuda.synchronize()
        freed = [torch.empty(s, dtype=torch.float16, device="cuda") for s in shapes for _ in range(4)]
        places = {t.data_ptr() for t in freed}
        del freed
        results = call()
        mine = {t.data_ptr() for t in results}
        assert not places & mine
        torch.cuda.synchronize()
        del results
        again = [torch.empty(s, dtype=torch.float16, device="cuda") for s in shapes for _ in range(8)]
        assert not mine & {t.data_ptr() for t in again}
    with torch.cuda.stream(side):  # the default stream by its number
        out = cache.read(0, rows, stream=0)
    torch.cuda.synchronize()
    assert torch.equal(out[0], cache.read(0, rows)[0])
    cache.status()


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("new,lengths", [([1, 1], [700, 9000]), ([5, 3], [333, 4097]), ([150, 40], [500, 3000])])
def test_pages_that_the_window_has_left_behind_are_not_looked_at(cache_type, page, new, lengths):
    for window in (1, 30, 100, 257):
        cache, rows, _, _, _ = filled(cache_type, 2, 64, new, lengths, page, seed=2)
        qs = queries(cache_type, rows.tokens, 8, 64, seed=3)
        clean = cache.attend(0, rows, qs, window=window).clone()
        cache.status()
        for s, (n, length) in enumerate(zip(new, lengths)):
            rows.table[s, :max(0, length - n - window + 1) // page] = -1  # given back
        assert torch.equal(cache.attend(0, rows, qs, window=window), clean)
        cache.status()


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("hd,new,lengths", [(64, [1, 1, 1], [40, 40, 40]), (128, [1] * 3, [5000, 9000, 3000]), (64, [3, 3, 3], [900, 20001, 70]), (128, [70, 70, 70], [70, 90, 4000]),
                                            (256, [40, 40, 40], [100, 2000, 300]), (128, [64, 64, 64], [9000, 20000, 9000]), (64, [1, 130, 3], [3000, 9000, 40])])
def test_a_sequence_with_a_page_that_is_not_there_is_left_out(cache_type, hd, new, lengths):
    """Nothing is written for it, whether one block has it whole or many have ranges of it; the others are as they were."""
    cache, rows, _, _, _ = filled(cache_type, 2, hd, new, lengths, 16, seed=2)
    qs = queries(cache_type, rows.tokens, 8, hd, seed=3)
    clean = cache.attend(0, rows, qs).clone()
    cache.status()
    a, b = rows.starts[1:3].tolist()
    for at, page in ((0, -1), ((lengths[1] - 1) // 16, cache.pages), (lengths[1] // 40, 1 << 30)):
        table = rows.table.clone()
        table[1, at] = page
        out = cache.attend(0, q.PagedRows(rows.starts, rows.lengths, table, rows.tokens, max(new), max(lengths)), qs, out=torch.full_like(qs, 4))
        assert torch.equal(out[:a], clean[:a]) and torch.equal(out[b:], clean[b:])
        seen = (out[a:b] != 4).flatten(1).any(1)
        see = torch.arange(lengths[1] - new[1], lengths[1], device="cuda") >= at * 16  # tokens that see a position of the page
        assert not bool(seen[see].any())
        assert torch.equal(out[a:b][seen], clean[a:b][seen])  # (tokens that do not see the page may have been answered)
        assert reported(cache)[0] == 5
    assert torch.equal(cache.attend(0, rows, qs), clean)
    cache.status()


def test_chunks_longer_than_announced():
    rows, pages, _ = make_rows(q, [2, 5, 2], [40, 40, 40], 16, seed=2)
    cache = q.PagedCache(1, pages, 16, 2, 64)
    every = whole(q, rows)
    x = randn(120, 2, 64, seed=1, dtype=torch.float16)
    cache.append(0, every, None, x, x)
    qs = randn(9, 4, 64, seed=3, dtype=torch.float16)
    short = q.PagedRows(rows.starts, rows.lengths, rows.table, 9, 4, 40)
    clean = cache.attend(0, rows, qs)
    cache.status()
    before = cache.read(0, every)
    out = cache.append(0, short, qs, x[20:29], x[30:39], q_out=torch.full_like(qs, 4))
    assert bool((out[2:7] == 4).all()) and torch.equal(out[:2], qs[:2]) and reported(cache)[0] == 5
    after = cache.read(0, every)
    assert all(torch.equal(a[40:80], b[40:80]) and not torch.equal(a, b) for a, b in zip(after, before))
    cache.append(0, every, None, x, x)
    k, _ = cache.read(0, short, k_out=torch.full((9, 2, 64), 4.0, dtype=torch.float16, device="cuda"))
    assert bool((k[2:7] == 4).all()) and torch.equal(k[:2], x[38:40]) and reported(cache)[0] == 5
    out = cache.attend(0, short, qs, out=torch.full_like(qs, 4))
    assert bool((out[2:7] == 4).all()) and torch.equal(out[:2], clean[:2]) and torch.equal(out[7:], clean[7:]) and reported(cache)[0] == 5


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("hd,new", [(64, 1), (64, 3), (64, 60), (128, 1), (128, 3), (128, 5), (128, 20), (128, 60), (256, 1), (256, 3), (256, 60)])
@pytest.mark.parametrize("cap", [50.0, 64.0, 64.1, 1e3, 1e5, 1e9, 1e30, 3e38])
def test_caps_far_above_the_scores(cache_type, hd, new, cap):
    """A cap changes a score z by z^3 / (3 cap^2); what is computed is off no further than scores without a cap."""
    cache, rows, k, v, first = filled(cache_type, 2, hd, [new], [200], 16)
    qs = queries(cache_type, new, 8, hd, seed=3)
    out = cache.attend(0, rows, qs, out=torch.empty(new, 8, hd, device="cuda"), scale=1.0, cap=cap)
    want, mass, size = attention(qs, rows, k, v, first, 1.0, cap)
    # (the capped score is off by eight half steps more: the quotient, the tangent by 2^-20 of itself, the product)
    bound = attention_bound(want, mass, size * (1 + 16 / (hd + 8)), 200, hd, qs.dtype, torch.float32, v, cache_type == "q8", qs.dtype)
    off = (out.double() - want).abs()
    assert bool((off <= bound).all()), f"off by {float((off / bound).max()):.2f} bounds"


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("new", FEW_MANY)
def test_caps_and_scales_next_to_nothing(cache_type, new):
    """Scores below 2^-30 leave all weights equal."""
    cache, rows, k, v, first = filled(cache_type, 2, 64, [new], [200], 16)
    qs = queries(cache_type, new, 8, 64, seed=3)
    want, mass, size = attention(qs * 0, rows, k, v, first, 0.0)
    bound = attention_bound(want, mass, size, 200, 64, qs.dtype, torch.float32, v, cache_type == "q8", qs.dtype)
    for kw in (dict(cap=1e-10), dict(cap=1e-40), dict(scale=0.0), dict(scale=1e-12), dict(scale=1e-40), dict(scale=0.0, cap=1e-40), dict(scale=2.0 ** 30, cap=1e-30)):
        out = cache.attend(0, rows, qs, out=torch.empty(new, 8, 64, device="cuda"), **kw)
        assert bool(((out.double() - want).abs() <= bound).all()), kw
    for scale in (2.0 ** 31, -3e38, float('inf')):
        with pytest.raises(q.QuintritError) as e:
            cache.attend(0, rows, qs, scale=scale)
        assert e.value.code == 2


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new,group,lengths", [([1], 1, [20011]), ([1], 4, [65431]), ([3], 1, [20011]), ([20], 4, [20011]), ([130], 4, [9001]), ([700], 2, [2900]), ([1, 1, 1], 4, [9001, 40, 20011]),
                                               ([1, 3, 1, 2] * 10, 3, [100 + 471 * i for i in range(40)]), ([1, 70, 3, 200], 4, [9001, 3000, 20011, 700])])
@pytest.mark.parametrize("window", [0, 4097])
def test_every_position_counts_once(cache_type, hd, new, group, lengths, window):
    """All scores are zero and a value is 0 or 1: a result is a count over a count, and one position too many or too few among 65431 is seen, at whatever edge of a tile, range or segment."""
    rows, pages, _ = make_rows(q, new, lengths, 64, seed=4)
    cache = q.PagedCache(1, pages, 64, 1, hd, cache_type)
    every = whole(q, rows)
    k, v = randn(every.tokens, 1, hd, seed=1), (randn(every.tokens, 1, hd, seed=2) > 0).float()
    cache.append(0, every, None, k, v)
    qs = torch.zeros(rows.tokens, group, hd, device="cuda", dtype=torch.bfloat16 if cache_type == "bf16" else torch.float16)
    out = cache.attend(0, rows, qs, out=torch.empty(qs.shape, device="cuda"), window=window)
    count = torch.cat([torch.zeros(1, hd, device="cuda", dtype=torch.float64), v[:, 0].double().cumsum(0)])
    s, p = (torch.tensor(x, device="cuda") for x in zip(*places(rows)))
    first = every.starts.long()[s]
    low = (p - window + 1).clamp_min(0) if window else torch.zeros_like(p)
    want = (count[first + p + 1] - count[first + low]) / (p + 1 - low)[:, None].double()
    # The weights are one and counts are exact, but for two roundings of the quotient. Q8 adds reciprocals of scales: up to 64 in a row, a range's tiles and the ranges, fewer than 256 terms, half a step each.
    assert bool(((out.double() - want[:, None]).abs() <= want[:, None] * 2.0 ** (-16 if cache_type == "q8" else -22)).all())
    cache.status()


@pytest.mark.parametrize("hd,in_type", [(64, "f32"), (128, "bf16"), (256, "f32")])
def test_norms_of_values_whose_squares_leave_32_bits(hd, in_type):
    """A head of such values is as long as any other behind its norm; its neighbours in a warp are what they are without it."""
    rows, pages, _ = make_rows(q, [6], [6], 16)
    cache = q.PagedCache(1, pages, 16, 3, hd, "f16")
    size = torch.tensor([1.0, 1e19, 1e25, 3e37, 1e-3, 1e20], device="cuda")[:, None, None]
    x = randn(6, 10, hd, seed=1)
    x = (x / x.abs().amax(-1, keepdim=True) * torch.where(torch.arange(10, device="cuda")[:, None] % 2 == 0, size, torch.ones_like(size))).to(DT[in_type])
    w = 1 + 0.3 * randn(hd, seed=2)
    out = cache.append(0, rows, x[:, :4], x[:, 4:7], x[:, 7:], q_norm=w, k_norm=w, eps=1e-6, q_out=torch.empty(6, 4, hd, device="cuda"))
    k, _ = cache.read(0, rows, dtype=torch.float32)
    at = torch.arange(6, device="cuda")
    for got, heads, half in ((out, x[:, :4], 0.0), (k, x[:, 4:7], EPS[torch.float16])):
        want = written(heads, w, 1e-6, None, False, at)
        bound = want.abs() * half + want.abs().amax(-1, keepdim=True) * (hd / 2 + 16) * 2.0 ** -24
        assert bool(((got.double() - want).abs() <= bound).all())
    with pytest.raises(q.QuintritError):  # the values themselves are too large for F16
        cache.status()
