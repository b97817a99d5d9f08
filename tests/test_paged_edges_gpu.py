"""The paged cache on a B200 at its edges: sequences shorter than their chunks, segments that follow one another in a block, what tables and lengths may say, the ends of a type's range."""
import pytest

torch = pytest.importorskip("torch")
import quintrit_b200 as q
from tests.paged_reference import make_rows
from tests.test_paged_gpu import TYPES, check_attention, filled, randn

pytestmark = pytest.mark.gpu


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
