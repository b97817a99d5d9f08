"""The paged cache on a B200 at its edges: sequences shorter than their chunks, segments that follow one another in a block, what tables and lengths may say, the ends of a type's range."""
import pytest

torch = pytest.importorskip("torch")
import quintrit_b200 as q
from tests.paged_reference import make_rows
from tests.test_paged_gpu import DT, TYPES, filled, randn

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
