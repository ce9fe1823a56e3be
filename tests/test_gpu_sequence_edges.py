"""The sequence operators where one call meets what another leaves: shares of many short units, and the like. Plain forms in 64 bits and
tolerances are test_gpu_sequence.py's, where they are derived, unless a test says otherwise."""
import pytest

torch = pytest.importorskip("torch")
from test_gpu_sequence import T, Batch, Cache, check_attention, rng, seq  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim, dtype", [(32, "bf16"), (64, "f16"), (96, "bf16"), (128, "f16"), (128, "bf16")])
@pytest.mark.parametrize("group", [1, 9])
def test_shares_of_many_short_units(seq, rng, dim, dtype, group):  # noqa: F811
    """A block's share holds several units, each of which reuses the memory that the one before joined its sums in: as in 64 bits, and the same
    every time."""
    sequences, heads = 125, 16
    lens = torch.randint(1, 160, (sequences,), generator=rng, device="cuda").tolist()
    batch = Batch(seq, [1] * sequences, lens, 32, rng)
    batch.desc.max_len = 4000  # sizes the launch: shares, not a block for each unit
    cache = Cache(seq, batch.pages, 32, heads, dim).random(rng)
    q = torch.randn(batch.rows, heads * group, dim, device="cuda", generator=rng).to(T[dtype])
    assert seq.cache_attention_workspace_bytes(cache.desc, batch.desc, heads * group) > 0
    first = check_attention(seq, cache, batch, q, dtype).clone()
    for _ in range(3):
        assert torch.equal(first, check_attention(seq, cache, batch, q, dtype))
