"""The sequence operators where one call meets what another leaves: shares of many short units, and the like. Plain forms in 64 bits and
tolerances are test_gpu_sequence.py's, where they are derived, unless a test says otherwise."""
import pytest

torch = pytest.importorskip("torch")
from test_gpu_sequence import T, Batch, Cache, check_attention, rng, rows_of, seq, stream  # noqa: E402, F401

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


@pytest.mark.parametrize("far, freq", [(10, 1e-4), (100, 1e-2), (1000, 2e-6), (1 << 20, 1e-9), (1000000, 1.0), (1 << 30, 1.0), (100, 30.0), (3, 1e-12)])
@pytest.mark.parametrize("adjacent", [False, True])
def test_small_sines_have_their_digits(seq, rng, far, freq, adjacent):  # noqa: F811
    """Pairs (1, 0) in f32 come out as cosine and sine themselves.

    Each is good to 10 roundings of 2^-24 of itself: where the coarse part of the angle is zero or as small as the fine one, five of the fine part
    (its conversion, the constant, their product, two additions) and, in the series, the factor 1 - y / 2, its product, two additions; one is spare.
    Beside that the angle, in radians: |position * frequency| 2^-51 (the constant 1 / 2 pi, its product and the one of the 64-bit form here, 2^-53
    each, and a margin of 4/3), |position| 2^-62 (a frequency's last place, half of 2^-64 of a turn) and 2^-55 (an angle's: 2^-58 of a turn)."""
    rows, pairs = 4096, 32
    pos = torch.randint(-far, far, (1, rows), device="cuda", generator=rng, dtype=torch.int32)
    f = (torch.rand(pairs, device="cuda", generator=rng) * 0.9 + 0.1) * freq
    x = torch.zeros(rows, 1, 2 * pairs, device="cuda")
    i = torch.arange(pairs, device="cuda")
    a, b = (2 * i, 2 * i + 1) if adjacent else (i, i + pairs)
    x[..., a] = 1
    y = torch.empty_like(x)
    r = seq.Rotation(2 * pairs, [pairs], f.data_ptr(), pos.data_ptr(), adjacent=adjacent)
    seq.rotary(stream(), r, rows, 2 * pairs, rows_of(seq, x), rows_of(seq, y))
    angle = pos[0].double()[:, None] * f.double()
    off = angle.abs() * 2.0**-51 + pos[0].double().abs()[:, None] * 2.0**-62 + 2.0**-55
    for got, want in ((y[:, 0, a], angle.cos()), (y[:, 0, b], angle.sin())):
        err = (got.double() - want).abs()
        assert (err <= 10 * 2.0**-24 * want.abs() + off).all(), (err / (2.0**-24 * want.abs() + off)).max().item()
