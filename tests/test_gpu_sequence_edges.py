"""The sequence operators where one call meets what another leaves: shares of many short units, and the like. Plain forms in 64 bits and
tolerances are test_gpu_sequence.py's, where they are derived, unless a test says otherwise."""
import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_sequence import T, Batch, Cache, append_plain, check_attention, pair_size, rng, rows_of, seq, stream, turned  # noqa: E402, F401

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
    Beside that the angle, in radians: |position * frequency| 2^-52 (the product of the 64-bit form here, 2^-53 where it has more than 53 bits, and its
    cosine), |position| 2^-61 (a frequency's last place, one of 2^-64 of a turn: 2^-61.3) and 2^-55 (an angle's: 2^-58 of a turn)."""
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
    off = angle.abs() * 2.0**-52 + pos[0].double().abs()[:, None] * 2.0**-61 + 2.0**-55
    for got, want in ((y[:, 0, a], angle.cos()), (y[:, 0, b], angle.sin())):
        err = (got.double() - want).abs()
        assert (err <= 10 * 2.0**-24 * want.abs() + off).all(), (err / (2.0**-24 * want.abs() + off)).max().item()


@pytest.fixture
def lose(seq):  # noqa: F811
    """Lets a copy of one block of threads never count as done, for the calls of a test."""
    set_block = seq._lib.cck_set_lost_copy_test
    set_block.restype = None
    yield set_block
    set_block(-1)


def attend(seq, cache, batch, q, out, lse):  # noqa: F811
    need = seq.cache_attention_workspace_bytes(cache.desc, batch.desc, q.shape[1])
    ws = torch.full((need + 16,), 0, dtype=torch.uint8, device="cuda")  # sums of zero, were slots not written
    seq.cache_attention(stream(), cache.desc, batch.desc, rows_of(seq, q), rows_of(seq, out), 0.1, ws.data_ptr(), need, lse=lse.data_ptr())
    torch.cuda.synchronize()


def lost_rows(seq, cache, batch, q, lose, block):  # noqa: F811
    """(row, head) that are NaN when a copy of this block gets lost; all others, and all in the next call, are as they were."""
    want, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
    attend(seq, cache, batch, q, want, lse)
    assert not want.isnan().any()
    out, lost_lse = torch.full_like(q, 5.0), torch.full_like(lse, 5.0)
    for places in range(2):  # apart, and the answer in the queries' place
        x = out if places == 0 else q.clone()
        lose(block)
        attend(seq, cache, batch, q if places == 0 else x, x, lost_lse)
        lose(-1)
        gone = lost_lse.isnan()
        assert torch.equal(gone, x.isnan().any(-1)) and torch.equal(gone, x.isnan().all(-1))
        assert torch.equal(x[~gone], want[~gone]) and torch.equal(lost_lse[~gone], lse[~gone])
    again = torch.empty_like(q)
    attend(seq, cache, batch, q, again, lost_lse)
    assert torch.equal(again, want)
    return gone


@pytest.mark.parametrize("group, new", [(1, 1), (5, 2)])
def test_lost_copy_few_rows(seq, rng, lose, group, new):  # noqa: F811
    """A wait that gives up makes the rows NaN that the rest of the block's share has a part of, and no other."""
    sequences, heads = 125, 16
    lens = torch.randint(40, 160, (sequences,), generator=rng, device="cuda").tolist()
    batch = Batch(seq, [new] * sequences, lens, 32, rng)
    cache = Cache(seq, batch.pages, 32, heads, 64).random(rng)
    q = torch.randn(batch.rows, heads * group, 64, device="cuda", generator=rng).bfloat16()
    whole = lost_rows(seq, cache, batch, q, lose, 23)  # a block for each (sequence, head): sequence 1, head 7
    want = torch.zeros_like(whole)
    want[new : 2 * new, 7 * group : 8 * group] = True
    assert torch.equal(whole, want)
    batch.desc.max_len = 4000  # equal shares of 4 units and more
    gone = lost_rows(seq, cache, batch, q, lose, 100)
    units = gone.view(sequences, new, heads, group).any(3).any(1).flatten()  # in the order of the line
    assert torch.equal(units, gone.view(sequences, new, heads, group).all(3).all(1).flatten())
    first, last, count = units.nonzero().min().item(), units.nonzero().max().item(), units.sum().item()
    assert count == last - first + 1 and 4 <= count <= 12


def test_lost_copy_of_one_long_sequence(seq, rng, lose):  # noqa: F811
    batch = Batch(seq, [1], [30000], 64, rng)
    cache = Cache(seq, batch.pages, 64, 2, 128).random(rng)
    q = torch.randn(1, 8, 128, device="cuda", generator=rng).bfloat16()
    gone = lost_rows(seq, cache, batch, q, lose, 3)  # of the first head's shares
    assert gone[0].tolist() == [True] * 4 + [False] * 4


@pytest.mark.parametrize("dim, dtype", [(64, "bf16"), (128, "f16")])
@pytest.mark.parametrize("group, new", [(1, 40), (2, 140)])
def test_lost_copy_many_rows(seq, rng, lose, group, new, dim, dtype):  # noqa: F811
    """The same for the kernel of many rows: a unit is 256 rows of a head, two of them where a sequence has 280; the block's whole share is NaN."""
    sequences, heads = 60 // group, 8
    lens = torch.randint(new, 300, (sequences,), generator=rng, device="cuda").tolist()
    batch = Batch(seq, [new] * sequences, lens, 32, rng)
    cache = Cache(seq, batch.pages, 32, heads, dim).random(rng)
    q = torch.randn(batch.rows, heads * group, dim, device="cuda", generator=rng).to(T[dtype])
    tiles = -(-new * group // 256)
    unit = torch.arange(new * group, device="cuda").view(new, group) // 256  # of a sequence's rows

    def units(gone):
        """Whether each unit is NaN, in the order of the line: sequence, tile, head."""
        x = gone.view(sequences, new, heads, group)
        parts = [x.permute(0, 2, 1, 3)[..., unit == t] for t in range(tiles)]
        assert all(torch.equal(p.any(-1), p.all(-1)) for p in parts)
        return torch.stack([p.all(-1) for p in parts], 1).flatten()

    whole = units(lost_rows(seq, cache, batch, q, lose, 21))  # a block for each unit, the last tile first
    assert whole.nonzero().flatten().tolist() == [(sequences * tiles - 1 - 21 // heads) * heads + 21 % heads]
    batch.desc.max_len = 4000  # equal shares of 2 units and more
    some = units(lost_rows(seq, cache, batch, q, lose, 70)).nonzero().flatten().tolist()
    assert some == list(range(some[0], some[-1] + 1)) and 2 <= len(some) <= 10


def test_lost_copy_of_one_long_prompt(seq, rng, lose):  # noqa: F811
    batch = Batch(seq, [200], [9000], 64, rng)
    cache = Cache(seq, batch.pages, 64, 2, 64).random(rng)
    q = torch.randn(200, 2, 64, device="cuda", generator=rng).bfloat16()
    gone = lost_rows(seq, cache, batch, q, lose, 3)  # of the first head's shares
    assert gone[:, 0].all() and not gone[:, 1].any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("what, value, status", [("max_new", 0, 1), ("rows", 0, 1), ("max_new", 0, 0)])
def test_append_without_room_says_so(seq, rng, what, value, status, dtype):  # noqa: F811
    """max_new or rows of zero leave every row out: the cache stays, the status is set if there were any."""
    batch = Batch(seq, [3, 0, 2] if status else [0, 0, 0], [40, 9, 20], 32, rng)
    cache = Cache(seq, batch.pages, 32, 2, 64).random(rng)
    old = [x.clone() for x in (cache.k, cache.v, cache.ks, cache.vs)]
    k = torch.randn(5, 2, 64, device="cuda", generator=rng).to(T[dtype])
    setattr(batch.desc, what, value)
    got = torch.zeros(1, dtype=torch.int32, device="cuda")
    seq.cache_append(stream(), cache.desc, batch.desc, rows_of(seq, k), rows_of(seq, k), status=got.data_ptr())
    assert got.item() == status
    assert all(torch.equal(a, b) for a, b in zip(old, (cache.k, cache.v, cache.ks, cache.vs)))


def test_nothing_of_a_batch_without_sequences_is_read(seq, rng):  # noqa: F811
    """Rows of nobody, and no arrays: nothing is written, queries stay."""
    cache = Cache(seq, 2, 32, 2, 64).random(rng)
    old = [x.clone() for x in (cache.k, cache.ks)]
    x, q = (torch.randn(6, n, 64, device="cuda", generator=rng).bfloat16() for n in (2, 4))
    out, freq, pos = torch.full_like(q, 5.0), torch.rand(32, device="cuda", generator=rng), torch.zeros(1, 6, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    batch = seq.Batch(0, 6, 3, 40, 1, None, None, None)
    r = seq.Rotation(64, [32], freq.data_ptr(), pos.data_ptr())
    seq.cache_append(stream(), cache.desc, batch, rows_of(seq, x), rows_of(seq, x), r, rows_of(seq, q), rows_of(seq, out), status=status.data_ptr())
    seq.cache_attention(stream(), cache.desc, batch, rows_of(seq, q), rows_of(seq, out), 0.1)
    torch.cuda.synchronize()
    assert (out == 5.0).all() and status.item() == 0 and all(torch.equal(a, b) for a, b in zip(old, (cache.k, cache.ks)))


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("power", [4, 20, 24, 26, 27, 28, 30, 60, 100, 118])
@pytest.mark.parametrize("dtype, new, dim", [("bf16", 1, 128), ("f16", 3, 64), ("bf16", 40, 128), ("f16", 33, 64), ("bf16", 70, 32)])
def test_scores_of_any_size(seq, rng, dtype, new, dim, power, sign):  # noqa: F811
    """Scores of up to 2^127 either way, all of one sign: one key is ahead of all others by 2^power, and the row is that key's values.

    q is one dimension, a power of two; products with the codes are exact. The probability of the key is rounded to f16 in the product and not in
    the sum, 2^-11, and the result to its type; that of the others is 2^-2^power or less each, so that they add at most 700 times that to the
    logarithm of the sum."""
    length = 700
    batch = Batch(seq, [new], [length], 32, rng)
    cache = Cache(seq, batch.pages, 32, 1, dim).random(rng)
    k, v = (c.clone() for c in cache.views())
    codes = torch.tensor([64.0, 128, 256, 448] if sign < 0 else [64.0, 128, 256], device="cuda")[torch.randint(0, 3 + (sign < 0), (length,), device="cuda", generator=rng)]
    best = 400
    codes[best] = 32 if sign < 0 else 416
    at = torch.tensor(batch.lists[0], device="cuda")[torch.arange(length, device="cuda") // 32], torch.arange(length, device="cuda") % 32
    k[at[0], 0, at[1], 5] = codes.to(torch.float8_e4m3fn).view(torch.uint8)
    cache.put(k, v, torch.full_like(cache.ks, 2.0**30), cache.vs.clone())
    q = torch.zeros(new, 2, dim, device="cuda")
    q[:, :, 5] = sign * 4.0
    scale = 1.1 * 2.0 ** (power - 5 - 30 - 2) / 1.4426950408889634  # the least distance of codes is 32
    q = q.to(T[dtype])
    out, lse = torch.full_like(q, 5.0), torch.full((new, 2), 5.0, device="cuda")
    need = seq.cache_attention_workspace_bytes(cache.desc, batch.desc, 2)
    ws = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
    seq.cache_attention(stream(), cache.desc, batch.desc, rows_of(seq, q), rows_of(seq, out), scale, ws.data_ptr(), need, lse=lse.data_ptr())
    want = cache.token_values(batch.lists[0], length)[1][0, best].expand_as(out)
    assert ((out.double() - want).abs() <= (2.0**-11 + torch.finfo(T[dtype]).eps / 2 + length * 2.0 ** -(2.0**power)) * 1.01 * 448 * cache.vs.double().max()).all()
    top = sign * 4.0 * 2.0**30 * codes[best].item() * scale
    assert ((lse.double() - top).abs() <= 2.0**-20 * (1 + abs(top)) + length * 2.0 ** -(2.0**power)).all()


@pytest.mark.parametrize("dtype, new, dim", [("bf16", 1, 128), ("f16", 3, 64), ("bf16", 40, 128), ("f16", 33, 64)])
def test_scores_whose_last_place_is_sixteen(seq, rng, dtype, new, dim):  # noqa: F811
    """Scores (times log2 e) of 2^27 + 16, then one of 2^27 + 32: as far ahead as a last place, and 2^16 times as probable.

    q, codes and scale are powers of two, so that scores are exact and probabilities powers of two, which f16 holds. What is left is one rounding of
    the result to its type (2^-8 of itself for bf16, of up to 448 here: more than 0.875) and the sums of 501 products in f32, truncated: 501 * 2^-23 of
    the largest, below 2^-14."""
    length, first, best = 700, 500, 600
    batch = Batch(seq, [new], [length], 32, rng)
    cache = Cache(seq, batch.pages, 32, 1, dim).random(rng)
    k, v = (c.clone() for c in cache.views())
    rows = torch.zeros(length, dim, device="cuda")
    rows[:first, 0] = rows[best, 0] = 256
    rows[:first, 1], rows[best, 1] = 2.0**-6, 2.0**-5
    at = torch.tensor(batch.lists[0], device="cuda")[torch.arange(length, device="cuda") // 32], torch.arange(length, device="cuda") % 32
    k[at[0], 0, at[1]] = rows.to(torch.float8_e4m3fn).view(torch.uint8)
    cache.put(k, v, torch.ones_like(cache.ks), torch.ones_like(cache.vs))
    q = torch.zeros(new, 1, dim, device="cuda").to(T[dtype])
    q[..., 0], q[..., 1] = 4.0, 2.0**-7
    scale = 2.0**17 * 0.6931471824645996  # times log2 e in f32: 2^17
    out = torch.full_like(q, 5.0)
    need = seq.cache_attention_workspace_bytes(cache.desc, batch.desc, 1)
    ws = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
    seq.cache_attention(stream(), cache.desc, batch.desc, rows_of(seq, q), rows_of(seq, out), scale, ws.data_ptr(), need)
    values = cache.token_values(batch.lists[0], length)[1][0]
    want = (values[best] + values[:first].sum(0) * 2.0**-16) / (1 + first * 2.0**-16)
    assert ((out.double() - want).abs() <= torch.finfo(T[dtype]).eps / 2 * want.abs() + 2.0**-14 * 448).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize(
    "new, lens, page, dim, rot",
    [([128, 1, 70], [128, 257, 300], 128, 128, 128), ([128], [255], 128, 128, 64), ([64, 5, 0, 33], [64, 70, 9, 100], 64, 96, 96), ([20, 1], [50, 33], 16, 96, 48),
     ([40, 3], [40, 1000], 32, 32, 32), ([1, 1, 1], [1, 128, 129], 128, 128, 128), ([17, 16], [17, 48], 16, 64, 48), ([33], [95], 32, 128, 96)],
)  # fmt: skip
def test_append_rotates_every_size(seq, rng, new, lens, page, dim, rot, adjacent, dtype):  # noqa: F811
    """Rotated keys of all dimensions, types and pairings, pages that are filled at once among them: half a step of e4m3 (2^-4 of itself, or 2^-10 of the
    page's scale) beside the rotation's 2^-20 (|a| + |b|), which half a step more can follow: 1 + 2^-4. Queries to half a step of their type."""
    heads = 3
    batch = Batch(seq, new, lens, page, rng)
    cache = Cache(seq, batch.pages, page, heads, dim).random(rng)
    before = [(c.view(torch.float8_e4m3fn).double(), s.double().clone()) for c, s in zip(cache.views(), (cache.ks, cache.vs))]
    q, k, v = (torch.randn(batch.rows, n, dim, device="cuda", generator=rng).to(T[dtype]) for n in (5, heads, heads))
    pos = torch.randint(-(1 << 20), 1 << 20, (3, batch.rows), device="cuda", generator=rng, dtype=torch.int32)
    freq = torch.rand(rot // 2, device="cuda", generator=rng)
    sections = [rot // 2 - 9, 4, 5]
    r = seq.Rotation(rot, sections, freq.data_ptr(), pos.data_ptr(), batch.rows, adjacent=adjacent)
    out = torch.full_like(q, math.nan)
    seq.cache_append(stream(), cache.desc, batch.desc, rows_of(seq, k), rows_of(seq, v), r, rows_of(seq, q), rows_of(seq, out))
    want_q, want_k = turned(q, pos, freq, sections, adjacent), turned(k, pos, freq, sections, adjacent)
    assert ((out.double() - want_q).abs() <= torch.finfo(T[dtype]).eps / 2 * want_q.abs() + 2.0**-20 * pair_size(q, rot, adjacent)).all()
    want, scale = append_plain(cache, batch, v.double(), before[1])
    assert torch.equal(cache.vs.double(), scale) and torch.equal(cache.views()[1].view(torch.float8_e4m3fn).double(), want)
    want, scale = append_plain(cache, batch, want_k, before[0])
    assert torch.equal(cache.ks.double(), scale)
    got, off = cache.views()[0].view(torch.float8_e4m3fn).double(), pair_size(k, rot, adjacent)
    written = torch.zeros(cache.n, page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(new):
        for i in range(n):
            place = lens[b] - n + i
            p, slot, row = batch.lists[b][place // page], place % page, batch.start(b) + i
            written[p, slot] = True
            s = scale[p][:, None]
            bound = torch.maximum(2.0**-4 * want_k[row].abs(), 2.0**-10 * s) + (1 + 2.0**-4) * 2.0**-20 * off[row]
            assert ((got[p, :, slot] * s - want_k[row]).abs() <= bound).all(), (b, i)
    rest = ~written[:, None, :, None].expand_as(got)  # older tokens, brought to the new scale, and slots of nobody
    assert torch.equal(got[rest], want[rest])


@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("rot", [96, 80, 64])
def test_append_full_pages_of_every_table(seq, rng, rot, adjacent):  # noqa: F811
    """A page of 128 new tokens whose angles take 48 KB, all that a block has without asking for more: beside them it has arrays of its own."""
    batch = Batch(seq, [141, 300], [141, 400], 128, rng)
    cache = Cache(seq, batch.pages, 128, 3, 96).random(rng)
    before = cache.views()[0].view(torch.float8_e4m3fn).double(), cache.ks.double().clone()
    k = torch.randn(batch.rows, 3, 96, device="cuda", generator=rng).bfloat16()
    pos = torch.randint(0, 5000, (1, batch.rows), device="cuda", generator=rng, dtype=torch.int32)
    freq = torch.rand(rot // 2, device="cuda", generator=rng)
    r = seq.Rotation(rot, [rot // 2], freq.data_ptr(), pos.data_ptr(), adjacent=adjacent)
    seq.cache_append(stream(), cache.desc, batch.desc, rows_of(seq, k), rows_of(seq, k), r)
    want, scale = append_plain(cache, batch, turned(k, pos, freq, [rot // 2], adjacent), before)
    assert torch.equal(cache.ks.double(), scale) and torch.equal(cache.views()[0].view(torch.float8_e4m3fn).double(), want)


def test_workspace_of_heads_that_are_refused_is_zero(seq, rng):  # noqa: F811
    batch = Batch(seq, [1], [5000], 32, rng)
    cache = Cache(seq, batch.pages, 32, 1, 64)
    assert seq.cache_attention_workspace_bytes(cache.desc, batch.desc, 1 << 16) > 0
    assert seq.cache_attention_workspace_bytes(cache.desc, batch.desc, (1 << 16) + 16) == 0


@pytest.mark.parametrize("far", [8192, 1 << 28])
@pytest.mark.parametrize("dtype, adjacent, page, dim", [("f16", True, 16, 64), ("bf16", False, 64, 128), ("bf16", True, 32, 96), ("f32", False, 64, 64), ("f16", False, 128, 32)])
def test_rotated_codes_bit_for_bit(seq, rng, dtype, adjacent, page, dim, far):  # noqa: F811
    """The codes of rotated keys are those of the rotation in 64 bits, rounded once: of several million values, none differs. (64 bits leave 2^-50 of a
    value open beside a border, which none of so many comes near to; a position of 28 bits times a frequency of 24 is exact in 64.)"""
    heads, lens = 20, [1500, 1100, 2000, 900]
    batch = Batch(seq, lens, [n + 13 * b for b, n in enumerate(lens)], page, rng)
    cache = Cache(seq, batch.pages, page, heads, dim).random(rng)
    before = cache.views()[0].view(torch.float8_e4m3fn).double(), cache.ks.double().clone()
    k = torch.randn(batch.rows, heads, dim, device="cuda", generator=rng).to(T[dtype])
    pos = torch.randint(0, far, (2, batch.rows), device="cuda", generator=rng, dtype=torch.int32)
    pos[:, ::50] = 0  # exact values, many of them on a border
    pos[1, 1::50] = 0
    freq = (10000.0 ** (-torch.arange(dim // 2, device="cuda") / (dim // 2))).float()
    sections = [dim // 4, dim // 4]
    r = seq.Rotation(dim, sections, freq.data_ptr(), pos.data_ptr(), batch.rows, adjacent=adjacent)
    seq.cache_append(stream(), cache.desc, batch.desc, rows_of(seq, k), rows_of(seq, torch.zeros_like(k)), r)
    want, scale = append_plain(cache, batch, turned(k, pos, freq, sections, adjacent), before)
    assert torch.equal(cache.ks.double(), scale)
    got = cache.views()[0].view(torch.float8_e4m3fn).double()
    assert (got != want).sum().item() == 0


@pytest.mark.parametrize("rot", [None, 0, 32, 96])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_append_of_zeros_of_both_signs(seq, rng, dtype, rot):  # noqa: F811
    """Zero has two codes and is one value: nothing lies on a border there, rotated or not."""
    batch = Batch(seq, [40, 1, 70], [60, 33, 70], 32, rng)
    cache = Cache(seq, batch.pages, 32, 3, 96).random(rng)
    before = [(c.view(torch.float8_e4m3fn).double(), s.double().clone()) for c, s in zip(cache.views(), (cache.ks, cache.vs))]
    k, v = (torch.randn(batch.rows, 3, 96, device="cuda", generator=rng) for _ in range(2))
    for x in (k, v):
        x[torch.rand(x.shape, device="cuda", generator=rng) < 0.5] = 0.0
        x[torch.rand(x.shape, device="cuda", generator=rng) < 0.3] = -0.0
        x[::5], x[1::7] = 0.0, -0.0
    k, v = k.to(T[dtype]), v.to(T[dtype])
    want_k, r = k.double(), None
    if rot is not None:
        pos = torch.randint(0, 3, (2, batch.rows), device="cuda", generator=rng, dtype=torch.int32)
        freq = torch.rand(rot // 2, device="cuda", generator=rng)
        sections = [rot // 2 - 7, 7] if rot else [0, 0]
        r = seq.Rotation(rot, sections, freq.data_ptr(), pos.data_ptr(), batch.rows)
        want_k = turned(k, pos, freq, sections, False)
    seq.cache_append(stream(), cache.desc, batch.desc, rows_of(seq, k), rows_of(seq, v), r)
    for x, codes, scale, old in zip((want_k, v.double()), cache.views(), (cache.ks, cache.vs), before):
        want, want_scale = append_plain(cache, batch, x, old)
        assert torch.equal(scale.double(), want_scale)
        assert torch.equal(codes.view(torch.float8_e4m3fn).double(), want)
