"""The sequence operators against plain implementations in 64 bits.

Tolerances count roundings. u(t) = finfo(t).eps / 2 is the largest relative error of one rounding to t.
 rotary     u(t) |y| for the output, and (|a| + |b|) 2^-20: the angle in turns is good to 2^-26 (rounded to f32 at most 1/2) and, at
            positions up to 2^30, 2^-24 (two roundings in 64 bits of up to 2^28 turns), which is at most 2^-21.3 radians; cosine
            and sine to 2 units in the last place (2^-23), the two products and their sum to 3 * 2^-24.
 append     values are codes times a power of two: equal to the rounding done in 64 bits, bit for bit. Rotated keys: half a step of
            e4m3 (2^-4 |x|, or 2^-10 of the scale below its normal range) plus the rotation's own error.
 attention  E = (D + 8) 2^-23 sum|q k| softmax_scale bounds the error of a score's sum (products of codes are exact, f32 sums truncate). q,
            scaled such that its row's largest lies in [128, 256), is split into e4m3 terms, which hold 8 bits of a bf16 (11 of an
            f16) down to the last term's smallest step of 2^-9, half of which stays open: at most 2^-10 / 128 = 2^-17 of the row's
            largest a dim, so 2^-17 max|q| sum|k| softmax_scale is added to E. A probability is off by 2 E (itself and the sum) + 2^-20
            (exponentials, rescaling, the sum); for the matrix product it is rounded to f16, 2^-11 of itself or 2^-25 where it is
            small, of the largest term; and u(t) |out| for the output.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

T = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def half_step(dtype):
    return torch.finfo(T[dtype]).eps / 2


@pytest.fixture(scope="module")
def seq(product_lib_path):
    from colabfold_cuda_kernels import sequence

    return sequence


@pytest.fixture
def rng():
    return torch.Generator(device="cuda").manual_seed(7)


def stream():
    return torch.cuda.current_stream().cuda_stream


def rows_of(seq, x):
    return seq.Rows(x.data_ptr(), {v: k for k, v in T.items()}[x.dtype], x.shape[1], x.stride(0), x.stride(1))


def i32(*v):
    return torch.tensor(*v, dtype=torch.int32, device="cuda")


# ---- plain forms


def turned(x, pos, freq, sections, adjacent, inverse=False):
    """x [rows][heads][dim] in 64 bits, rotated."""
    rot = 2 * len(freq)
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).cuda()
    angle = (pos.double()[axis] * freq.double()[:, None]).T[:, None]
    c, s = angle.cos(), angle.sin() * (-1 if inverse else 1)
    y = x.double().clone()
    i = torch.arange(rot // 2).cuda()
    i, j = (2 * i, 2 * i + 1) if adjacent else (i, i + rot // 2)
    a, b = x[..., i].double(), x[..., j].double()
    y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    return y


def pair_size(x, rot, adjacent):
    """|a| + |b| of the pair that each value belongs to; 0 where nothing turns."""
    out = torch.zeros_like(x, dtype=torch.float64)
    i = torch.arange(rot // 2).cuda()
    i, j = (2 * i, 2 * i + 1) if adjacent else (i, i + rot // 2)
    out[..., i] = out[..., j] = x[..., i].double().abs() + x[..., j].double().abs()
    return out


class Cache:
    """A cache's buffers, and its contents by token."""

    def __init__(self, seq, pages, page, heads, dim, fill=0x7F):
        self.n, self.p, self.h, self.d = pages, page, heads, dim
        self.k, self.v = (torch.full((pages * heads * page * dim,), fill, dtype=torch.uint8, device="cuda") for _ in range(2))
        self.ks, self.vs = (torch.full((pages, heads), math.nan, device="cuda") for _ in range(2))
        self.desc = seq.Cache(self.k.data_ptr(), self.v.data_ptr(), self.ks.data_ptr(), self.vs.data_ptr(), pages, page, heads, dim)

    def views(self):
        """Codes as [pages][heads][tokens][dim]."""
        k = self.k.view(self.n, self.h, self.p // 8, self.d // 16, 8, 16).permute(0, 1, 2, 4, 3, 5)
        v = self.v.view(self.n, self.h, self.p // 16, self.d, 16).permute(0, 1, 2, 4, 3)
        return k.reshape(self.n, self.h, self.p, self.d), v.reshape(self.n, self.h, self.p, self.d)

    def put(self, k, v, ks, vs):
        """Codes [pages][heads][tokens][dim] and scales."""
        self.k.copy_(k.view(torch.uint8).view(self.n, self.h, self.p // 8, 8, self.d // 16, 16).permute(0, 1, 2, 4, 3, 5).reshape(-1))
        self.v.copy_(v.view(torch.uint8).view(self.n, self.h, self.p // 16, 16, self.d).permute(0, 1, 2, 4, 3).reshape(-1))
        self.ks.copy_(ks), self.vs.copy_(vs)

    def token_values(self, pages, length):
        """Keys and values [heads][length][dim] of a sequence in 64 bits."""
        at = torch.as_tensor(pages, device="cuda").long()
        got = []
        for codes, scale in zip(self.views(), (self.ks, self.vs)):
            x = codes[at].view(torch.float8_e4m3fn).double() * scale[at].double()[..., None, None]
            got.append(x.transpose(0, 1).reshape(self.h, -1, self.d)[:, :length])
        return got

    def random(self, rng, spread=0):
        """Every page filled; with `spread`, scales over 2^spread."""
        shape = (self.n, self.h, self.p, self.d)
        k, v = (torch.randn(shape, device="cuda", generator=rng).clamp(-3.5, 3.5) * 128 for _ in range(2))
        scale = lambda: torch.exp2(torch.randint(-7 - spread, -6 + spread, shape[:2], device="cuda", generator=rng).float())  # noqa: E731
        self.put(k.to(torch.float8_e4m3fn), v.to(torch.float8_e4m3fn), torch.exp2(torch.randint(-8, -6, shape[:2], device="cuda", generator=rng).float()), scale())
        return self


class Batch:
    def __init__(self, seq, new, lens, page, rng=None, pages=None, wide=0, rows=0):
        self.new, self.lens = list(new), list(lens)
        each = [-(-n // page) for n in lens]
        self.pages = pages or sum(each) + 2
        order = torch.randperm(self.pages, device="cuda", generator=rng).tolist() if rng is not None else list(range(self.pages))
        self.lists, at = [], 0
        for n in each:
            self.lists.append(order[at : at + n])
            at += n
        wide = max(1, wide, max(each, default=0))
        self.table = i32([x + [-1] * (wide - len(x)) for x in self.lists] or [[-1] * wide])
        self.first, self.len = i32([sum(new[:b]) for b in range(len(new) + 1)]), i32(self.lens or [0])
        self.rows = rows or sum(new)
        self.make(seq)

    def make(self, seq):
        self.desc = seq.Batch(len(self.new), self.rows, max(self.new, default=0), max(self.lens, default=0), self.table.shape[1], self.first.data_ptr(), self.len.data_ptr(),
                              self.table.data_ptr(), self.table.stride(0))

    def start(self, b):
        return sum(self.new[:b])


# ---- rotary


ROTARY = [
    # rows, heads, dim, rot, sections, adjacent
    (1, 1, 2, 2, [1], False), (1, 40, 128, 128, [64], False), (17, 3, 64, 64, [8, 24], True), (33, 5, 80, 42, [7, 7, 7], True), (33, 5, 80, 42, [0, 20, 1], False),
    (5, 2, 48, 32, [4, 4, 4, 4], False), (129, 7, 96, 96, [48], True), (4, 2, 1024, 512, [200, 56], False), (3, 2, 1022, 1022, [511], True), (9, 4, 24, 8, [4], False),
    (2500, 1, 32, 16, [8], True), (3, 9, 7, 4, [2], False), (6, 2, 64, 0, [0], False),
]  # fmt: skip


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows, heads, dim, rot, sections, adjacent", ROTARY)
def test_rotary(seq, rng, rows, heads, dim, rot, sections, adjacent, dtype, inverse):
    x = torch.randn(rows, heads, dim, device="cuda", generator=rng).to(T[dtype])
    pos = torch.randint(-(1 << 30), 1 << 30, (len(sections), rows), device="cuda", generator=rng, dtype=torch.int32)
    freq = torch.rand(rot // 2, device="cuda", generator=rng)
    r = seq.Rotation(rot, sections, freq.data_ptr() or 16, pos.data_ptr(), rows, adjacent=adjacent)
    y = torch.full_like(x, math.nan)
    seq.rotary(stream(), r, rows, dim, rows_of(seq, x), rows_of(seq, y), inverse=inverse)
    want = turned(x, pos, freq, sections, adjacent, inverse)
    assert ((y.double() - want).abs() <= half_step(dtype) * want.abs() + 2.0**-20 * pair_size(x, rot, adjacent)).all()
    seq.rotary(stream(), r, rows, dim, rows_of(seq, x), rows_of(seq, x), inverse=inverse)  # in place
    assert torch.equal(x, y)


@pytest.mark.parametrize("offset, row_pad, transposed", [(0, 8, False), (1, 0, False), (3, 5, False), (0, 0, True), (8, 0, True)])
def test_rotary_strides(seq, rng, offset, row_pad, transposed):
    rows, heads, dim = 37, 6, 64
    buffers = []
    for _ in range(2):
        flat = torch.randn(offset + rows * (heads * dim + row_pad), device="cuda", generator=rng).bfloat16()
        if transposed:
            buffers.append((flat, flat[offset : offset + rows * heads * dim].view(heads, rows, dim).transpose(0, 1)))
        else:
            buffers.append((flat, flat[offset:].view(rows, heads * dim + row_pad)[:, : heads * dim].view(rows, heads, dim)))
    (_, x), (flat, y) = buffers
    before = flat.clone()
    pos, freq = torch.arange(rows, dtype=torch.int32, device="cuda")[None], torch.rand(32, device="cuda", generator=rng)
    seq.rotary(stream(), seq.Rotation(64, [32], freq.data_ptr(), pos.data_ptr()), rows, dim, rows_of(seq, x), rows_of(seq, y))
    want = turned(x, pos, freq, [32], False)
    assert ((y.double() - want).abs() <= half_step("bf16") * want.abs() + 2.0**-20 * pair_size(x, 64, False)).all()
    got = y.clone()
    y.copy_(before.as_strided(y.shape, y.stride(), y.storage_offset()))  # what lies between the rows is as it was
    assert torch.equal(flat.view(torch.int16), before.view(torch.int16)) and not torch.equal(got, y)


@pytest.mark.parametrize("adjacent", [False, True])
def test_rotary_gradient(seq, rng, adjacent):
    """The inverse is the gradient: against the plain form's by autograd, and against differences of sum(g * y), which is linear in x."""
    rows, heads, dim, rot, sections = 19, 3, 40, 24, [5, 7]
    x, g, step = (torch.randn(rows, heads, dim, device="cuda", generator=rng) for _ in range(3))
    pos = torch.randint(0, 5000, (2, rows), device="cuda", generator=rng, dtype=torch.int32)
    freq = torch.rand(12, device="cuda", generator=rng)
    r = seq.Rotation(rot, sections, freq.data_ptr(), pos.data_ptr(), rows, adjacent=adjacent)
    dx, up, down = (torch.empty_like(x) for _ in range(3))
    seq.rotary(stream(), r, rows, dim, rows_of(seq, g), rows_of(seq, dx), inverse=True)
    leaf = x.double().requires_grad_()
    axis = torch.repeat_interleave(torch.arange(2), torch.tensor(sections)).cuda()
    angle = (pos.double()[axis] * freq.double()[:, None]).T[:, None]
    i = torch.arange(12).cuda()
    i, j = (2 * i, 2 * i + 1) if adjacent else (i, i + 12)
    a, b, gd = leaf[..., i], leaf[..., j], g.double()
    loss = ((a * angle.cos() - b * angle.sin()) * gd[..., i]).sum() + ((b * angle.cos() + a * angle.sin()) * gd[..., j]).sum() + (leaf[..., rot:] * gd[..., rot:]).sum()
    loss.backward()
    assert ((dx.double() - leaf.grad).abs() <= half_step("f32") * leaf.grad.abs() + 2.0**-20 * pair_size(g, rot, adjacent)).all()
    xu, xd = x + step, x - step
    seq.rotary(stream(), r, rows, dim, rows_of(seq, xu), rows_of(seq, up))
    seq.rotary(stream(), r, rows, dim, rows_of(seq, xd), rows_of(seq, down))
    slope = ((up.double() - down.double()) * gd).sum() / 2
    size = (2.0**-20 * 2 * (xu.abs() + xd.abs() + 2 * step.abs()).double().amax() * gd.abs()).sum() + (2.0**-20 * 2 * g.abs().double().amax() * step.abs().double()).sum()
    assert abs(slope - (dx.double() * step.double()).sum()) <= size


# ---- append


def nearest_code(x):
    """The e4m3 value nearest to x, ties to even."""
    step = torch.exp2((torch.frexp(x.abs())[1] - 1).clamp(min=-6).double() - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def scale_for(top):
    return 2.0 ** min(40, max(-40, math.ceil(math.log2(top / 448)))) if top > 0 else 2.0**-40


def append_plain(cache, batch, values, before):
    """Expected values [pages][heads][tokens][dim] and scales after rows `values` (64 bits) were appended to `before` = (values, scales)."""
    x, s = before[0].clone(), before[1].clone()
    for b, n in enumerate(batch.new):
        for i in range(n):
            place = batch.lens[b] - n + i
            if place < 0:
                continue
            page, slot, p0 = batch.lists[b][place // cache.p], place % cache.p, place // cache.p * cache.p
            if slot != 0 and i > 0 and place - 1 >= 0:
                continue  # a block is done with its first new row
            rows = [j for j in range(i, n) if batch.lens[b] - n + j < p0 + cache.p]
            new = values[batch.start(b) + rows[0] : batch.start(b) + rows[-1] + 1].transpose(0, 1)
            for h in range(cache.h):
                fit = scale_for(new[h].abs().max().item())
                if slot:
                    fit = max(fit, s[page, h].item())
                    if fit > s[page, h].item():
                        x[page, h, :slot] = nearest_code(x[page, h, :slot] * (s[page, h].item() / fit))
                s[page, h] = fit
                x[page, h, slot : slot + len(rows)] = nearest_code(new[h] / fit)
    return x, s


def filled(seq, rng, batch, page, heads, dim):
    cache = Cache(seq, batch.pages, page, heads, dim).random(rng)
    return cache, [(c.view(torch.float8_e4m3fn).double(), s.double().clone()) for c, s in zip(cache.views(), (cache.ks, cache.vs))]


APPEND = [
    # new rows, lengths with them, page, heads, dim
    ([1], [1], 16, 1, 32), ([1, 1, 1], [1, 17, 64], 16, 2, 64), ([1, 0, 1, 0], [65, 9, 128, 0], 64, 3, 128), ([5, 1, 40], [5, 33, 100], 32, 2, 96),
    ([130, 0, 257, 3], [130, 77, 300, 200], 64, 2, 128), ([129], [400], 128, 1, 128), ([16, 16], [16, 32], 16, 5, 32), ([300], [300], 128, 2, 64),
]  # fmt: skip


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("new, lens, page, heads, dim", APPEND)
def test_append_unrotated_bit_for_bit(seq, rng, new, lens, page, heads, dim, dtype):
    batch = Batch(seq, new, lens, page, rng)
    cache, before = filled(seq, rng, batch, page, heads, dim)
    k, v = (torch.randn(batch.rows + 3, heads, dim, device="cuda", generator=rng).mul(8.0**w).to(T[dtype]) for w in (1, 2))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    seq.cache_append(stream(), cache.desc, batch.desc, rows_of(seq, k), rows_of(seq, v), status=status.data_ptr())
    for x, codes, scale, old in zip((k, v), cache.views(), (cache.ks, cache.vs), before):
        want, want_scale = append_plain(cache, batch, x.double(), old)
        assert torch.equal(scale.double(), want_scale)
        assert torch.equal(codes.view(torch.float8_e4m3fn).double(), want)
    assert status.item() == 0


@pytest.mark.parametrize("adjacent, rot", [(False, 64), (True, 64), (False, 32), (True, 30), (False, 0)])
@pytest.mark.parametrize("new, lens, page", [([1, 1], [70, 5], 32), ([70, 3, 0, 129], [200, 3, 10, 129], 64)])
def test_append_rotates(seq, rng, new, lens, page, adjacent, rot):
    heads, dim = 2, 64
    batch = Batch(seq, new, lens, page, rng)
    cache, before = filled(seq, rng, batch, page, heads, dim)
    qkv = torch.randn(batch.rows, (6 + 2 * heads) * dim + 8, device="cuda", generator=rng).bfloat16()  # one projection's rows
    q, k, v = (qkv[:, a * dim : b * dim].unflatten(1, (-1, dim)) for a, b in ((0, 6), (6, 6 + heads), (6 + heads, 6 + 2 * heads)))
    pos = torch.randint(0, 1 << 20, (2, batch.rows), device="cuda", generator=rng, dtype=torch.int32)
    freq = torch.rand(rot // 2, device="cuda", generator=rng)
    sections = [rot // 2 - 3, 3] if rot else [0, 0]
    r = seq.Rotation(rot, sections, freq.data_ptr() or 16, pos.data_ptr(), batch.rows, adjacent=adjacent)
    want_k, want_q, size = turned(k, pos, freq, sections, adjacent), turned(q, pos, freq, sections, adjacent), pair_size(q, rot, adjacent)
    size_k, q_old = pair_size(k, rot, adjacent), q.clone()
    out = torch.full((batch.rows, 6, dim), math.nan, device="cuda").bfloat16()
    seq.cache_append(stream(), cache.desc, batch.desc, rows_of(seq, k), rows_of(seq, v), r, rows_of(seq, q), rows_of(seq, out))
    assert ((out.double() - want_q).abs() <= half_step("bf16") * want_q.abs() + 2.0**-20 * size).all()
    want, scale = append_plain(cache, batch, v.double(), before[1])
    assert torch.equal(cache.vs.double(), scale) and torch.equal(cache.views()[1].view(torch.float8_e4m3fn).double(), want)
    _, scale = append_plain(cache, batch, want_k, before[0])
    assert torch.equal(cache.ks.double(), scale)
    for b, n in enumerate(new):
        got = cache.token_values(batch.lists[b], lens[b])[0][:, lens[b] - n :].transpose(0, 1)
        rows = slice(batch.start(b), batch.start(b) + n)
        step = torch.cat([cache.ks[batch.lists[b]].double().T[:, i // page, None] for i in range(lens[b] - n, lens[b])], 1).T[..., None] * 2.0**-10 if n else 0
        assert ((got - want_k[rows]).abs() <= (2.0**-4 * want_k[rows].abs()).clamp(min=step) + 1.07 * 2.0**-20 * size_k[rows]).all()
    assert torch.equal(q, q_old)
    cache2, _ = filled(seq, torch.Generator(device="cuda").manual_seed(1), batch, page, heads, dim)
    seq.cache_append(stream(), cache2.desc, batch.desc, rows_of(seq, k), rows_of(seq, v), r, rows_of(seq, q), rows_of(seq, q))  # queries in place
    assert torch.equal(q, out)


def test_append_token_by_token_grows_the_scale(seq, rng):
    page, heads, dim = 32, 2, 64
    batch = Batch(seq, [1], [70], page, rng)
    cache = Cache(seq, batch.pages, page, heads, dim, fill=0)
    cache.ks.fill_(1.0), cache.vs.fill_(1.0)
    x = [(torch.randn(1, heads, dim, device="cuda", generator=rng) * 1.3**t).bfloat16() for t in range(70)]
    state = [(torch.zeros(batch.pages, heads, page, dim, dtype=torch.float64, device="cuda"), torch.ones(batch.pages, heads, dtype=torch.float64, device="cuda"))] * 2
    for t in range(70):
        batch.lens[0] = t + 1
        batch.len.fill_(t + 1)
        seq.cache_append(stream(), cache.desc, batch.desc, rows_of(seq, x[t]), rows_of(seq, x[69 - t]))
        state = [append_plain(cache, batch, x[u].double(), s) for u, s in zip((t, 69 - t), state)]
    for codes, scale, (want, want_scale) in zip(cache.views(), (cache.ks, cache.vs), state):
        assert torch.equal(codes.view(torch.float8_e4m3fn).double(), want) and torch.equal(scale.double(), want_scale)


@pytest.mark.parametrize("value, scale", [(0.0, 2.0**-40), (1e-30, 2.0**-40), (1e38, 2.0**40), (448.0, 1.0), (450.0, 2.0), (2.0**-40 * 448, 2.0**-40)])
def test_append_scale_limits(seq, value, scale):
    batch = Batch(seq, [16], [16], 16)
    cache = Cache(seq, batch.pages, 16, 1, 32)
    k, v = torch.zeros(16, 1, 32, device="cuda"), torch.zeros(16, 1, 32, device="cuda")
    k[3, 0, 5], v[15, 0, 31] = value, -value
    seq.cache_append(stream(), cache.desc, batch.desc, rows_of(seq, k), rows_of(seq, v))
    want = nearest_code(torch.tensor([value / scale], dtype=torch.float64)).item() * scale
    got_k, got_v = cache.token_values(batch.lists[0], 16)
    assert cache.ks[0, 0].item() == scale == cache.vs[0, 0].item()
    assert got_k[0, 3, 5].item() == want and got_v[0, 15, 31].item() == -want and got_k.abs().sum() == abs(want) == got_v.abs().sum()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("where, value", [("k", math.nan), ("k", math.inf), ("v", math.nan), ("v", -math.inf)])
def test_append_token_that_is_not_finite(seq, rng, where, value, dtype):
    """Its keys are NaN and its values zero in that head; the others' codes and the scale are as without it."""
    batch = Batch(seq, [20], [30], 16, rng)
    cache, before = filled(seq, rng, batch, 16, 2, 64)
    x = {n: torch.randn(20, 2, 64, device="cuda", generator=rng).to(T[dtype]) for n in "kv"}
    x[where][9, 1, 33] = value
    seq.cache_append(stream(), cache.desc, batch.desc, rows_of(seq, x["k"]), rows_of(seq, x["v"]))
    for n, codes, scale, old in zip("kv", cache.views(), (cache.ks, cache.vs), before):
        plain = x[n].double().clone()
        plain[9, 1] = 0
        want, want_scale = append_plain(cache, batch, plain, old)
        if n == "k":
            want[batch.lists[0][19 // 16], 1, 19 % 16] = math.nan
        assert torch.equal(scale.double(), want_scale)
        got = codes.view(torch.float8_e4m3fn).double()
        assert torch.equal(got.nan_to_num(777), want.nan_to_num(777))


@pytest.mark.parametrize("what", ["page", "table", "max_new", "rows", "negative"])
def test_append_leaves_out_what_has_no_place(seq, rng, what):
    batch = Batch(seq, [20, 3], [40, 10], 16, rng)
    cache, _ = filled(seq, rng, batch, 16, 2, 64)
    k, v = (torch.randn(23, 2, 64, device="cuda", generator=rng).bfloat16() for _ in range(2))
    old = [c.clone() for c in cache.views()]
    lost = []  # places of sequence 0 that are left out, by (page, slot)
    pages = batch.lists[0]
    place = lambda t: (pages[t // 16], t % 16)  # noqa: E731
    if what == "page":
        batch.table[0, 1] = cache.n
        lost = [place(t) for t in range(20, 32)]
    elif what == "table":
        batch.table[0, 2] = -3
        lost = [place(t) for t in range(32, 40)]
    elif what == "max_new":
        batch.desc.max_new = 17
        lost = [place(t) for t in range(37, 40)]
    elif what == "rows":
        batch.desc.rows = 20
    else:
        batch.len[1] = 2
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    seq.cache_append(stream(), cache.desc, batch.desc, rows_of(seq, k), rows_of(seq, v), status=status.data_ptr())
    assert status.item() == 1
    new = [c for c in cache.views()]
    for t in range(20, 40):
        at = place(t)
        same = all(torch.equal(a[at[0], :, at[1]], b[at[0], :, at[1]]) for a, b in zip(old, new))
        assert same == (at in lost)
    if what == "negative":  # the last two of the three rows are its places 0 and 1
        got = cache.token_values(batch.lists[1], 2)[1].transpose(0, 1)
        assert ((got - v[21:23].double()).abs() <= 2.0**-4 * v[21:23].double().abs() + 2.0**-10 * cache.vs.double().max()).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("other", [1.0, math.nan])
def test_append_rotation_past_the_largest(seq, rng, dtype, other):
    """A pair whose rotation is over the largest float saturates like every other magnitude, whatever other tokens hold."""
    batch = Batch(seq, [2], [2], 16, rng)
    cache = Cache(seq, batch.pages, 16, 1, 32, fill=0)
    k = torch.full((2, 1, 32), 3e38, device="cuda").to(T[dtype])
    k[1] = other
    pos, freq = i32([[1, 0]]), torch.full((16,), math.pi / 4, device="cuda")  # (0, 1.4) * 3e38
    r = seq.Rotation(32, [16], freq.data_ptr(), pos.data_ptr())
    seq.cache_append(stream(), cache.desc, batch.desc, rows_of(seq, k), rows_of(seq, torch.ones_like(k)), r)
    got = cache.views()[0].view(torch.float8_e4m3fn)[batch.lists[0][0], 0, :2].float()
    assert cache.ks[batch.lists[0][0], 0].item() == 2.0**40
    assert (got[0, 16:] == 448).all() and not got[0].isnan().any() and got[1].isnan().all() == math.isnan(other)


@pytest.mark.parametrize("dtype, offset", [("bf16", 0), ("bf16", 1), ("f32", 0)])
def test_append_leaves_rows_of_nobody(seq, rng, dtype, offset):
    """Queries behind the last sequence stay, and positions of theirs do not matter; an odd alignment of q takes another kernel."""
    batch = Batch(seq, [3, 20], [40, 20], 32, rng, rows=40)
    cache = Cache(seq, batch.pages, 32, 2, 64, fill=0)
    cache.ks.fill_(1.0), cache.vs.fill_(1.0)
    k, v = (torch.randn(40, 2, 64, device="cuda", generator=rng).to(T[dtype]) for _ in range(2))
    q, out = (torch.randn(40 * 320 + 1, device="cuda", generator=rng).to(T[dtype])[offset : offset + 40 * 320].unflatten(0, (40, 5, 64)) for _ in range(2))
    old = out.clone()
    pos = torch.randint(0, 1000, (1, 40), device="cuda", generator=rng, dtype=torch.int32)
    freq = torch.rand(32, device="cuda", generator=rng)
    r = seq.Rotation(64, [32], freq.data_ptr(), pos.data_ptr())
    seq.cache_append(stream(), cache.desc, batch.desc, rows_of(seq, k), rows_of(seq, v), r, rows_of(seq, q), rows_of(seq, out))
    want = torch.empty(23, 5, 64, device="cuda").to(T[dtype])
    seq.rotary(stream(), r, 23, 64, rows_of(seq, q), rows_of(seq, want))
    assert torch.equal(out[:23], want) and torch.equal(out[23:], old[23:])
    codes = [c.clone() for c in cache.views()]
    again = Cache(seq, batch.pages, 32, 2, 64, fill=0)
    again.ks.fill_(1.0), again.vs.fill_(1.0)
    seq.cache_append(stream(), again.desc, batch.desc, rows_of(seq, k), rows_of(seq, v), r)
    assert all(torch.equal(a, b) for a, b in zip(codes, again.views())) and torch.equal(cache.ks, again.ks)


@pytest.mark.parametrize("adjacent", [False, True])
def test_append_many_queries(seq, rng, adjacent):
    """Queries that get a launch of their own: as rotated alone, keys as appended alone, what is behind them stays; in a graph too."""
    new = [2000, 1, 2900, 500]
    batch = Batch(seq, new, [2000, 90, 3000, 517], 64, rng, rows=sum(new) + 30)
    k, v = (torch.randn(batch.rows, 2, 64, device="cuda", generator=rng).bfloat16() for _ in range(2))
    q = torch.randn(batch.rows, 6, 64, device="cuda", generator=rng).bfloat16()
    pos = torch.randint(0, 5000, (1, batch.rows), device="cuda", generator=rng, dtype=torch.int32)
    freq = torch.rand(32, device="cuda", generator=rng)
    r = seq.Rotation(64, [32], freq.data_ptr(), pos.data_ptr(), adjacent=adjacent)
    caches = []
    for _ in range(2):
        caches.append(Cache(seq, batch.pages, 64, 2, 64, fill=0))
        caches[-1].ks.fill_(1.0), caches[-1].vs.fill_(1.0)
    want, out = torch.full_like(q, 5.0), torch.full_like(q, 5.0)
    seq.rotary(stream(), r, sum(new), 64, rows_of(seq, q), rows_of(seq, want))
    seq.cache_append(stream(), caches[0].desc, batch.desc, rows_of(seq, k), rows_of(seq, v), r)
    seq.cache_append(stream(), caches[1].desc, batch.desc, rows_of(seq, k), rows_of(seq, v), r, rows_of(seq, q), rows_of(seq, out))
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    same = lambda: all(torch.equal(getattr(caches[0], n), getattr(caches[1], n)) for n in ("k", "v", "ks", "vs"))  # noqa: E731
    assert same()
    for x in (caches[1].k, caches[1].v, caches[1].ks, caches[1].vs):
        x.fill_(1)
    for c in caches:
        c.k.zero_(), c.v.zero_(), c.ks.fill_(1.0), c.vs.fill_(1.0)
    seq.cache_append(stream(), caches[0].desc, batch.desc, rows_of(seq, k), rows_of(seq, v), r)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out.fill_(7.0)
        seq.cache_append(stream(), caches[1].desc, batch.desc, rows_of(seq, k), rows_of(seq, v), r, rows_of(seq, q), rows_of(seq, out))
        copy = out.clone()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(copy[: sum(new)], want[: sum(new)]) and (copy[sum(new) :] == 7.0).all() and same()


@pytest.mark.parametrize("length", [(1 << 31) - 1, (1 << 30) + 1, -5, -(1 << 31)])
def test_append_length_that_cannot_be(seq, rng, length):
    batch = Batch(seq, [3, 3], [40, 20], 32, rng)
    cache, _ = filled(seq, rng, batch, 32, 2, 64)
    k = torch.randn(6, 2, 64, device="cuda", generator=rng).bfloat16()
    batch.len[0] = length
    old, status = [c.clone() for c in cache.views()], i32([0])
    seq.cache_append(stream(), cache.desc, batch.desc, rows_of(seq, k), rows_of(seq, k), status=status.data_ptr())
    assert status.item() == 1
    for a, b in zip(old, cache.views()):
        assert torch.equal(a[batch.lists[0]], b[batch.lists[0]]) and not torch.equal(a[batch.lists[1]], b[batch.lists[1]])


# ---- attention


def attention_plain(q, k, v, scale, causal, window):
    """out, lse, sum|q k| and sum p |v| of one sequence: q [n][q heads][dim], k and v [heads][len][dim]."""
    n, heads, d = q.shape
    group, size = heads // k.shape[0], k.shape[1]
    k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
    place, at = torch.arange(size - n, size, device="cuda")[:, None], torch.arange(size, device="cuda")[None]
    seen = torch.ones(n, size, dtype=torch.bool, device="cuda")
    if causal:
        seen &= at <= place
    if window:
        seen &= at > place - window
    score = torch.einsum("nhd,htd->hnt", q.double(), k) * scale
    weight = torch.einsum("nhd,htd->hnt", q.double().abs(), k.abs()).masked_fill(~seen, 0).amax(-1) * abs(scale) if size else torch.zeros(heads, n, device="cuda")
    score = score.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(score, -1) if size else torch.full((heads, n), -math.inf, dtype=torch.float64, device="cuda")
    p = torch.exp(score - lse[..., None]).masked_fill(~seen, 0)
    some = seen.any(-1)
    mix = lambda x: torch.einsum("hnt,htd->nhd", p, x)  # noqa: E731
    seen_nan = torch.einsum("nt,ht->nh", seen.double(), (k.isnan().any(-1)).double()) > 0
    out, size_v = mix(v.nan_to_num(0)), mix(v.nan_to_num(0).abs())
    out[seen_nan] = math.nan
    rest = (q.double().abs().amax(-1).T * k.abs().sum(-1).nan_to_num(0).amax(-1, keepdim=True) * abs(scale)).nan_to_num(0) if size else torch.zeros_like(weight)
    return out, lse.T, weight.T, rest.T, size_v, some


def check_attention(seq, cache, batch, q, dtype, causal=True, window=0, scale=None, out=None, poison=()):
    dim, q_heads = cache.d, q.shape[1]
    scale = dim**-0.5 if scale is None else scale
    out = torch.full((q.shape[0], q_heads, dim), 5.0, device="cuda").to(T[dtype]) if out is None else out
    lse = torch.full((q.shape[0], q_heads), 5.0, device="cuda")
    need = seq.cache_attention_workspace_bytes(cache.desc, batch.desc, q_heads)
    ws = torch.full((need + 16,), 0xFF, dtype=torch.uint8, device="cuda")  # NaN, were it read before it is written
    seq.cache_attention(stream(), cache.desc, batch.desc, rows_of(seq, q), rows_of(seq, out), scale, ws.data_ptr(), need, causal=causal, window=window, lse=lse.data_ptr())
    torch.cuda.synchronize()
    assert (ws[need:] == 0xFF).all()
    used = 0
    for b, n in enumerate(batch.new):
        rows = slice(batch.start(b), batch.start(b) + n)
        used += n
        if n == 0:
            continue
        k, v = cache.token_values(batch.lists[b], batch.lens[b])
        if n > batch.lens[b]:  # rows before the sequence's first place see nothing
            early = slice(rows.start, rows.stop - batch.lens[b])
            if causal or batch.lens[b] == 0:
                assert (out[early] == 0).all() and (lse[early] == -math.inf).all()
            rows = slice(early.stop, rows.stop)
            n = batch.lens[b]
            if n == 0:
                continue
        want, want_lse, weight, rest, size_v, some = attention_plain(q[rows], k, v, scale, causal, window)
        got, got_lse = out[rows].double(), lse[rows].double()
        assert torch.equal(got.isnan(), want.isnan().any(-1, keepdim=True).expand_as(got) | want.isnan())
        fine = ~want.isnan()
        err = (dim + 8) * 2.0**-23 * weight + 2.0**-17 * rest
        rel = 2 * err + 2.0**-20 + 2.0**-11
        vs = cache.vs[batch.lists[b]].double().max()
        bound = half_step(dtype) * want.abs() + rel[..., None] * size_v * 1.01 + batch.lens[b] * 2.0**-25 * 448 * vs
        assert ((got - want).abs() <= bound)[fine].all(), ((got - want).abs() / bound)[fine].max().item()
        for r in range(n):
            if not some[r]:
                assert (got[r] == 0).all() and (got_lse[r] == -math.inf).all()
            else:
                ok = ~want[r].isnan().any(-1)
                assert ((got_lse[r] - want_lse[r]).abs() <= err[r] + 2.0**-20 * (1 + want_lse[r].abs()))[ok].all()
    assert (out[used:] == 5.0).all() and (lse[used:] == 5.0).all()
    return out


ATTENTION = [
    # new rows, lengths, page, heads, group, dim
    ([1], [1], 16, 1, 1, 32), ([1], [700], 16, 8, 4, 128), ([1, 1, 1], [33, 0, 64], 32, 2, 8, 64), ([1, 0, 1], [129, 50, 31], 64, 3, 3, 96), ([2, 1, 5], [2, 300, 77], 128, 2, 7, 128),
    ([5, 5], [4000, 5], 32, 5, 1, 64), ([1], [9001], 128, 2, 16, 128), ([3, 9], [200, 1500], 64, 1, 20, 96), ([40, 1, 0, 17], [100, 5000, 9, 17], 64, 2, 4, 128),
    ([130, 61], [130, 700], 16, 2, 2, 64), ([257], [1025], 64, 1, 3, 128), ([300, 7], [300, 4096], 32, 2, 5, 32), ([3, 4], [2, 0], 16, 2, 2, 64),
    ([5, 5], [300, 4000], 32, 2, 4, 64), ([3, 1, 0, 2], [900, 40, 7, 2], 64, 3, 8, 128), ([1, 1], [5000, 33], 16, 1, 17, 96),
]  # fmt: skip


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("new, lens, page, heads, group, dim", ATTENTION)
def test_attention(seq, rng, new, lens, page, heads, group, dim, dtype):
    batch = Batch(seq, new, lens, page, rng, rows=sum(new) + 2)
    cache = Cache(seq, batch.pages, page, heads, dim).random(rng)
    q = torch.randn(batch.rows, heads * group, dim, device="cuda", generator=rng).to(T[dtype])
    check_attention(seq, cache, batch, q, dtype)


@pytest.mark.parametrize("causal, window", [(False, 0), (True, 1), (True, 17), (True, 300), (False, 40)])
@pytest.mark.parametrize("new, lens, page, heads, group, dim", [([1, 1], [1000, 40], 32, 2, 4, 128), ([70, 3, 1], [500, 300, 1], 16, 2, 3, 64), ([200], [1000], 64, 1, 4, 128)])
def test_attention_masks(seq, rng, new, lens, page, heads, group, dim, causal, window):
    batch = Batch(seq, new, lens, page, rng)
    cache = Cache(seq, batch.pages, page, heads, dim).random(rng)
    q = torch.randn(batch.rows, heads * group, dim, device="cuda", generator=rng).bfloat16()
    check_attention(seq, cache, batch, q, "bf16", causal, window)


@pytest.mark.parametrize("causal, window", [(True, 0), (True, 70), (False, 33)])
@pytest.mark.parametrize("new, lens, page, heads, group, dim", [([150, 20], [900, 33], 16, 1, 2, 96), ([40], [800], 128, 3, 7, 32), ([2, 2], [700, 50], 128, 2, 6, 32)])
def test_attention_masks_and_pages(seq, rng, new, lens, page, heads, group, dim, causal, window):
    batch = Batch(seq, new, lens, page, rng)
    cache = Cache(seq, batch.pages, page, heads, dim).random(rng)
    q = torch.randn(batch.rows, heads * group, dim, device="cuda", generator=rng).to(torch.float16)
    check_attention(seq, cache, batch, q, "f16", causal, window)


@pytest.mark.parametrize("sequences, new, most, heads, dim", [(70, 1, 2300, 1, 128), (40, 20, 700, 1, 64), (112, 1, 2300, 32, 32), (75, 18, 500, 16, 32), (33, 40, 500, 1, 96)])
def test_attention_many_sequences(seq, rng, sequences, new, most, heads, dim):
    """More than a warp looks over at once, cut into shares and, with many heads, in whole units; some have nothing new, some no tokens."""
    lens = torch.randint(0, 200, (sequences,), generator=rng, device="cuda").tolist()
    lens[1], lens[-1] = most, most // 2
    news = [min(n, 0 if b % 7 == 5 else 1 + b % new) for b, n in enumerate(lens)]
    batch = Batch(seq, news, lens, 16, rng)
    batch.desc.max_new = new
    cache = Cache(seq, batch.pages, 16, heads, dim).random(rng)
    q = torch.randn(batch.rows, heads, dim, device="cuda", generator=rng).bfloat16()
    check_attention(seq, cache, batch, q, "bf16")


@pytest.mark.parametrize("causal, window", [(True, 0), (True, 17), (False, 0), (True, (1 << 31) - 1)])
@pytest.mark.parametrize("new", [[1, 1, 1], [60, 30, 50]])
def test_attention_length_that_cannot_be(seq, rng, new, causal, window):
    """Rows past the table are NaN, rows before the first place see nothing, and both come to an end; the others are as they were."""
    batch = Batch(seq, new, [200, 300, 90], 32, rng)
    cache = Cache(seq, batch.pages, 32, 2, 64).random(rng)
    q = torch.randn(batch.rows, 2, 64, device="cuda", generator=rng).bfloat16()
    want = check_attention(seq, cache, batch, q, "bf16", causal, window).clone()
    batch.len[0], batch.len[2] = (1 << 31) - 1, -(1 << 31)
    out, need = torch.empty_like(q), seq.cache_attention_workspace_bytes(cache.desc, batch.desc, 2)
    ws = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
    seq.cache_attention(stream(), cache.desc, batch.desc, rows_of(seq, q), rows_of(seq, out), 0.125, ws.data_ptr(), need, causal=causal, window=window)
    a, b = new[0], new[0] + new[1]
    assert out[:a].isnan().all() and torch.equal(out[a:b], want[a:b]) and (out[b:] == 0).all()


def test_attention_window_leaves_old_pages_alone(seq, rng):
    """Pages that no row sees any more may be gone from the table."""
    batch = Batch(seq, [2, 150], [1000, 1000], 16, rng)
    cache = Cache(seq, batch.pages, 16, 2, 64).random(rng)
    q = torch.randn(152, 4, 64, device="cuda", generator=rng).bfloat16()
    want = check_attention(seq, cache, batch, q, "bf16", True, 100)
    batch.table[0, : (999 - 100) // 16] = -1
    batch.table[1, : (851 - 100) // 16] = 1 << 30
    assert torch.equal(want, check_attention(seq, cache, batch, q, "bf16", True, 100))


@pytest.mark.parametrize("new, lens, page", [([1], [40], 64), ([6], [70], 16), ([100], [161], 128)])
def test_attention_unused_slots_hold_anything(seq, rng, new, lens, page):
    """NaN codes behind a sequence's last token and in pages that nobody has change nothing."""
    batch = Batch(seq, new, lens, page, rng)
    cache = Cache(seq, batch.pages, page, 2, 64).random(rng)
    q = torch.randn(batch.rows, 6, 64, device="cuda", generator=rng).half()
    want = check_attention(seq, cache, batch, q, "f16")
    k, v = (c.clone() for c in cache.views())
    used = torch.zeros(cache.n, page, dtype=torch.bool, device="cuda")
    for t in range(lens[0]):
        used[batch.lists[0][t // page], t % page] = True
    free = ~used[:, None, :, None].expand_as(k)
    for codes in (k, v):
        codes[free] = 0x7F
    ks, vs = cache.ks.clone(), cache.vs.clone()
    ks[~used.any(1)], vs[~used.any(1)] = math.nan, math.nan
    cache.put(k, v, ks, vs)
    assert torch.equal(want, check_attention(seq, cache, batch, q, "f16"))


@pytest.mark.parametrize("bad", [-1, -(1 << 31), 1 << 30, "n"])
@pytest.mark.parametrize("new, lens, page", [([1, 1], [100, 300], 32), ([60, 20], [100, 300], 16), ([150, 20], [150, 300], 64)])
def test_attention_bad_page(seq, rng, new, lens, page, bad):
    """Rows that see a page that is not there are NaN, all others as they were."""
    batch = Batch(seq, new, lens, page, rng)
    cache = Cache(seq, batch.pages, page, 2, 64).random(rng)
    q = torch.randn(batch.rows, 4, 64, device="cuda", generator=rng).bfloat16()
    want = check_attention(seq, cache, batch, q, "bf16").clone()
    col = 90 // page
    batch.table[0, col] = cache.n if bad == "n" else bad
    out = torch.empty_like(q)
    need = seq.cache_attention_workspace_bytes(cache.desc, batch.desc, 4)
    ws = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
    seq.cache_attention(stream(), cache.desc, batch.desc, rows_of(seq, q), rows_of(seq, out), 0.125, ws.data_ptr(), need)
    see = torch.tensor([lens[0] - new[0] + i >= col * page for i in range(new[0])] + [False] * new[1], device="cuda")
    assert out[see].isnan().all() and torch.equal(out[~see], want[~see])


@pytest.mark.parametrize("new", [[1], [30]])
def test_attention_table_shorter_than_the_sequence(seq, rng, new):
    batch = Batch(seq, new, [200], 32, rng)
    cache = Cache(seq, batch.pages, 32, 1, 64).random(rng)
    q = torch.randn(new[0], 2, 64, device="cuda", generator=rng).bfloat16()
    batch.desc.table_pages = 5
    out = torch.zeros_like(q)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    seq.cache_attention(stream(), cache.desc, batch.desc, rows_of(seq, q), rows_of(seq, out), 0.125, ws.data_ptr(), 1 << 20)
    assert out.isnan().all()


@pytest.mark.parametrize("new", [[3], [140]])
def test_attention_poisoned_token(seq, rng, new):
    """A key that is NaN makes the rows that see it NaN and no other."""
    batch = Batch(seq, new, [300], 32, rng)
    cache = Cache(seq, batch.pages, 32, 2, 64).random(rng)
    k, v = (c.clone() for c in cache.views())
    k[batch.lists[0][298 // 32], 1, 298 % 32], v[batch.lists[0][298 // 32], 1, 298 % 32] = 0x7F, 0
    cache.put(k, v, cache.ks.clone(), cache.vs.clone())
    q = torch.randn(new[0], 4, 64, device="cuda", generator=rng).bfloat16()
    out = check_attention(seq, cache, batch, q, "bf16")
    assert out[-2:, 2:].isnan().all() and not out[:-2].isnan().any() and not out[:, :2].isnan().any()


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("new", [[3], [140]])
def test_attention_query_that_is_not_finite(seq, rng, new, value):
    batch = Batch(seq, new, [200], 32, rng)
    cache = Cache(seq, batch.pages, 32, 2, 64).random(rng)
    q = torch.randn(new[0], 4, 64, device="cuda", generator=rng).bfloat16()
    want = check_attention(seq, cache, batch, q, "bf16").clone()
    q[1, 2, 9] = value
    out = torch.empty_like(q)
    ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    seq.cache_attention(stream(), cache.desc, batch.desc, rows_of(seq, q), rows_of(seq, out), 0.125, ws.data_ptr(), 1 << 24)
    assert out[1, 2].isnan().all()
    out[1, 2] = want[1, 2]
    assert torch.equal(out, want)


@pytest.mark.parametrize("new, lens", [([1], [600]), ([140], [600])])
def test_attention_scales_far_apart(seq, rng, new, lens):
    """Pages whose values differ by 2^40, values that are all zero, queries of any size."""
    batch = Batch(seq, new, lens, 32, rng)
    cache = Cache(seq, batch.pages, 32, 2, 64).random(rng, spread=20)
    k, v = (c.clone() for c in cache.views())
    v[batch.lists[0][3]] = 0
    vs = cache.vs.clone()
    vs[batch.lists[0][3]] = 2.0**-40
    cache.put(k, v, cache.ks.clone(), vs)
    q = torch.randn(new[0], 4, 64, device="cuda", generator=rng) * torch.logspace(-20, 3, 4, device="cuda")[None, :, None]
    check_attention(seq, cache, batch, q.bfloat16(), "bf16", scale=0.01)
    cache.vs.mul_(1.37), cache.ks.mul_(0.77)  # a cache that was filled in another way: scales need not be powers of two
    check_attention(seq, cache, batch, q.bfloat16(), "bf16", scale=-0.01)
    cache.views()
    cache.v.zero_()
    check_attention(seq, cache, batch, q.bfloat16(), "bf16", scale=0.0)


@pytest.mark.parametrize("new", [[2, 3], [150, 20]])
def test_attention_strides(seq, rng, new):
    batch = Batch(seq, new, [160, 300], 32, rng)
    cache = Cache(seq, batch.pages, 32, 2, 64).random(rng)
    rows = sum(new)
    wide = torch.randn(rows, 10 * 64 + 8, device="cuda", generator=rng).bfloat16()
    q = wide[:, 128 : 128 + 256].unflatten(1, (4, 64))
    out = torch.full((4, rows + 3, 72), 5.0, device="cuda").bfloat16()
    view = out[:, :rows, :64].transpose(0, 1)
    check_attention(seq, cache, batch, q, "bf16", out=view)
    assert (out[:, rows:] == 5.0).all() and (out[:, :, 64:] == 5.0).all()


def test_attention_sizes_that_are_only_bounds(seq, rng):
    """max_new and max_len may be larger than what the arrays hold; a length over max_len is still read whole."""
    batch = Batch(seq, [1, 3], [2000, 600], 32, rng)
    cache = Cache(seq, batch.pages, 32, 2, 64).random(rng)
    q = torch.randn(4, 8, 64, device="cuda", generator=rng).bfloat16()
    for max_new, max_len in ((3, 2000), (9, 100000), (200, 2000), (3, 100), ((1 << 31) - 1, 1 << 30)):
        batch.desc.max_new, batch.desc.max_len = max_new, max_len
        check_attention(seq, cache, batch, q, "bf16")


@pytest.mark.parametrize("new", [1, 130])
def test_offsets_past_32_bits(seq, rng, new):
    """A pool of more than 2^32 bytes whose last pages are in use."""
    page, heads, dim, pages = 128, 8, 128, 33000
    batch = Batch(seq, [new], [300], page)
    batch.lists = [[pages - 1, pages - 3, pages - 2]]
    batch.table.copy_(i32(batch.lists))
    k, v = (torch.empty(pages * heads * page * dim, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.ones(pages, heads, device="cuda") for _ in range(2))
    small = Cache(seq, 3, page, heads, dim).random(rng)
    for big, part in ((k, small.k), (v, small.v)):
        big[-part.numel() :] = part
    ks[-3:], vs[-3:] = small.ks, small.vs
    small.desc = seq.Cache(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages, page, heads, dim)
    batch.lists = [[2, 0, 1]]
    q, nk, nv = (torch.randn(new, n, dim, device="cuda", generator=rng).bfloat16() for n in (16, 8, 8))
    check_attention(seq, small, batch, q, "bf16")
    seq.cache_append(stream(), small.desc, batch.desc, rows_of(seq, nk), rows_of(seq, nv))
    for big, part in ((k, small.k), (v, small.v)):
        part.copy_(big[-part.numel() :])
    small.ks.copy_(ks[-3:]), small.vs.copy_(vs[-3:])
    got = small.token_values([2, 0, 1], 300)[1][:, 300 - new :].transpose(0, 1)
    assert ((got - nv.double()).abs() <= 2.0**-4 * nv.double().abs() + 2.0**-10 * small.vs.double().max()).all()
    check_attention(seq, small, batch, q, "bf16")


# ---- together


def step(seq, cache, batch, x, r, out, ws, need, on=None):
    on = stream() if on is None else on
    seq.cache_append(on, cache.desc, batch.desc, rows_of(seq, x["k"]), rows_of(seq, x["v"]), r, rows_of(seq, x["q"]), rows_of(seq, x["q"]))
    seq.cache_attention(on, cache.desc, batch.desc, rows_of(seq, x["q"]), rows_of(seq, out), 0.125, ws.data_ptr(), need)


def test_prompt_then_tokens(seq, rng):
    """Prompts, then tokens one by one, as a captured step that is replayed: the same rows as from the cache read back in 64 bits, and near those of
    exact keys and values."""
    page, heads, group, dim, steps = 32, 2, 3, 64, 20
    lens = [70, 1, 33]
    batch = Batch(seq, lens, [n + steps for n in lens], page, rng)  # pages for all that comes
    cache = Cache(seq, batch.pages, page, heads, dim)
    freq = (100.0 ** (-torch.arange(32, device="cuda") / 32)).float()

    def inputs(rows):
        return {n: torch.randn(rows, m, dim, device="cuda", generator=rng).bfloat16() for n, m in (("q", heads * group), ("k", heads), ("v", heads))}

    history = [[] for _ in lens]

    def keep(x, pos, new):
        k, at = turned(x["k"], pos, freq, [32], False), 0
        for b, n in enumerate(new):
            history[b].append((k[at : at + n], x["v"][at : at + n].double()))
            at += n

    batch.lens = list(lens)
    batch.len.copy_(i32(lens))
    batch.make(seq)
    x = inputs(sum(lens))
    pos = torch.cat([torch.arange(n) for n in lens]).int().cuda()[None]
    keep(x, pos, lens)
    out = torch.empty_like(x["q"])
    need = seq.cache_attention_workspace_bytes(cache.desc, batch.desc, heads * group)
    ws = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
    step(seq, cache, batch, x, seq.Rotation(64, [32], freq.data_ptr(), pos.data_ptr()), out, ws, need)

    batch.new, batch.rows, batch.first = [1] * 3, 3, i32([0, 1, 2, 3])
    batch.lens = [n + steps for n in lens]  # the bound that the launch is sized by
    batch.make(seq)
    need = seq.cache_attention_workspace_bytes(cache.desc, batch.desc, heads * group)
    ws = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
    x, out, pos = inputs(3), torch.empty(3, heads * group, dim, device="cuda").bfloat16(), torch.zeros(1, 3, dtype=torch.int32, device="cuda")
    r = seq.Rotation(64, [32], freq.data_ptr(), pos.data_ptr())
    batch.len.copy_(i32(lens))
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        batch.len.add_(1)
        step(seq, cache, batch, x, r, out, ws, need)
    batch.len.copy_(i32(lens))
    for t in range(steps):
        for n, fresh in inputs(3).items():
            x[n].copy_(fresh)
        pos.copy_(i32([[n + t for n in lens]]))
        keep(x, pos, [1] * 3)
        graph.replay()
        torch.cuda.synchronize()
        batch.lens = [n + t + 1 for n in lens]
        assert batch.len.tolist() == batch.lens
        check_attention(seq, cache, batch, x["q"], "bf16")
        for b in range(3):
            k, v = (torch.cat([h[i] for h in history[b]]).transpose(0, 1) for i in (0, 1))
            got = cache.token_values(batch.lists[b], batch.lens[b])
            for exact, stored, scale in ((k, got[0], cache.ks), (v, got[1], cache.vs)):  # half a step, and what rescaling lost below the normal range
                assert ((stored - exact).abs() <= 2.0**-4 * exact.abs() + 2.0**-9 * scale[batch.lists[b]].max().double() + 2.0**-18).all()
            want = attention_plain(x["q"][b : b + 1], *got, 0.125, True, 0)[0]
            bound = half_step("bf16") * want.abs() + 2.0**-10 * got[1].abs().max()
            assert ((out[b : b + 1].double() - want).abs() <= bound).all()


@pytest.mark.parametrize("new", [1, 140])
def test_two_streams_and_two_graphs(seq, rng, new):
    """Calls that overlap, eager and captured, each with a workspace of its own, give what they give alone."""
    sets = []
    for b in range(2):
        batch = Batch(seq, [new] * 4, [3000 + 500 * b] * 4, 64, rng)
        cache = Cache(seq, batch.pages, 64, 2, 128).random(rng)
        q = torch.randn(batch.rows, 8, 128, device="cuda", generator=rng).bfloat16()
        need = seq.cache_attention_workspace_bytes(cache.desc, batch.desc, 8)
        ws = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
        out = torch.empty_like(q)
        go = lambda on, c=cache, a=batch, q=q, out=out, ws=ws, need=need: seq.cache_attention(on, c.desc, a.desc, rows_of(seq, q), rows_of(seq, out), 0.09, ws.data_ptr(), need)  # noqa: E731
        go(stream())
        torch.cuda.synchronize()
        sets.append((go, out, out.clone(), torch.cuda.Stream(), torch.cuda.CUDAGraph(), (cache, batch, q, ws)))
    for go, out, _, side, graph, _ in sets:
        with torch.cuda.graph(graph, stream=side):
            go(stream())
    for turn in range(4):
        for go, out, _, side, graph, _ in sets:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                out.fill_(7)
                if turn % 2:
                    graph.replay()
                else:
                    go(side.cuda_stream)
        torch.cuda.synchronize()
        for _, out, want, _, _, _ in sets:
            assert torch.equal(out, want)


@pytest.mark.parametrize("new, heads, group, dim", [([1, 1, 1], 2, 4, 128), ([5, 1, 3], 1, 4, 64), ([150, 40, 300], 2, 2, 64)])
def test_in_place_and_replayed_with_other_lengths(seq, rng, new, heads, group, dim):
    """Queries overwritten by the answer, and a captured call whose sequences' lengths and rows have changed since, both cut into shares."""
    most = [5000, 3000, 7000]
    batch = Batch(seq, new, most, 32, rng)
    cache = Cache(seq, batch.pages, 32, heads, dim).random(rng)
    q = torch.randn(batch.rows, heads * group, dim, device="cuda", generator=rng).bfloat16()
    need = seq.cache_attention_workspace_bytes(cache.desc, batch.desc, heads * group)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    assert need > 0

    def attend(out):
        seq.cache_attention(stream(), cache.desc, batch.desc, rows_of(seq, q if out is not place else place), rows_of(seq, out), 0.1, ws.data_ptr(), need)

    place, out = q.clone(), torch.empty_like(q)
    attend(out), attend(place)
    assert torch.equal(out, place)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend(out)
    for lens, rows in (([700, 3000, 20], new), ([0, 17, 6999], [0, 1, new[2]]), ([5000, 1, 1], [new[0], 1, 0])):
        batch.len.copy_(i32(lens)), batch.first.copy_(i32([0, rows[0], rows[0] + rows[1], sum(rows)]))
        out.fill_(5.0)
        graph.replay()
        replayed = out.clone()
        out.fill_(5.0)
        attend(out)
        torch.cuda.synchronize()
        assert torch.equal(replayed, out)
        batch.new, batch.lens = rows, lens
        check_attention(seq, cache, batch, q, "bf16", scale=0.1)


def test_same_result_every_time(seq, rng):
    batch = Batch(seq, [1, 2, 150], [5000, 40, 900], 32, rng)
    cache = Cache(seq, batch.pages, 32, 2, 128).random(rng)
    q = torch.randn(batch.rows, 8, 128, device="cuda", generator=rng).bfloat16()
    first = check_attention(seq, cache, batch, q, "bf16").clone()
    for _ in range(3):
        assert torch.equal(first, check_attention(seq, cache, batch, q, "bf16"))


def test_nothing_to_do(seq):
    batch = Batch(seq, [], [], 16)
    cache = Cache(seq, 2, 16, 1, 32)
    x = torch.zeros(1, 1, 32, device="cuda").bfloat16()
    old = cache.k.clone()
    for b in (batch, Batch(seq, [0, 0], [5, 0], 16)):
        seq.cache_append(stream(), cache.desc, b.desc, rows_of(seq, x), rows_of(seq, x))
        seq.cache_attention(stream(), cache.desc, b.desc, rows_of(seq, x), rows_of(seq, x), 1.0)
    pos = i32([[0]])
    seq.rotary(stream(), seq.Rotation(0, [0], pos.data_ptr(), pos.data_ptr()), 0, 32, rows_of(seq, x), rows_of(seq, x))
    torch.cuda.synchronize()
    assert torch.equal(cache.k, old) and (x == 0).all()


def test_refusals_that_need_a_device(seq, rng):
    batch = Batch(seq, [1], [5000], 32, rng)
    cache = Cache(seq, batch.pages, 32, 1, 64).random(rng)
    q = torch.zeros(1, 1, 64, device="cuda").bfloat16()
    need = seq.cache_attention_workspace_bytes(cache.desc, batch.desc, 1)
    ws = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
    assert need > 0  # a long sequence on one head is split
    for ptr, size in ((ws.data_ptr(), need - 1), (None, need), (ws.data_ptr() + 4, need)):
        with pytest.raises(ValueError, match="workspace"):
            seq.cache_attention(stream(), cache.desc, batch.desc, rows_of(seq, q), rows_of(seq, q), 1.0, ptr, size)
    memory = torch.zeros(64, dtype=torch.int32)  # of the host
    for owner, name in [(cache.desc, n) for n in ("k", "v", "k_scale", "v_scale")] + [(batch.desc, n) for n in ("first", "len", "table")]:
        was = getattr(owner, name)
        setattr(owner, name, memory.data_ptr())
        with pytest.raises(RuntimeError, match="device memory"):
            seq.cache_attention(stream(), cache.desc, batch.desc, rows_of(seq, q), rows_of(seq, q), 1.0, ws.data_ptr(), need)
        with pytest.raises(RuntimeError, match="device memory"):
            seq.cache_append(stream(), cache.desc, batch.desc, rows_of(seq, q), rows_of(seq, q))
        setattr(owner, name, was)
    with pytest.raises(RuntimeError, match="device memory"):
        seq.cache_attention(stream(), cache.desc, batch.desc, rows_of(seq, q), rows_of(seq, q), 1.0, ws.data_ptr(), need, lse=memory.data_ptr())
    with pytest.raises(RuntimeError, match="device memory"):
        seq.rotary(stream(), seq.Rotation(64, [32], ws.data_ptr(), memory.data_ptr()), 1, 64, rows_of(seq, q), rows_of(seq, q))
    host = torch.zeros(1, 1, 64).bfloat16()
    with pytest.raises(RuntimeError, match="device memory"):
        seq.cache_attention(stream(), cache.desc, batch.desc, rows_of(seq, host), rows_of(seq, q), 1.0, ws.data_ptr(), need)
