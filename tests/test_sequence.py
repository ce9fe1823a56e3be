"""The sequence operators' refusals: every call here is answered before anything of CUDA is touched, so they run without a GPU."""
import ctypes

import pytest

P = 1 << 20  # an address that is aligned for everything and never read


@pytest.fixture(scope="module")
def seq(product_lib_path):
    from colabfold_cuda_kernels import sequence

    return sequence


def good(seq):
    rows = lambda heads, **k: seq.Rows(**dict(dict(data=P, dtype="bf16", heads=heads, row_stride=heads * 64, head_stride=64), **k))  # noqa: E731
    return dict(
        cache=seq.Cache(P, P, P, P, 10, 64, 2, 64),
        batch=seq.Batch(3, 5, 2, 100, 4, P, P, P),
        rotation=seq.Rotation(64, [10, 22], P, P, 5),
        k=rows(2), v=rows(2), q=rows(4), out=rows(4),
    )  # fmt: skip


def call(seq, op, a):
    if op == "rotary":
        return seq.rotary(None, a["rotation"], a.get("rows", 5), a.get("dim", 64), a["q"], a["out"])
    if op == "append":
        return seq.cache_append(None, a["cache"], a["batch"], a["k"], a["v"], a["rotation"], a["q"], a["out"], a.get("status"))
    return seq.cache_attention(None, a["cache"], a["batch"], a["q"], a["out"], a.get("scale", 0.125), a.get("ws", P), 1 << 40, window=a.get("window", 0), lse=a.get("lse"))


def field(name, attribute, value):
    def change(a):
        setattr(a[name], attribute, value)

    change.__name__ = "%s_%s_%s" % (name, attribute, value)
    return change


def apart(attribute, value):
    """An output of its own whose elements overlap."""

    def change(a):
        a["out"].data = 2 * P
        setattr(a["out"], attribute, value)

    change.__name__ = "out_apart_%s_%s" % (attribute, value)
    return change


def entry(name, value):
    def change(a):
        a[name] = value

    change.__name__ = "%s_%s" % (name, value)
    return change


ROTATION = [field("rotation", "dims", 63), field("rotation", "dims", 66), field("rotation", "dims", -2), field("rotation", "axes", 0), field("rotation", "axes", 5),
            field("rotation", "freq", None), field("rotation", "pos", None), field("rotation", "pos", P + 2)]  # fmt: skip
CACHE = [field("cache", n, None) for n in ("k", "v", "k_scale", "v_scale")] + [
    field("cache", "pages", 0), field("cache", "heads", 0), field("cache", "heads", 65537), field("cache", "page_tokens", 48), field("cache", "page_tokens", 256), field("cache", "page_tokens", 0),
    field("cache", "dim", 48), field("cache", "dim", 256), field("cache", "k", P + 8), field("cache", "v_scale", P + 2), entry("cache", None),
]  # fmt: skip
BATCH = [field("batch", n, None) for n in ("first", "len", "table")] + [field("batch", n, -1) for n in ("sequences", "rows", "max_new", "max_len", "table_stride")] + [
    field("batch", "table_pages", 0), field("batch", "max_len", (1 << 30) + 1), field("batch", "first", P + 1), entry("batch", None),
]  # fmt: skip
QUERIES = [field("q", "heads", 1 << 17), field("q", "data", None), field("out", "data", None), field("q", "dtype", 1), field("out", "heads", 2), field("q", "dtype", 3), field("q", "dtype", -1),
           field("q", "row_stride", -64), field("q", "data", P + 1), apart("row_stride", 248), apart("row_stride", 0), apart("head_stride", 56), apart("head_stride", 0)]  # fmt: skip
REFUSED = (
    [("rotary", c) for c in ROTATION + QUERIES + [entry("rows", -1), entry("dim", 0), entry("dim", 1025), field("out", "row_stride", 8), entry("q", None), entry("rotation", None)]]
    + [("append", c) for c in ROTATION + CACHE + BATCH + QUERIES]
    + [("append", c) for c in (field("k", "heads", 4), field("v", "dtype", 1), field("k", "data", P + 8), field("v", "row_stride", 132), field("k", "head_stride", 4),
                               entry("status", P + 1), entry("rotation", None), entry("out", None), entry("k", None), field("out", "head_stride", 72))]
    + [("attention", c) for c in CACHE + BATCH + QUERIES]
    + [("attention", c) for c in (field("q", "dtype", 2), field("q", "data", P + 8), field("out", "head_stride", 68), entry("window", -1), entry("scale", float("nan")),
                                  entry("scale", float("inf")), entry("lse", P + 2), entry("q", None))]
)  # fmt: skip


@pytest.mark.parametrize("op, change", REFUSED, ids=lambda x: x if isinstance(x, str) else x.__name__)
def test_refused(seq, op, change):
    a = good(seq)
    change(a)
    with pytest.raises(ValueError, match="cck_"):
        call(seq, op, a)


@pytest.mark.parametrize("op", ["rotary", "append", "attention"])
def test_tensors_without_rows_may_be_null(seq, op):
    """They get as far as the device."""
    a = good(seq)
    a["rows"] = a["batch"].rows = 0
    for name in "q", "out", "k", "v":
        a[name].data = None
    a["rotation"].pos = None
    with pytest.raises(RuntimeError, match="device"):
        call(seq, op, a)


def test_heads_no_multiple(seq):
    a = good(seq)
    a["q"].heads = a["out"].heads = 3
    with pytest.raises(ValueError, match="multiple"):
        call(seq, "attention", a)


@pytest.mark.parametrize("op", ["rotary", "append", "attention"])
def test_right_arguments_get_as_far_as_the_device(seq, op):
    """The arguments that the refusals above vary are fine: without a GPU the call ends at the device, with one at the address."""
    with pytest.raises(RuntimeError, match="device"):
        call(seq, op, good(seq))


def test_workspace_of_what_is_refused_is_zero(seq):
    a = good(seq)
    assert seq.cache_attention_workspace_bytes(a["cache"], a["batch"], 3) == 0
    a["cache"].dim = 80
    assert seq.cache_attention_workspace_bytes(a["cache"], a["batch"], 4) == 0


def test_too_many_axes(seq):
    with pytest.raises(ValueError):
        seq.Rotation(64, [8, 8, 8, 4, 4], P, P)


def test_descriptors_have_the_headers_layout(seq):
    """Offsets of the C structs on a 64-bit ABI."""
    assert [ctypes.sizeof(t) for t in (seq.Rows, seq.Rotation, seq.Cache, seq.Batch)] == [32, 56, 48, 56]
    assert (seq.Rows.dtype.offset, seq.Rotation.freq.offset, seq.Cache.pages.offset, seq.Batch.first.offset, seq.Batch.table_stride.offset) == (24, 32, 32, 24, 48)


def test_lookup():
    import colabfold_cuda_kernels as cck

    assert cck.SEQUENCE_KERNELS == ("rotary", "cache_append", "cache_attention")
    for name in cck.SEQUENCE_KERNELS:
        assert cck.available(100, name) and not cck.available(90, name)
        assert cck.symbol(name, 100).startswith("Cck")
