"""What the sequence operators' entry points take although it looks like nothing: answered before anything of CUDA is touched."""
import pytest

from test_sequence import call, good, seq  # noqa: F401


@pytest.mark.parametrize("op", ["append", "attention"])
def test_arrays_of_a_batch_without_sequences_may_be_null(seq, op):  # noqa: F811
    a = good(seq)
    a["batch"].sequences = 0
    a["batch"].first = a["batch"].len = a["batch"].table = None
    with pytest.raises(RuntimeError, match="device"):  # as far as the device
        call(seq, op, a)


@pytest.mark.parametrize("name", ["first", "len", "table"])
@pytest.mark.parametrize("op", ["append", "attention"])
def test_arrays_of_a_batch_with_sequences_may_not(seq, op, name):  # noqa: F811
    a = good(seq)
    a["batch"].rows = 0
    setattr(a["batch"], name, None)
    with pytest.raises(ValueError, match="null"):
        call(seq, op, a)


@pytest.mark.parametrize("op", ["rotary", "append"])
def test_frequencies_of_no_rows_may_be_null(seq, op):  # noqa: F811
    a = good(seq)
    a["rotation"].freq = a["rotation"].pos = None
    with pytest.raises(ValueError, match="freq"):
        call(seq, op, a)
    a["rows"] = a["batch"].rows = 0
    with pytest.raises(RuntimeError, match="device"):
        call(seq, op, a)


@pytest.mark.parametrize("op", ["rotary", "append"])
def test_negative_stride_of_positions(seq, op):  # noqa: F811
    """As those of tensors and tables."""
    a = good(seq)
    a["rotation"].pos_stride = -5
    with pytest.raises(ValueError, match="stride"):
        call(seq, op, a)
