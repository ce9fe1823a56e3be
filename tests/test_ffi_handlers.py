"""The XLA handlers of the sequence operators, compiled against a stand-in for jax's header, with the C entry points replaced by ones that write
down what they get: every buffer is checked for its type and all of its dimensions before an address goes on."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "colabfold-cuda-kernels_b200", "csrc")
pytestmark = pytest.mark.skipif(not shutil.which("g++") or not os.path.isdir("/usr/local/cuda/include"), reason="needs a host compiler and CUDA's headers")


@pytest.fixture(scope="module")
def call(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("handlers") / "handlers")
    fake = os.path.join(HERE, "fake_xla")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-x", "c++", "-I", fake, "-I", CSRC, "-I", "/usr/local/cuda/include", os.path.join(fake, "handlers.cpp"), "-o", exe], check=True)

    def run(*what):
        return subprocess.run([exe, *what], check=True, capture_output=True, text=True).stdout.strip()

    return run


def test_what_fits_is_passed_on(call):
    rows = {"q": " rows(4 256 64 0)", "k": " rows(2 128 64 0)"}
    turn, cache, batch = " rotation(64 2 %d 20 12 6)", " cache(10 16 2 64)", " batch(3 6 3 70 5 5)"
    assert call("rotary", "-", "-") == "called" + turn % 1 + " 6 64" + rows["q"] * 2 + " 1"
    assert call("append", "-", "-") == "called" + cache + batch + rows["k"] * 2 + turn % 0 + rows["q"] * 2
    assert call("attention", "-", "-") == "called" + cache + batch + rows["q"] * 2 + " 0.125000 1 7 4096"


# buffers of 8-bit codes may come in any 8-bit type and shape
@pytest.mark.parametrize("target, name, what", [("append", "kc", "s8"), ("attention", "vc", "f8"), ("attention", "kc", "20x1024"), ("attention", "ws", "f32")])
def test_fine_too(call, target, name, what):
    assert call(target, name, what).startswith("called")


OUTPUTS = [("rotary", "y"), ("append", "out"), ("attention", "out")]
REFUSED = (
    [(t, n, d) for t, n in OUTPUTS for d in ("3x4x128", "6x2x128", "6x8x32", "6x4x64x1", "1536", "12x4x32")]  # as many elements as the input
    + [(t, "freq", d) for t in ("rotary", "append") for d in ("bf16", "f16", "f64", "s32", "32x1", "4x8")]
    + [(t, "pos", d) for t in ("rotary", "append") for d in ("s64", "f32", "6x2", "12", "2x7", "2x6x1", "1x12")]
    + [("rotary", "section", "10x10x12"), ("append", "section", "32"), ("rotary", "x", "7x4x64")]
    + [(t, n, d) for t in ("append", "attention") for n in ("ks", "vs") for d in ("bf16", "f64", "20", "2x10", "5x4", "10x2x1")]
    + [(t, n, d) for t in ("append", "attention") for n in ("kc", "vc") for d in ("bf16", "f32", "10x2x16x32", "10x2x16x65")]
    + [(t, n, "s64") for t in ("append", "attention") for n in ("first", "len", "table")]
    + [(t, n, d) for t in ("append", "attention") for n, d in (("first", "3"), ("first", "4x1"), ("len", "4"), ("len", "1x3"), ("table", "15"), ("table", "5x3"), ("table", "3x5x1"))]
    + [("attention", "lse", d) for d in ("bf16", "f64", "24", "4x6", "6x4x1")]
    + [("append", n, d) for n, d in (("v", "12x1x64"), ("v", "6x4x32"), ("k", "6x2x32"), ("q", "6x4x32"), ("q", "7x4x64"), ("kc_out", "10x2x16x32"), ("ks_out", "20"))]
    + [("attention", "q", "6x4x32")]
)


@pytest.mark.parametrize("target, name, what", REFUSED)
def test_what_does_not_fit_is_refused(call, target, name, what):
    answer = call(target, name, what)
    assert answer.startswith("refused Cck") and "AFTER" not in answer


@pytest.mark.parametrize(
    "target, name, what, field",
    [("rotary", "x+y", "6x%dx64" % (2**32 + 4), " rows(-1 "), ("attention", "q+out", "6x4x%d" % (2**32 + 64), "refused"), ("rotary", "section", "%dx12" % (2**32 + 20), " 2 1 -1 12 6)"),
     ("append", "k+v", "6x%dx64" % (2**32 + 2), " rows(-1 "), ("append", "kc+vc+kc_out+vc_out", "10x2x16x%d" % (2**32 + 64), "refused")],
)  # fmt: skip
def test_sizes_past_32_bits(call, target, name, what, field):
    """They are refused, or reach the C entry points as -1, which those refuse: not cut to fit."""
    assert field in call(target, name, what)
