"""Host side of the operators beside the softmax at the edges of what they accept."""
import contextlib
import glob
import os
import re
import resource
import subprocess

import pytest

import causal_softmax as cs
from causal_softmax import operators as ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rows_of_a_group_up_to_the_largest_matrix(tmp_path):
    """The kernels' own cursor, compiled as C++: a signed one passes 2^31 - 1 and never ends."""
    exe = str(tmp_path / "turns_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                    os.path.join(cs.PKG_DIR, "csrc"), "-o", exe, os.path.join(ROOT, "tests", "turns_check.cpp")],
                   check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout + out.stderr


VECTORS = r"reinterpret_cast<(?:const )?(?:float2|float4|uint2|uint4|double2)\*>\(&?(\w+)\["


def test_shared_arrays_read_as_vectors_are_declared_aligned():
    """A neighbour's size would otherwise decide whether a vector access of a float array is aligned."""
    found = 0
    for path in sorted(glob.glob(os.path.join(cs.PKG_DIR, "csrc", "kernels", "*.cuh"))):
        with open(path, encoding="utf-8") as fh:
            text = fh.read()
        shared = {}
        for declaration in re.findall(r"__shared__([^;]*);", text):
            for name in re.findall(r"(\w+)\s*\[", re.sub(r"\[[^\]]*\]", "[", declaration)):
                shared[name] = "__align__(16)" in declaration
        for name in set(re.findall(VECTORS, text)) & set(shared):
            assert shared[name], f"{os.path.basename(path)}: {name}"
            found += 1
    assert found >= 2


def test_whole_numbers_are_not_cut_down_to_whole_ones():
    for v in (3.5, -0.25, 2.0 ** 31, float("nan"), float("inf"), 2 ** 31):
        with pytest.raises(ValueError):
            ops._int("window", v)
    assert [ops._int("window", v) for v in (3, 3.0, -5, 2 ** 31 - 1, True)] == [3, 3, -5, 2 ** 31 - 1, 1]


def test_bucket_starts_are_not_taken_modulo_2_to_the_32():
    assert list(ops._starts_array((0, 1, 8192))) == [0, 1, 8192]
    for starts in ((0, 1, 2 ** 32 + 2), (2 ** 32, 1), (0, -2 ** 32 + 5), (0, 1.5)):
        with pytest.raises((TypeError, ValueError)):
            ops._starts_array(starts)


def test_bucket_counts_that_are_refused_cost_no_memory():
    before = resource.getrusage(resource.RUSAGE_SELF).ru_maxrss
    for buckets in (2 ** 28, 2 ** 31 - 1):
        with pytest.raises(cs.CausalSoftmaxError):
            cs.bias_buckets(buckets, 8000)
    with pytest.raises(ValueError):
        cs.bias_buckets(2 ** 40, 8000)
    assert resource.getrusage(resource.RUSAGE_SELF).ru_maxrss - before < 1 << 18  # KB


@pytest.mark.parametrize("device,want", [(None, 1), ("cuda", 1), ("cuda:0", 0), (0, 0), (2, 2)])
def test_status_of_the_current_device_unless_one_is_named(monkeypatch, device, want):
    seen = []

    class Library:
        def cs_attention_status(self, bits, stream):
            return 0

    monkeypatch.setattr(ops.torch.cuda, "current_device", lambda: 1)
    monkeypatch.setattr(ops, "lib", Library)
    monkeypatch.setattr(ops, "_on", lambda d, stream: seen.append(d) or contextlib.nullcontext())
    monkeypatch.setattr(ops, "_current", lambda d: 0)
    assert ops.attention_status(device=device) == (0, 0)
    assert [d.index for d in seen] == [want]
