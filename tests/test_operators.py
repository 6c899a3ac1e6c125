"""Host side of the operators beside the softmax: bucket borders, the positional
mask's arithmetic, and every refusal, which comes before any use of a GPU."""
import ctypes
import os
import subprocess

import pytest

import causal_softmax as cs
from causal_softmax import operators as ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 1 << 20  # a 16-byte aligned address that nothing reads


@pytest.fixture(scope="module", autouse=True)
def built():
    import build

    build.build_library()


def plain_starts(buckets, max_distance):
    e = buckets // 2
    m = buckets - e
    starts = list(range(e))
    for t in range(m):
        n = starts[-1] + 1
        while n ** m < max_distance ** t * e ** (m - t):
            n += 1
        starts.append(n)
    return tuple(starts)


@pytest.mark.parametrize("buckets", [2, 3, 16, 32, 33, 64, 128])
@pytest.mark.parametrize("max_distance", [65, 128, 200, 1024, 8000])
def test_bucket_borders(buckets, max_distance):
    assert cs.bias_buckets(buckets, max_distance) == plain_starts(buckets, max_distance)


def test_bucket_borders_that_are_exact_roots():
    # 16 buckets for distances 16..256 by the ratio 2^(1/4): every fourth border is a power of two.
    assert cs.bias_buckets(32, 256)[16::4] == (16, 32, 64, 128)


@pytest.mark.parametrize("buckets,max_distance", [(1, 8), (0, 8), (129, 8000), (32, 16), (32, 8193), (-4, 8)])
def test_bucket_refusals(buckets, max_distance):
    with pytest.raises(cs.CausalSoftmaxError):
        cs.bias_buckets(buckets, max_distance)


def test_positions_by_brute_force(tmp_path):
    exe = str(tmp_path / "positions_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                    os.path.join(cs.PKG_DIR, "csrc"), "-o", exe, os.path.join(ROOT, "tests", "positions_check.cpp")],
                   check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout + out.stderr


def test_division_by_brute_force(tmp_path):
    exe = str(tmp_path / "divider_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                    os.path.join(cs.PKG_DIR, "csrc"), "-o", exe, os.path.join(ROOT, "tests", "divider_check.cpp")],
                   check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout + out.stderr


def bias_args(starts=(0, 1, 2, 3), **kw):
    array = (ctypes.c_int32 * max(1, len(starts)))(*starts)
    f = dict(type=0, batch=1, heads=2, rows=8, cols=8, pitch=8, row_offset=0, window=0, sinks=0, buckets=len(starts),
             bucket_starts=ctypes.addressof(array), scale=1.0)
    f.update(kw)
    a = ops._BiasArgs(**f)
    a.keep = array
    return a


@pytest.mark.parametrize("change,code", [
    (dict(type=2), "ARG"), (dict(batch=0), "EMPTY"), (dict(heads=-1), "EMPTY"), (dict(rows=0), "EMPTY"),
    (dict(cols=0), "EMPTY"), (dict(pitch=7), "PITCH"), (dict(cols=9), "PITCH"), (dict(pitch=12), "PITCH"),
    (dict(row_offset=-1), "WRONG_LENGTH"), (dict(row_offset=2**31 - 8), "WRONG_LENGTH"),
    (dict(batch=2**31 - 1, heads=2**31 - 1, rows=2**31 - 1), "WRONG_LENGTH"),
    (dict(window=-1), "ARG"), (dict(sinks=-1), "ARG"), (dict(scale=-1.0), "BAD_SCALE"),
    (dict(scale=float("nan")), "BAD_SCALE"), (dict(scale=2e30), "BAD_SCALE"), (dict(buckets=0), "ARG"),
    (dict(buckets=129), "ARG"), (dict(bucket_starts=None), "NULL"), (dict(starts=(1, 2)), "ARG"),
    (dict(starts=(0, 2, 2)), "ARG"), (dict(starts=(0, 8193)), "ARG"),
])
def test_bias_refusals(change, code):
    L, a = cs.lib(), bias_args(**change)
    ref, work = ctypes.byref(a), L.cs_bias_softmax_backward_workspace
    assert cs.ERR[L.cs_bias_softmax(ref, FAKE, FAKE, 2 * FAKE, None)] == code
    assert cs.ERR[L.cs_bias_softmax_backward(ref, FAKE, 2 * FAKE, 3 * FAKE, FAKE, FAKE, 1 << 20, None)] == code
    assert cs.ERR[work(ref)] == code
    assert L.cs_last_error_detail()


def test_bias_pointer_refusals():
    L, a = cs.lib(), bias_args()
    ref = ctypes.byref(a)

    def forward(x, table, p):
        return cs.ERR[L.cs_bias_softmax(ref, x, table, p, None)]

    def backward(p, dp, ds, dtable, work, size=1 << 20):
        return cs.ERR[L.cs_bias_softmax_backward(ref, p, dp, ds, dtable, work, size, None)]

    assert forward(None, FAKE, 2 * FAKE) == "NULL" and forward(FAKE, None, 2 * FAKE) == "NULL"
    assert forward(FAKE, FAKE, None) == "NULL" and forward(FAKE + 8, FAKE, 2 * FAKE) == "ALIGNMENT"
    assert forward(FAKE, 4 * FAKE, FAKE) == "ARG" and forward(FAKE, 4 * FAKE, FAKE + 128) == "ARG"
    assert backward(FAKE, 2 * FAKE, 2 * FAKE, FAKE, FAKE) == "ARG"
    assert backward(FAKE, 2 * FAKE, 3 * FAKE, None, FAKE) == "NULL"
    assert backward(FAKE, 2 * FAKE, 3 * FAKE, FAKE, None) == "NULL"
    assert backward(FAKE, 2 * FAKE, 3 * FAKE, FAKE, FAKE + 4) == "ALIGNMENT"
    assert cs.ERR[L.cs_bias_softmax(None, FAKE, FAKE, 2 * FAKE, None)] == "NULL"


def attention_args(**kw):
    def tensor(heads, data=FAKE):
        return ops._Tensor(data, 16 * heads * 64, heads * 64, 64)

    f = dict(type=1, batch=2, heads=4, kv_heads=2, head_dim=64, q_len=16, kv_len=16, window=0, sinks=0, scale=0.125,
             q_lens=None, kv_lens=None, q=tensor(4), k=tensor(2), v=tensor(2), o=tensor(4), lse=FAKE)
    f.update(kw)
    return ops._AttentionArgs(**f)


def t(data=FAKE, batch=4096, token=256, head=64):
    return ops._Tensor(data, batch, token, head)


@pytest.mark.parametrize("change,code", [
    (dict(type=7), "ARG"), (dict(batch=0), "EMPTY"), (dict(heads=0), "EMPTY"), (dict(kv_heads=0), "EMPTY"),
    (dict(head_dim=0), "EMPTY"), (dict(q_len=0), "EMPTY"), (dict(kv_len=0), "EMPTY"), (dict(kv_heads=3), "ARG"),
    (dict(head_dim=60), "UNSUPPORTED"), (dict(head_dim=136), "UNSUPPORTED"), (dict(batch=1 << 19), "WRONG_LENGTH"),
    (dict(q_len=2**31 - 1), "WRONG_LENGTH"), (dict(kv_len=2**31 - 1), "WRONG_LENGTH"), (dict(window=-1), "ARG"),
    (dict(sinks=-2), "ARG"), (dict(scale=-0.1), "BAD_SCALE"), (dict(scale=1025.0), "BAD_SCALE"),
    (dict(scale=float("inf")), "BAD_SCALE"), (dict(q=t(data=None)), "NULL"), (dict(k=t(data=FAKE + 2)), "ALIGNMENT"),
    (dict(v=t(token=0)), "PITCH"), (dict(v=t(token=132)), "PITCH"), (dict(q=t(head=32)), "PITCH"),
    (dict(o=t(batch=-4096)), "PITCH"), (dict(k=t(token=1 << 38)), "PITCH"),
])
def test_attention_refusals(change, code):
    L, a = cs.lib(), attention_args(**change)
    ref, grads = ctypes.byref(a), ops._AttentionGrads(t(), t(), t(token=128), t(token=128))
    assert cs.ERR[L.cs_attention(ref, FAKE, 1 << 30, None)] == code
    assert cs.ERR[L.cs_attention_workspace(ref)] == code
    assert cs.ERR[L.cs_attention_backward(ref, ctypes.byref(grads), FAKE, 1 << 30, None)] == code
    assert cs.ERR[L.cs_attention_backward_workspace(ref)] == code
    assert L.cs_last_error_detail()


def test_attention_backward_refusals():
    L, good = cs.lib(), attention_args()

    def call(a=good, work=FAKE, size=1 << 30, **kw):
        g = dict(d_o=t(), dq=t(), dk=t(token=128), dv=t(token=128))
        g.update(kw)
        return cs.ERR[L.cs_attention_backward(ctypes.byref(a), ctypes.byref(ops._AttentionGrads(**g)), work, size, None)]

    assert call(a=attention_args(lse=None)) == "NULL"
    assert call(d_o=t(data=None)) == "NULL" and call(dk=t(data=FAKE + 8, token=128)) == "ALIGNMENT"
    assert call(dv=t(token=4)) == "PITCH" and call(dq=t(head=60)) == "PITCH"
    assert call(work=None) == "NULL" and call(work=FAKE + 4) == "ALIGNMENT" and call(size=3) == "WRONG_LENGTH"
    assert cs.ERR[L.cs_attention_backward(ctypes.byref(good), None, FAKE, 1 << 30, None)] == "NULL"
    assert cs.ERR[L.cs_attention_status(None, None)] == "NULL"


def test_refusals_of_overlaps_and_misaligned_words():
    L = cs.lib()

    def forward(**kw):
        return cs.ERR[L.cs_attention(ctypes.byref(attention_args(**kw)), FAKE, 1 << 30, None)]

    def backward(lse=FAKE, **kw):
        g = dict(d_o=t(), dq=t(2 * FAKE), dk=t(3 * FAKE, token=128), dv=t(4 * FAKE, token=128))
        g.update(kw)
        return cs.ERR[L.cs_attention_backward(ctypes.byref(attention_args(lse=lse)), ctypes.byref(ops._AttentionGrads(**g)),
                                              FAKE, 1 << 30, None)]

    assert forward(o=t()) == "ARG"
    for words in (dict(lse=FAKE + 2), dict(q_lens=FAKE + 1), dict(kv_lens=FAKE + 2)):
        assert forward(o=t(2 * FAKE), **words) == "ALIGNMENT"
    assert backward(dq=t()) == "ARG" and backward(dk=t(2 * FAKE, token=128)) == "ARG"
    assert backward(dv=t(3 * FAKE, token=128)) == "ARG" and backward(lse=FAKE + 2) == "ALIGNMENT"
    a = bias_args()
    assert cs.ERR[L.cs_bias_softmax(ctypes.byref(a), FAKE, FAKE + 2, 2 * FAKE, None)] == "ALIGNMENT"
    assert cs.ERR[L.cs_bias_softmax_backward(ctypes.byref(a), FAKE, 2 * FAKE, 3 * FAKE, FAKE + 2, FAKE, 1 << 20,
                                             None)] == "ALIGNMENT"
