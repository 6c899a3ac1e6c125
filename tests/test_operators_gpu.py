"""GPU tests of the operators beside the softmax against plain 64-bit forms
(attention_ref.py, where the bounds are derived): lengths from one token on,
odd sizes, strides, masks that leave rows empty, infinities and NaN where
nothing is seen, other streams, and calls captured into a graph."""
import math

import pytest
import torch

import attention_ref as ref
import causal_softmax as cs

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def randn(*shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def within(got, want, bound, what):
    got = got.double()
    same = torch.isneginf(got) & torch.isneginf(want)
    over = ((got - want).abs() - bound).masked_fill(same, -1.0)
    assert not torch.isnan(over).any(), f"{what}: NaN"
    assert (over <= 0).all(), f"{what}: {float(over.max()):.3g} over its bound at {over.argmax().item()} of {tuple(got.shape)}"


# ---------------------------------------------------------------- biased softmax

BIAS = [
    # batch, heads, rows, cols, row_offset, window, sinks, buckets, max_distance
    (1, 1, 1, 1, 0, 0, 0, 32, 128),
    (2, 3, 37, 37, 0, 0, 0, 16, 64),
    (1, 2, 64, 129, 65, 0, 0, 32, 128),
    (2, 2, 100, 75, 0, 0, 0, 32, 128),      # rows beyond the columns
    (1, 2, 90, 33, 0, 5, 0, 32, 128),       # and windows that have left them: empty rows
    (1, 2, 90, 33, 3, 5, 3, 32, 128),
    (2, 2, 257, 257, 0, 16, 4, 32, 128),
    (1, 3, 200, 1037, 837, 300, 9, 64, 1024),
    (1, 2, 33, 2100, 2067, 0, 0, 32, 128),   # one vector more than 8 a lane
    (1, 1, 40, 4100, 4060, 0, 0, 128, 8000),
    (1, 1, 5, 9001, 8996, 0, 0, 32, 4096),
    (1, 1, 3, 34000, 33997, 0, 0, 32, 128),  # several warps a row
    (1, 1, 2, 70001, 69999, 0, 0, 2, 128),   # in chunks
    (1, 1, 3, 40000, 39997, 20000, 100, 32, 512),
]


def bias_inputs(case, dtype, seed=1):
    batch, heads, rows, cols, row_offset, window, sinks, nb, md = case
    pitch = cs.padded_pitch(cols) + (8 if rows % 2 else 0)
    starts = cs.bias_buckets(nb, md)
    how = dict(cols=cols, scale=0.3, row_offset=row_offset, window=window, sinks=sinks)
    x = randn(batch, heads, rows, pitch, dtype=dtype, seed=seed, scale=8.0)
    table = randn(heads, nb, dtype=torch.float32, seed=seed + 1)
    return x, table, starts, how


def hide(x, how, value):
    """x with `value` wherever a row sees nothing."""
    pos = torch.arange(x.shape[2], device="cuda") + how["row_offset"]
    keep = torch.zeros(x.shape[2:], dtype=torch.bool, device="cuda")
    keep[:, :how["cols"]] = ref.mask(pos, how["cols"], how["window"], how["sinks"])
    return torch.where(keep, x, torch.tensor(value, dtype=x.dtype, device="cuda"))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", BIAS)
def test_bias_softmax(case, dtype):
    x, table, starts, how = bias_inputs(case, dtype)
    got = cs.bias_softmax(hide(x, how, math.nan), table, starts, **how)
    want, bound = ref.bias_softmax(x, table, starts, **how)
    within(got, want, bound, "p")
    zero = got.view(torch.int16)[want == 0]
    assert (hide(got, how, 0.0).view(torch.int16) == got.view(torch.int16)).all(), "masked columns are +0.0"
    assert not (zero < 0).any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", BIAS)
def test_bias_softmax_backward(case, dtype):
    x, table, starts, how = bias_inputs(case, dtype)
    p = ref.bias_softmax(x, table, starts, **how)[0].to(dtype)
    dp = randn(*x.shape, dtype=dtype, seed=7)
    ds, dtable = cs.bias_softmax_backward(hide(p, how, math.inf), hide(dp, how, math.nan), starts, **how)
    want, bound, wt, bt = ref.bias_backward(p, dp, starts, len(starts), **how)
    within(ds, want, bound, "ds")
    within(dtable, wt, bt, "dtable")
    assert (hide(ds, how, 0.0).view(torch.int16) == ds.view(torch.int16)).all()
    again = cs.bias_softmax_backward(p, dp, starts, **how)
    assert torch.equal(again[0], ds) and torch.equal(again[1], dtable), "the same inputs give the same bits"


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", [
    (8, 16, 300, 300, 0, 0, 0, 32, 128),
    (4, 8, 400, 2500, 2100, 0, 0, 32, 128),
    (4, 8, 400, 2500, 2300, 700, 9, 64, 512),  # the last rows are beyond the columns
    (450, 1, 2, 120000, 119998, 0, 0, 32, 128),  # rows that stay in global memory
    (40, 16, 120, 120, 0, 0, 0, 32, 128),  # short rows, and many
    (40, 16, 120, 700, 590, 60, 4, 16, 64),
])
def test_bias_several_rows_a_group(case, dtype):
    """Matrices enough that a group of lanes works on several rows, one after the other."""
    test_bias_softmax(case, dtype)
    torch.cuda.empty_cache()
    test_bias_softmax_backward(case, dtype)
    torch.cuda.empty_cache()


def test_bias_of_more_than_2_to_the_31_elements():
    """The last matrix of a batch as if it were alone, bit for bit."""
    x, dp = (torch.empty(130, 1, 4096, 4096, dtype=F16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(n))
             for n in (1, 2))
    starts, table = cs.bias_buckets(32, 128), randn(1, 32, dtype=torch.float32, seed=3)
    how = dict(cols=4096, scale=0.3, window=900, sinks=3)
    p = cs.bias_softmax(x, table, starts, **how)
    alone = cs.bias_softmax(x[-1:], table, starts, **how)
    assert torch.equal(p[-1:], alone) and float(alone.sum()) > 4000
    ds = cs.bias_softmax_backward(p, dp, starts, **how)[0]
    assert torch.equal(ds[-1:], cs.bias_softmax_backward(alone, dp[-1:], starts, **how)[0])
    del x, dp, p, ds
    torch.cuda.empty_cache()


def test_bias_infinities_in_seen_places():
    x, table, starts, how = bias_inputs((1, 1, 40, 40, 0, 0, 0, 32, 128), F16)
    x[0, 0, 3, :] = -math.inf       # a row of -infinity only: zeros
    x[0, 0, 5, :3] = -math.inf
    x[0, 0, 7, :] = -65504.0        # the type's lowest value everywhere
    x[0, 0, 9, 2] = math.nan
    got = cs.bias_softmax(x, table, starts, **how)[0, 0].double()
    y = x.clone()
    y[0, 0, 9, 2] = 0
    want, bound = ref.bias_softmax(y, table, starts, **how)
    for row in (3, 5, 7, 8, 10):
        within(got[row], want[0, 0, row], bound[0, 0, row], f"row {row}")
    assert (got[3] == 0).all() and torch.isnan(got[9, :10]).all() and (got[9, 10:] == 0).all()


def test_bias_large_scale_and_custom_buckets():
    x = randn(1, 2, 24, 24, dtype=F16, seed=3)
    x[..., :2] = 4.0
    table = torch.zeros(2, 3, device="cuda")
    got = cs.bias_softmax(x, table, (0, 5, 11), cols=24, scale=1e30)
    assert (got[..., 1:, :2] == 0.5).all() and (got[..., 2:] == 0).all()
    how = dict(cols=24, scale=0.5)
    table = randn(2, 3, dtype=torch.float32, seed=4)
    want, bound = ref.bias_softmax(x, table, (0, 5, 11), **how)
    within(cs.bias_softmax(x, table, [0, 5, 11], **how), want, bound, "p")
    want, bound = ref.bias_softmax(x, table[:, :1].contiguous(), (0,), **how)
    within(cs.bias_softmax(x, table[:, :1].contiguous(), (0,), **how), want, bound, "one bucket")


def test_bias_gradients_against_differences():
    x, table, starts, how = bias_inputs((1, 2, 20, 20, 0, 9, 2, 8, 12), BF16)
    w = randn(*x.shape, dtype=BF16, seed=9)

    def loss(x, table):
        return float((ref.bias_softmax(x, table, starts, **how)[0] * w.double()).sum())

    p = cs.bias_softmax(x, table, starts, **how)
    ds, dtable = cs.bias_softmax_backward(p, w, starts, **how)
    for seed in range(3):
        dx, dt = randn(*x.shape, dtype=torch.float64, seed=20 + seed), randn(*table.shape, dtype=torch.float64, seed=30 + seed)
        h = 1e-5
        slope = (loss(x.double() + h * dx, table.double() + h * dt) - loss(x.double() - h * dx, table.double() - h * dt)) / (2 * h)
        got = float((ds.double() * dx).sum() + (dtable.double() * dt).sum())
        # p and ds are rounded to bf16 (2^-9 of each), some 800 terms of a standard normal direction.
        size = float((ds.double() * dx).abs().sum() + (dtable.double() * dt).abs().sum())
        assert abs(got - slope) <= 4 * 2 ** -8 * size, (got, slope)


# ---------------------------------------------------------------- attention

ATTENTION = [
    # batch, q_len, kv_len, heads, kv_heads, dim, window, sinks
    (1, 1, 1, 1, 1, 64, 0, 0),
    (2, 1, 300, 8, 8, 64, 0, 0),
    (2, 1, 300, 8, 2, 128, 100, 4),
    (1, 1, 2000, 32, 1, 128, 0, 0),
    (3, 1, 130, 12, 4, 80, 16, 1),
    (1, 3, 515, 8, 2, 128, 0, 0),
    (2, 7, 700, 6, 3, 64, 64, 2),
    (1, 17, 65, 4, 1, 32, 0, 0),
    (2, 64, 64, 2, 2, 64, 0, 0),
    (1, 127, 127, 3, 3, 128, 0, 0),
    (1, 129, 129, 4, 2, 128, 1, 0),          # each query sees itself
    (2, 300, 300, 4, 1, 64, 50, 4),
    (1, 257, 1000, 4, 2, 128, 0, 0),          # a chunk over a cache
    (1, 260, 900, 2, 1, 128, 130, 7),
    (1, 400, 60, 2, 2, 64, 0, 0),             # queries before the first key see nothing
    (2, 333, 333, 4, 4, 96, 128, 128),
    (1, 513, 513, 2, 1, 8, 200, 300),          # more sinks than window
    (1, 1025, 1025, 2, 2, 120, 0, 0),
    (1, 640, 640, 2, 1, 128, 256, 1),
    (1, 18, 3000, 16, 2, 128, 0, 0),           # few queries of many heads: shared tiles, split keys
    (2, 40, 2500, 12, 1, 64, 1500, 5),
    (1, 33, 700, 64, 1, 16, 0, 0),
    (2, 150, 150, 24, 2, 64, 60, 2),           # groups of 12: packs of 4
]


def attention_inputs(case, dtype, seed=1):
    batch, q_len, kv_len, heads, kv_heads, dim, window, sinks = case
    q = randn(batch, q_len, heads, dim, dtype=dtype, seed=seed)
    k, v = (randn(batch, kv_len, kv_heads, dim, dtype=dtype, seed=seed + i) for i in (1, 2))
    return q, k, v, dict(scale=dim ** -0.5, window=window, sinks=sinks)


def status_ok():
    assert cs.attention_status() == (0, 0)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", ATTENTION)
def test_attention(case, dtype):
    q, k, v, how = attention_inputs(case, dtype)
    out, lse = cs.attention(q, k, v, return_lse=True, **how)
    status_ok()
    want, bound, wl, bl = ref.attention(q, k, v, **how)
    within(out, want, bound, "out")
    within(lse, wl, bl, "lse")
    again = cs.attention(q, k, v, **how)
    assert torch.equal(again, out), "the same inputs give the same bits"


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", ATTENTION)
def test_attention_backward(case, dtype):
    q, k, v, how = attention_inputs(case, dtype)
    dout = randn(*q.shape, dtype=dtype, seed=8)
    out, lse = cs.attention(q, k, v, return_lse=True, **how)
    got = cs.attention_backward(dout, q, k, v, out, lse, **how)
    status_ok()
    want = ref.attention_backward(dout, q, k, v, **how)
    for n, t in zip(("dq", "dk", "dv"), got):
        within(t, *want[n], n)
    again = cs.attention_backward(dout, q, k, v, out, lse, **how)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


RAGGED = [
    # q_lens, kv_lens of q_len x kv_len
    (200, 200, (200, 0, 131, 1), (200, 0, 131, 1)),
    (200, 520, (200, 64, 200, 3), (520, 64, 300, 150)),   # the last one: more queries than are used
    (1, 700, (1, 1, 1, 0), (700, 1, 333, 0)),
    (1, 700, (1, 1, 1, 1), (0, 129, 128, 512)),             # a sequence without keys
    (9, 300, (9, 2, 9, 9), (300, 2, 5, 64)),                # fewer keys than queries
    (150, 90, (150, 10, 999, -5), (90, 90, 2000, 7)),        # lengths beyond the tensors are clipped
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
@pytest.mark.parametrize("q_len,kv_len,q_lens,kv_lens", RAGGED)
def test_ragged_batch_with_garbage_behind_the_sequences(q_len, kv_len, q_lens, kv_lens, window, sinks, dtype):
    q, k, v, how = attention_inputs((4, q_len, kv_len, 4, 2, 64, window, sinks), dtype)
    dout = randn(*q.shape, dtype=dtype, seed=8)
    dev = dict(q_lens=torch.tensor(q_lens, dtype=torch.int32, device="cuda"),
               kv_lens=torch.tensor(kv_lens, dtype=torch.int32, device="cuda"))
    for b in range(4):
        nq, nk = min(max(q_lens[b], 0), q_len), min(max(kv_lens[b], 0), kv_len)
        k[b, nk:], v[b, nk:], q[b, nq:], dout[b, nq:] = math.nan, math.inf, math.nan, math.nan
        first = nk - nq - window + 1  # what no query sees any more
        if window and first > sinks:
            k[b, sinks:first], v[b, sinks:first] = math.inf, math.nan
    want, bound, wl, bl = ref.attention(q, k, v, **how, **dev)
    out = torch.full_like(q, 7.0)
    got, lse = cs.attention(q, k, v, out=out, return_lse=True, **how, **dev)
    assert got is out
    within(out, want, bound, "out")
    within(lse, wl, bl, "lse")
    grads = cs.attention_backward(dout, q, k, v, out, lse, **how, **dev)
    status_ok()
    want = ref.attention_backward(dout, q, k, v, **how, **dev)
    for n, t in zip(("dq", "dk", "dv"), grads):
        within(t, *want[n], n)
        for b in range(4):  # (a row inside may have the exact gradient 0 and be off by its bound)
            rows = min(max((q_lens if n == "dq" else kv_lens)[b], 0), t.shape[1])
            assert (t[b, rows:] == 0).all(), f"{n}: rows outside the sequences are zero"


SPLIT = [
    # calls whose keys several CTAs share, or whose few rows are tiles; kv_lens
    (1, 24, 700, 2, 1, 128, 0, 0, (650,)),               # a CTA per key tile
    (1, 40, 1100, 4, 2, 64, 900, 130, (1100,)),
    (2, 30, 6000, 3, 1, 80, 0, 0, (6000, 40)),           # most CTAs of a tile see no key
    (1, 20, 40000, 1, 1, 64, 0, 0, (39000,)),            # more than 64 CTAs a tile
    (1, 500, 2500, 2, 2, 128, 2100, 3, (2400,)),
    (75, 3, 200, 8, 2, 64, 0, 0, tuple(range(1, 151, 2))),  # 12 rows of 150 kv heads
    (3, 2, 5000, 16, 2, 128, 4000, 9, (5000, 130, 1)),   # 16 rows, split
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", SPLIT)
def test_split_keys(case, dtype):
    *case, kv_lens = case
    q, k, v, how = attention_inputs(case, dtype)
    how["kv_lens"] = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
    for b, n in enumerate(kv_lens):
        k[b, n:], v[b, n:] = math.inf, math.nan
    got, lse = cs.attention(q, k, v, return_lse=True, **how)
    status_ok()
    want, bound, wl, bl = ref.attention(q, k, v, **how)
    within(got, want, bound, "out")
    within(lse, wl, bl, "lse")
    assert torch.equal(cs.attention(q, k, v, **how), got)


@pytest.mark.parametrize("q_len,kv_len", [(1, 200), (190, 200)])
def test_strides(q_len, kv_len):
    """Heads before tokens, tokens apart, and one tensor that holds q, k and v."""
    b, h, d = 2, 4, 64
    how = dict(window=70, sinks=2)
    q0, k0, v0 = (randn(b, n, h, d, dtype=BF16, seed=i) for i, n in ((1, q_len), (2, kv_len), (3, kv_len)))
    dout0 = randn(b, q_len, h, d, dtype=BF16, seed=4)
    out0, lse0 = cs.attention(q0, k0, v0, return_lse=True, **how)
    grads0 = cs.attention_backward(dout0, q0, k0, v0, out0, lse0, **how)
    packed = torch.zeros(b, kv_len, 3, h + 1, d + 8, dtype=BF16, device="cuda")
    packed[:, :q_len, 0, :h, :d], packed[:, :, 1, 1:, 8:], packed[:, :, 2, :h, :d] = q0, k0, v0
    forms = [
        (packed[:, :q_len, 0, :h, :d], packed[:, :, 1, 1:, 8:], packed[:, :, 2, :h, :d]),
        tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q0, k0, v0)),
        tuple(t.permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3) for t in (q0, k0, v0)),
    ]
    for q, k, v in forms:
        buf = torch.full((b, h, q_len, d + 8), 3.0, dtype=BF16, device="cuda")
        out = buf[..., :d].transpose(1, 2)
        _, lse = cs.attention(q, k, v, out=out, return_lse=True, **how)
        assert torch.equal(out, out0) and torch.equal(lse, lse0)
        assert (buf[..., d:] == 3.0).all()
        dout = dout0.transpose(1, 2).contiguous().transpose(1, 2)
        for a, w in zip(cs.attention_backward(dout, q, k, v, out, lse, **how), grads0):
            assert torch.equal(a, w)
    status_ok()


def test_one_token_equals_the_prompts_last_row():
    q, k, v, how = attention_inputs((2, 333, 333, 8, 2, 128, 100, 4), BF16)
    whole, whole_lse = cs.attention(q, k, v, return_lse=True, **how)
    one, lse = cs.attention(q[:, -1:], k, v, return_lse=True, **how)
    want, bound, wl, bl = ref.attention(q, k, v, **how)
    for got, got_lse in ((whole[:, -1:], whole_lse[..., -1:]), (one, lse)):
        within(got, want[:, -1:], bound[:, -1:], "last row")
        within(got_lse, wl[..., -1:], bl[..., -1:], "lse")


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_extreme_magnitudes(dtype):
    """Scores in the thousands, far-off keys, zero scale, small and large gradients."""
    q, k, v, how = attention_inputs((1, 200, 200, 2, 1, 64, 0, 0), dtype)
    for factor, scale in ((8.0, 1.0), (1.0, 0.0), (1e-3, 1.0), (30.0, 0.125)):
        qs, hs = (q * factor).to(dtype), dict(how, scale=scale)
        out, lse = cs.attention(qs, k, v, return_lse=True, **hs)
        want, bound, wl, bl = ref.attention(qs, k, v, **hs)
        within(out, want, bound, f"out {factor} {scale}")
        within(lse, wl, bl, "lse")
        for size in (1e-4, 1.0, 300.0):
            dout = randn(*q.shape, dtype=dtype, seed=8, scale=size)
            got = cs.attention_backward(dout, qs, k, v, out, lse, **hs)
            grads = ref.attention_backward(dout, qs, k, v, **hs)
            for n, t in zip(("dq", "dk", "dv"), got):
                within(t, *grads[n], f"{n} {factor} {scale} {size}")
    status_ok()


def test_attention_gradients_against_differences():
    q, k, v, how = attention_inputs((1, 40, 40, 4, 2, 16, 11, 2), F16)
    w = randn(*q.shape, dtype=F16, seed=9)

    def loss(q, k, v):
        return float((ref.attention(q, k, v, **how)[0] * w.double()).sum())

    out, lse = cs.attention(q, k, v, return_lse=True, **how)
    grads = cs.attention_backward(w, q, k, v, out, lse, **how)
    for seed in range(3):
        d = [randn(*t.shape, dtype=torch.float64, seed=40 + 3 * seed + i) for i, t in enumerate((q, k, v))]
        h, base = 1e-5, (q.double(), k.double(), v.double())
        slope = (loss(*(t + h * e for t, e in zip(base, d))) - loss(*(t - h * e for t, e in zip(base, d)))) / (2 * h)
        terms = [float((g.double() * e).sum()) for g, e in zip(grads, d)]
        size = sum(float((g.double() * e).abs().sum()) for g, e in zip(grads, d))
        assert abs(sum(terms) - slope) <= 8 * 2 ** -11 * size, (terms, slope)


def test_a_chain_on_another_stream_and_in_a_graph():
    """Scores to probabilities and back, attention and its gradients: on a side stream, then captured
    twice into graphs that replay on new inputs, with an eager run in between."""
    x, table, starts, bias_how = bias_inputs((2, 2, 65, 65, 0, 20, 2, 32, 128), BF16)
    q, k, v, how = attention_inputs((2, 140, 140, 4, 2, 64, 50, 2), BF16)
    dout = randn(*q.shape, dtype=BF16, seed=5)

    def chain(stream=None):
        p = cs.bias_softmax(x, table, starts, stream=stream, **bias_how)
        ds, dt = cs.bias_softmax_backward(p, x, starts, stream=stream, **bias_how)
        out, lse = cs.attention(q, k, v, return_lse=True, stream=stream, **how)
        one = cs.attention(q[:, -1:], k, v, stream=stream, **how)
        grads = cs.attention_backward(dout, q, k, v, out, lse, stream=stream, **how)
        return [p, ds, dt, out, lse, one, *grads]

    eager = [t.clone() for t in chain()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for s in (side, side.cuda_stream):
        got = chain(stream=s)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
    graphs, results = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(chain())
        graphs.append(g)
    for t, seed in ((x, 51), (q, 52), (k, 53), (v, 54), (dout, 55)):
        t.copy_(randn(*t.shape, dtype=t.dtype, seed=seed))
    fresh = [t.clone() for t in chain()]
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(r, fresh))
    assert not torch.equal(fresh[0], eager[0])
    status_ok()


def test_calls_at_once_on_two_streams():
    """Each call has its workspace: calls that overlap do not meet."""
    cases = [((2, 300, 300, 8, 2, 64, 90, 2), 11), ((1, 40, 1100, 4, 2, 128, 0, 0), 12)]
    streams = [torch.cuda.Stream() for _ in cases]
    inputs, alone, together = [], [], [[], []]

    def step(q, k, v, dout, how):
        out, lse = cs.attention(q, k, v, return_lse=True, **how)
        return [out, lse, *cs.attention_backward(dout, q, k, v, out, lse, **how)]

    for case, seed in cases:
        q, k, v, how = attention_inputs(case, BF16, seed=seed)
        inputs.append((q, k, v, randn(*q.shape, dtype=BF16, seed=seed + 5), how))
        alone.append(step(*inputs[-1]))
    torch.cuda.synchronize()
    for _ in range(20):
        for n, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                together[n].append(step(*inputs[n]))
    torch.cuda.synchronize()
    status_ok()
    for want, runs in zip(alone, together):
        assert all(torch.equal(a, b) for got in runs for a, b in zip(got, want))


@pytest.mark.parametrize("q_len", [1, 40])
def test_a_cache_of_more_than_2_to_the_31_elements(q_len):
    n, heads, kv_heads, dim, sinks, window, tail = 2**21 + 300, 8, 8, 128, 4, 100, 300
    q = randn(1, q_len, heads, dim, dtype=BF16, seed=1)
    k, v = (torch.full((1, n, kv_heads, dim), math.nan, dtype=BF16, device="cuda") for _ in range(2))
    small = []
    for t, seed in ((k, 2), (v, 3)):  # only what some query sees, or next to it
        part = randn(1, sinks + tail, kv_heads, dim, dtype=BF16, seed=seed)
        t[:, :sinks], t[:, -tail:] = part[:, :sinks], part[:, sinks:]
        small.append(part)
    how = dict(scale=dim ** -0.5, window=window, sinks=sinks)
    out, lse = cs.attention(q, k, v, return_lse=True, **how)
    want, bound, wl, bl = ref.attention(q, *small, **how)
    within(out, want, bound, "out")
    within(lse, wl, bl, "lse")
    dout = randn(*q.shape, dtype=BF16, seed=4)
    grads = cs.attention_backward(dout, q, k, v, out, lse, **how)
    status_ok()
    want = ref.attention_backward(dout, q, *small, **how)
    within(grads[0], *want["dq"], "dq")
    for name, t in (("dk", grads[1]), ("dv", grads[2])):
        within(torch.cat([t[:, :sinks], t[:, -tail:]], 1), *want[name], name)
        assert not t[:, sinks:-tail].any(), "keys that no query sees have no gradient"
    del k, v, t, grads
    torch.cuda.empty_cache()


def test_python_refusals():
    q, k, v, how = attention_inputs((1, 8, 8, 2, 2, 64, 0, 0), BF16)
    x, table, starts, bias_how = bias_inputs((1, 2, 8, 8, 0, 0, 0, 8, 16), BF16)
    lens = torch.ones(1, dtype=torch.int32, device="cuda")
    for bad in (dict(q=q.float()), dict(k=k.half()), dict(v=v[:, :4]), dict(q=q.cpu()), dict(q=q[..., ::2]),
                dict(q_lens=lens.long()), dict(kv_lens=lens.cpu()), dict(q_lens=lens.repeat(2)), dict(window=2**40),
                dict(out=q.half()), dict(out=k[:, :4]), dict(stream=object)):
        args = dict(dict(q=q, k=k, v=v), **bad)
        with pytest.raises((TypeError, ValueError, AttributeError)):
            cs.attention(args.pop("q"), args.pop("k"), args.pop("v"), **args)
    with pytest.raises(cs.CausalSoftmaxError):  # a broadcast tensor: stride 0
        cs.attention(q, k[:, :1].expand(1, 8, 2, 64), v)
    out, lse = cs.attention(q, k, v, return_lse=True, **how)
    for bad in (lse.double(), lse[..., :4], lse.transpose(1, 2)):
        with pytest.raises((TypeError, ValueError)):
            cs.attention_backward(q, q, k, v, out, bad, **how)
    for args in ((x.float(), table, starts), (x, table.half(), starts), (x, table[:1], starts), (x[0, 0], table, starts),
                 (x.transpose(1, 2), table, starts), (x, table, starts[:4])):
        with pytest.raises((TypeError, ValueError)):
            cs.bias_softmax(*args, **bias_how)
    with pytest.raises(cs.CausalSoftmaxError):
        cs.bias_softmax(x, table, starts, out=x, **bias_how)
    with pytest.raises((TypeError, ValueError)):
        cs.bias_softmax_backward(x, x.half(), starts, **bias_how)
    status_ok()
