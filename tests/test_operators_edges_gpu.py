"""GPU tests of the operators beside the softmax at the edges of what they accept:
scores at the ends of the type's range, NaN and infinities in seen places, rows of
very different sizes."""
import math

import pytest
import torch

import attention_ref as ref
import causal_softmax as cs
from test_operators_gpu import BF16, F16, randn, status_ok, within

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- biased softmax

def shifted_bias_softmax(x, table, starts, *, cols, scale, row_offset=0, window=0, sinks=0):
    """The definition in 64 bits with each row's scores relative to its largest one (the softmax
    does not change), so that scores at the ends of the range keep their bias; and the bound of
    a result rounded once from exponentials of relative error 2^-16 (an argument above -128 in
    units of log2 rounded to 24 bits)."""
    pos = torch.arange(x.shape[2], device=x.device) + row_offset
    keep = ref.mask(pos, cols, window, sinks)
    s = torch.where(keep, x[..., :cols].double(), -math.inf)
    top = s.amax(-1, keepdim=True)
    s = s - torch.where(top.isinf(), 0.0, top)
    z = torch.where(keep, scale * s + table.double()[:, ref.buckets(pos, cols, starts)], -math.inf)
    p = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    p[..., :cols] = ref.softmax_rows(z)[0]
    return p, p * (ref.half_step(x.dtype) + 2 ** -15) + ref.tiny(x.dtype) + ref.FLUSHED


EXTREME = [
    # batch, heads, rows, cols, row_offset, window, sinks: rows of one lane's vectors to several warps' and unstaged ones
    (1, 2, 24, 24, 0, 0, 0),
    (40, 16, 120, 120, 0, 0, 0),
    (2, 2, 24, 700, 600, 200, 3),
    (1, 2, 24, 2500, 2476, 0, 0),
    (1, 1, 24, 9001, 8977, 0, 0),
    (1, 1, 24, 34000, 33976, 0, 0),
    (1, 1, 24, 70001, 69977, 0, 0),
]


@pytest.mark.parametrize("case", EXTREME)
@pytest.mark.parametrize("scale", [1.0, 0.125, 1e30])
def test_bias_scores_at_the_ends_of_the_range(case, scale):
    """Only infinite scores count as infinite: finite ones whose multiple of log2 e is not finite stay what they are."""
    batch, heads, rows, cols, row_offset, window, sinks = case
    starts = cs.bias_buckets(16, 64)
    how = dict(cols=cols, scale=scale, row_offset=row_offset, window=window, sinks=sinks)
    x = randn(batch, heads, rows, cs.padded_pitch(cols), dtype=BF16, seed=1)
    table = randn(heads, 16, dtype=torch.float32, seed=2)
    low, high = torch.finfo(BF16).min, torch.finfo(BF16).max
    x[:, :, 3] = low                       # masked by the lowest value everywhere: the softmax of the bias
    x[:, :, 4] = high
    x[:, :, 5, ::2], x[:, :, 5, 1::2] = low, high
    x[:, :, 6, ::3] = high                 # some at the top, others ordinary
    x[:, :, 7] = low
    x[:, :, 7, 2::5] = -3.1e38             # the lowest and a little above it
    x[:, :, 8] = 3.1e38
    x[:, :, 8, 1::4] = 2.9e38
    x[:, :, 9] = -math.inf                 # nothing but -infinity: zeros
    x[:, :, 10] = -math.inf
    x[:, :, 10, 3::2] = low                # the lowest value and -infinity
    x[:, :, 11] = -2.5e38
    x[:, :, 12] = 1e10
    x[:, :, 12, ::2] = 1.0078125e10
    got = cs.bias_softmax(x, table, starts, **how)
    want, bound = shifted_bias_softmax(x, table, starts, **how)
    within(got[:, :, 3:13], want[:, :, 3:13], bound[:, :, 3:13], "p")
    assert not got[:, :, 9].any()
    assert (got[:, :, 3:9].double().sum(-1) > 0.9).all()
    plain, plain_bound = ref.bias_softmax(x[:, :, :3], table, starts, **how)  # the rows beside them
    if scale <= 1:
        within(got[:, :, :3], plain, plain_bound, "ordinary rows")
    x[:, :, 3:9, 0] = math.nan             # the first sinks, or the first key where there is no window
    x[:, :, 10, 0] = math.inf
    got = cs.bias_softmax(x, table, starts, **how)
    seen = ref.mask(torch.arange(rows, device="cuda") + row_offset, cols, window, sinks)
    for row in (*range(3, 9), 10):
        if seen[row, 0]:
            assert torch.isnan(got[:, :, row, :cols][..., seen[row]]).all(), row
        assert not got[:, :, row, :cols][..., ~seen[row]].any()


def test_bias_tables_at_the_ends_of_the_range():
    starts, x = (0, 1, 2, 3, 11), randn(2, 3, 40, 40, dtype=BF16, seed=1)
    f = torch.finfo(torch.float32)
    for values in ((f.min, f.min, 0.0, 1.0, -1.0), (f.max, 0.0, f.max, 1.0, f.min), (-math.inf, f.min, -3e38, f.min, f.min),
                   (-math.inf, -math.inf, 0.5, -math.inf, -math.inf), (f.min, f.min, f.min, f.min, f.min)):
        table = torch.tensor([values] * 3, device="cuda")
        table[1] = randn(5, dtype=torch.float32, seed=3)  # a head with an ordinary one
        how = dict(cols=40, scale=0.125)
        want, bound = shifted_bias_softmax(x, table, starts, **how)
        # In 64 bits scores vanish beside a bias of 3e38, as they do here.
        within(cs.bias_softmax(x, table, starts, **how), want, bound + want * 2 ** -15, str(values))
    table = torch.tensor([[f.max, f.max]], device="cuda")  # cancels against the scores
    x = torch.full((1, 1, 4, 8), -3.3e38, dtype=BF16, device="cuda")
    x[..., 0] = 0.0
    got = cs.bias_softmax(x, table, (0, 2), cols=4, scale=1.0)[0, 0, :, :4]
    assert torch.equal(got, torch.eye(4, dtype=BF16, device="cuda")[[0, 0, 0, 0]])


# ---------------------------------------------------------------- attention

def one_key(value, dim, dtype):
    """A key whose product with a query of ones is value."""
    k = torch.zeros(dim, dtype=dtype, device="cuda")
    k[0] = value
    return k


UNUSUAL = [
    # batch, q_len, kv_len, heads, kv_heads: one token in one split and in several; few and many rows of tiles, split and whole
    (128, 1, 96, 4, 4),
    (300, 1, 300, 8, 8),
    (1, 1, 4000, 8, 1),
    (1, 1, 30000, 16, 1),
    (1, 2, 4000, 8, 1),
    (1, 40, 4000, 2, 1),
    (1, 200, 460, 2, 2),
    (1, 130, 20000, 1, 1),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", UNUSUAL)
@pytest.mark.parametrize("near", [True, False])
def test_nan_and_infinite_scores_at_seen_keys(case, dtype, near):
    """The largest score stands in the last key, an unusual one in the first keys (far from it in other splits or
    tiles) or next to it; scores differ by more than an exponential's range."""
    batch, q_len, kv_len, heads, kv_heads = case
    dim = 64
    q = torch.zeros(batch, q_len, heads, dim, dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    v = randn(batch, kv_len, kv_heads, dim, dtype=dtype, seed=1)
    where = kv_len - q_len if near else 3  # every query sees it

    def call(value, last=300.0, rest=0.0):
        k = torch.zeros(batch, kv_len, kv_heads, dim, dtype=dtype, device="cuda")
        k[..., 0] = rest
        k[:, kv_len - q_len - 1] = one_key(last, dim, dtype)
        k[:, where] = one_key(value, dim, dtype)
        out, lse = cs.attention(q, k, v, scale=1.0, return_lse=True)
        status_ok()
        return k, out, lse

    for value in (math.nan, math.inf):
        _, out, lse = call(value)
        assert torch.isnan(out).all() and torch.isnan(lse).all(), value
    _, out, lse = call(-math.inf)
    k = call(-30000.0)[0]  # the same probability 0 in 64 bits, and a finite bound
    k0 = k.clone()
    k0[k0 == -30000.0] = 0.0
    want, _, wl, _ = ref.attention(q, k, v, scale=1.0)
    _, bound, _, bl = ref.attention(q, k0, v, scale=1.0)  # bounds of the scores that count
    within(out, want, bound, "out")
    within(lse, wl, bl, "lse")
    _, out, lse = call(-math.inf, -math.inf, -math.inf)  # nothing but -infinity
    assert not out.any() and torch.isneginf(lse).all()
    _, out, lse = call(math.nan, -math.inf, -math.inf)
    assert torch.isnan(out).all() and torch.isnan(lse).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("q_len,kv_len,heads,kv_heads", [
    (1, 100, 4, 4), (3, 100, 8, 4), (2, 200, 8, 1), (3, 5000, 8, 4), (2, 5000, 8, 1), (40, 100, 8, 4), (40, 5000, 2, 2),
])
def test_rows_that_see_nothing_are_zero_beside_values_that_are_no_numbers(q_len, kv_len, heads, kv_heads, value, dtype):
    """Padded rows and queries before the first key, in batches whose other rows meet a NaN or an infinity."""
    q, k, v = (randn(3, n, h, 64, dtype=dtype, seed=i) for i, (n, h) in
               enumerate(((q_len, heads), (kv_len, kv_heads), (kv_len, kv_heads))))
    v[:, 0] = value
    q_lens = torch.tensor([max(0, q_len - 1), q_len, q_len], dtype=torch.int32, device="cuda")
    kv_lens = torch.tensor([kv_len, kv_len, max(0, q_len - 1)], dtype=torch.int32, device="cuda")
    out, lse = cs.attention(q, k, v, q_lens=q_lens, kv_lens=kv_lens, return_lse=True)
    status_ok()
    sees = torch.ones(3, q_len, dtype=torch.bool, device="cuda")
    sees[0, q_len - 1] = False  # behind the sequence's queries
    sees[2, 0] = False          # at position -1
    assert not out[~sees].any(), "rows that see nothing are zero"
    assert torch.isneginf(lse.transpose(1, 2)[~sees]).all() and not torch.isneginf(lse.transpose(1, 2)[sees]).any()
    assert not torch.isfinite(out[sees]).any(), "every other query sees key 0"
    assert torch.isfinite(lse.transpose(1, 2)[sees]).all()


def gradients_by_row(dout, q, k, v, *, scale, window):
    """ref.attention_backward for one sequence, with fp16's held ds off by what its own factor leaves: of each row for
    dq, of each tile of 128 keys for dk (2^-25 / 2^14 of the largest |dP| + |delta| there; tiles are taken 256 wider)."""
    n, heads, dim = q.shape[1:]
    group, u = heads // k.shape[2], ref.half_step(q.dtype)
    result = {m: tuple(torch.zeros(t.shape[1:], dtype=torch.float64, device="cuda") for _ in range(2))
              for m, t in (("dq", q), ("dk", k), ("dv", v))}
    pos = torch.arange(n, device="cuda")
    keep, wide = ref.mask(pos, n, window, 0), window + 256 if window else n
    near = (pos[None, :] <= pos[:, None] + 256) & (pos[:, None] - pos[None, :] <= wide + 256)  # [query, key]
    small = 2.0 ** -39 if q.dtype == F16 else 0.0
    for h in range(heads):
        hk = h // group
        Q, G, K, V = (t[0, :, i].double() for t, i in ((q, h), (dout, h), (k, hk), (v, hk)))
        p, _ = ref.softmax_rows(torch.where(keep, Q @ K.T * scale, -math.inf))
        e = float((Q.abs() @ K.abs().T).max()) * scale * (dim + 8) * 2 ** -24 + 2 ** -20
        O, dp = p @ V, G @ V.T
        delta = (G * O).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        off = (u + 4 * e) * ds.abs() + p * (u * (G * O).abs().sum(-1, keepdim=True) +
                                            (4 * e + (dim + 8) * 2 ** -24) * (G.abs() @ V.abs().T))
        off = off + keep * ref.FLUSHED * (dp.abs() + delta.abs())
        rows = torch.where(near, V.norm(dim=-1)[None, :], 0.0).amax(1, keepdim=True) * G.norm(dim=-1, keepdim=True) + delta.abs()
        group_rows = torch.stack([(dout[0, :, i].double().norm(dim=-1)) for i in range(hk * group, hk * group + group)]).amax(0)
        both = group_rows[:, None] * torch.where(near, V.norm(dim=-1)[None, :], 0.0).amax(1, keepdim=True) * 2
        keys = torch.where(near, both, 0.0).amax(0, keepdim=True)
        result["dq"][0][:, h] = scale * ds @ K
        result["dq"][1][:, h] = scale * (off + keep * small * rows) @ K.abs()
        result["dk"][0][:, hk] += scale * ds.T @ Q
        result["dk"][1][:, hk] += scale * (off + keep * small * keys).T @ Q.abs()
        small_p = 2.0 ** -40 if q.dtype == F16 else 0.0
        result["dv"][0][:, hk] += p.T @ G
        result["dv"][1][:, hk] += (u + 4 * e) * (p.T @ G.abs()) + (ref.FLUSHED + small_p) * G.abs().sum(0)
    return {m: (t[None], (bound + u * t.abs() + 2 * ref.tiny(q.dtype))[None]) for m, (t, bound) in result.items()}


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (4, 1, 64), (6, 2, 128)])
@pytest.mark.parametrize("window,large", [(0, "dout"), (300, "dout"), (300, "v"), (0, "one row")])
def test_gradients_of_rows_of_very_different_sizes(window, large, heads, kv_heads, dim, dtype):
    """Small rows of d_o keep their bits beside rows 2^19 times larger, and where the large values are out of sight."""
    n = 2048
    q, dout = (randn(1, n, heads, dim, dtype=dtype, seed=i) for i in (1, 2))
    k, v = (randn(1, n, kv_heads, dim, dtype=dtype, seed=i) for i in (3, 4))
    if large == "v":
        v[:, :200] *= 2.0 ** 9
        dout[:, 700:] *= 2.0 ** -8
    elif large == "one row":
        dout *= 2.0 ** -8
        dout[:, 1100] *= 2.0 ** 19
    else:
        dout[:, 128:] *= 2.0 ** -8
        dout[:, :128] *= 2.0 ** 11
    how = dict(scale=dim ** -0.5, window=window)
    out, lse = cs.attention(q, k, v, return_lse=True, **how)
    got = cs.attention_backward(dout, q, k, v, out, lse, **how)
    status_ok()
    want = gradients_by_row(dout, q, k, v, **how)
    for name, t in zip(("dq", "dk", "dv"), got):
        within(t, *want[name], name)
    again = cs.attention_backward(dout, q, k, v, out, lse, **how)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", [
    # batch, q_len, kv_len, heads, kv_heads, dim, window, sinks: one split and several, 8 and 16 rows, both dims
    (150, 1, 200, 4, 4, 64, 0, 0),
    (2, 1, 3000, 8, 2, 128, 0, 0),
    (1, 2, 4000, 16, 2, 64, 3000, 4),
    (2, 4, 900, 12, 3, 80, 0, 0),
    (1, 1, 40000, 16, 1, 128, 0, 0),
])
def test_single_tokens_round_nothing_but_the_result(case, dtype):
    """Probabilities meet the values in two 16-bit parts: what the second one rounds is the half step squared."""
    batch, q_len, kv_len, heads, kv_heads, dim, window, sinks = case
    q = randn(batch, q_len, heads, dim, dtype=dtype, seed=1)
    k, v = (randn(batch, kv_len, kv_heads, dim, dtype=dtype, seed=i) for i in (2, 3))
    how = dict(scale=dim ** -0.5, window=window, sinks=sinks)
    out = cs.attention(q, k, v, **how)
    status_ok()
    want, bound, _, _ = ref.attention(q, k, v, **how)
    magnitude, u = ref.attention(q, k, v.abs(), **how)[0], ref.half_step(dtype)
    # ref's bound has u (p |v|) for a probability rounded once; here it is u^2.
    within(out, want, bound - (u - u * u) * magnitude, "out")


@pytest.mark.parametrize("scale", [0.1, 0.25, 0.26, 0.49, 1.0])
def test_bias_of_lowest_scores_beside_a_lowest_table(scale):
    """Neither is -infinity, nor is their sum in binary64: every visible key has the same share."""
    for bias in (-2e38, torch.finfo(torch.float32).min):
        x = torch.full((1, 1, 24, 24), torch.finfo(BF16).min, dtype=BF16, device="cuda")
        got = cs.bias_softmax(x, torch.full((1, 2), bias, device="cuda"), (0, 5), cols=24, scale=scale)[0, 0]
        want = torch.tril(torch.ones(24, 24, device="cuda")) / torch.arange(1, 25, device="cuda")[:, None]
        assert torch.equal(got, want.to(BF16)), bias


def test_fp16_gradients_and_wide_rows_in_graphs_and_on_two_streams():
    """Captured twice and replayed on new inputs, some rows of them wide, then eagerly on two streams at once."""
    x, table = randn(2, 4, 100, 104, dtype=BF16, seed=1), randn(4, 32, dtype=torch.float32, seed=2)
    starts, how = cs.bias_buckets(32, 128), dict(cols=100, scale=1.0, window=40, sinks=2)
    q, dout = (randn(2, 300, 6, 80, dtype=F16, seed=i) for i in (3, 4))
    k, v = (randn(2, 300, 2, 80, dtype=F16, seed=i) for i in (5, 6))

    def chain():
        p = cs.bias_softmax(x, table, starts, **how)
        out, lse = cs.attention(q, k, v, window=90, sinks=3, return_lse=True)
        return [p, out, lse, *cs.attention_backward(dout, q, k, v, out, lse, window=90, sinks=3)]

    chain()
    torch.cuda.synchronize()
    graphs, results = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(chain())
        graphs.append(g)
    for seed in (10, 20):
        for t in (x, q, k, v, dout):
            t.copy_(randn(*t.shape, dtype=t.dtype, seed=seed))
            seed += 1
        x[:, :, seed % 7::7] = torch.finfo(BF16).min
        dout[:, ::3] *= 2.0 ** 10
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        fresh = chain()
        for r in results:
            assert all(torch.equal(a, b) for a, b in zip(r, fresh))
        assert (fresh[0].float().sum(-1) > 0.9).all()
    streams, runs = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                runs.append(chain())
    torch.cuda.synchronize()
    status_ok()
    assert all(torch.equal(a, b) for r in runs for a, b in zip(r, fresh))
