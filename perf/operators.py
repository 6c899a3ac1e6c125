"""The attention operators beside the causal softmax: cases, plain forms and 64-bit forms.

Five operators, all with the same positional mask: a query at absolute position p sees the keys
k <= p that are among the last `window` ones (p - k < window; window 0: all) or among the first
`sinks` ones.

  bias_softmax            P = softmax(scale S + table[head, bucket(p - k)]) of score matrices
  bias_softmax_backward   dS and dtable from P and dP
  attention               softmax(scale Q K^T) V with the log-sum-exp of each row, for prompts
  attention, one token    the same call, reading a cache
  attention step          forward, then dQ, dK and dV

Where `own` is false, `run` computes them from elementary torch operations in 32 bits; where it is
true, through this package's entry points. `exact` computes them in 64 bits, head by head.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

PACKAGE = "gb200-sm100a-tma-fused-causal-attention-softmax_b200"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_modules = {}


def package():
    """This repository's Python binding (its folder's name is no module name)."""
    if "cs" not in _modules:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, PACKAGE))
        import causal_softmax

        _modules["cs"] = causal_softmax
    return _modules["cs"]


# ------------------------------------------------------------------ cases

def softmax_case(op, batch, heads, rows, cols, dtype, *, window=0, sinks=0, row_offset=0, buckets=32,
                 max_distance=128):
    return {"op": op, "batch": batch, "heads": heads, "rows": rows, "cols": cols, "dtype": dtype,
            "window": window, "sinks": sinks, "row_offset": row_offset, "buckets": buckets,
            "max_distance": max_distance}


def attention_case(op, batch, q_len, kv_len, heads, kv_heads, dim, dtype, *, window=0, sinks=0, ragged=False):
    return {"op": op, "batch": batch, "q_len": q_len, "kv_len": kv_len, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "window": window, "sinks": sinks, "ragged": ragged}


def listed():
    return [
        # Training-size score matrices of one layer, the matrix size of the benchmark workload.
        dict(softmax_case("bias_softmax", 4, 16, 4096, 4096, "fp16"), name="bias softmax 64 x 4096^2"),
        # A block of new rows over a longer context, odd columns (as the 1000 x 1037 workload), windowed.
        dict(softmax_case("bias_softmax", 2, 12, 1000, 1037, "bf16", window=256, sinks=4, row_offset=37),
             name="bias softmax 1000 x 1037 window"),
        # The backward of a layer's score matrices.
        dict(softmax_case("bias_softmax_backward", 2, 16, 4096, 4096, "bf16", max_distance=512),
             name="bias backward 32 x 4096^2"),
        # A small model's backward: latency and the table's reduction count.
        dict(softmax_case("bias_softmax_backward", 3, 8, 257, 257, "fp16", buckets=16, max_distance=64),
             name="bias backward 24 x 257^2"),
        # A long prompt with grouped heads: the largest call.
        dict(attention_case("attention", 1, 16384, 16384, 16, 4, 128, "bf16", window=4096, sinks=4),
             name="prompt 16384 window 4096"),
        # A padded batch of prompts of odd lengths, as many heads of keys as of queries.
        dict(attention_case("attention", 4, 2047, 2047, 12, 12, 64, "fp16", window=512, sinks=1, ragged=True),
             name="prompts ragged 2047 fp16"),
        # A chunk of a prompt over a cache that holds its beginning, without a window.
        dict(attention_case("attention", 2, 512, 8192, 16, 2, 128, "bf16"), name="chunk 512 of 8192"),
        # Single tokens of a large batch, caches of different lengths.
        dict(attention_case("attention", 64, 1, 8192, 32, 8, 128, "bf16", window=4096, sinks=4, ragged=True),
             name="token batch 64 window 4096"),
        # One sequence's token over a long cache: the work is split along the keys.
        dict(attention_case("attention", 1, 1, 65536, 16, 2, 128, "fp16"), name="token batch 1 of 65536"),
        # The smallest call, where latency counts.
        dict(attention_case("attention", 2, 1, 300, 8, 8, 64, "bf16", window=128, sinks=2),
             name="token batch 2 of 300"),
        # A training step of one layer with grouped heads.
        dict(attention_case("step", 2, 4096, 4096, 16, 4, 128, "bf16", window=1024, sinks=4),
             name="step 4096 window 1024"),
        # A small model's training step: a padded batch, odd lengths and a head size between the powers of two.
        dict(attention_case("step", 3, 1000, 1000, 6, 6, 80, "fp16", ragged=True), name="step ragged 1000 fp16"),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["bias_softmax", "bias_softmax_backward", "attention", "token", "step"])
    dtype = rng.choice(["fp16", "bf16"])
    window, sinks = 0, 0
    if op.startswith("bias"):
        cols = size(24, 8192)
        rows = cols if rng.random() < 0.6 else size(24, 4096)
        row_offset = 0 if rows == cols else rng.randrange(0, max(1, cols - 8))
        heads = rng.choice([1, 3, 8, 12, 16])
        most = (1 << 30 if op == "bias_softmax" else 1 << 29) // (rows * (cols + 8) * heads)
        batch = max(1, min(most, size(1, 16)))
        while rows * (cols + 8) * heads * batch > (1 << 30 if op == "bias_softmax" else 1 << 29):
            heads = max(1, heads // 2)
        if rng.random() < 0.4:
            window, sinks = size(16, 2048), rng.choice([0, 1, 4, 16])
        return softmax_case(op, batch, heads, rows, cols, dtype, window=window, sinks=sinks, row_offset=row_offset,
                            buckets=rng.choice([16, 32, 64]), max_distance=rng.choice([128, 512, 1024]))
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 8])
    ragged = rng.random() < 0.5
    if rng.random() < 0.7:
        window, sinks = size(64, 4096), rng.choice([0, 1, 4, 64])
    if op == "token":
        kv_len = size(64, 65536)
        batch = max(1, min(size(1, 64), (1 << 30) // (2 * kv_len * kv_heads * dim)))
        return attention_case("attention", batch, 1, kv_len, heads, kv_heads, dim, dtype, window=window, sinks=sinks,
                              ragged=ragged)
    kv_len = size(100, 8192 if op == "attention" else 4096)
    q_len = kv_len if op == "step" or rng.random() < 0.6 else max(1, min(kv_len, size(16, 2048)))
    most = (1 << 31 if op == "attention" else 1 << 28) // (q_len * kv_len * heads)
    return attention_case(op, max(1, min(most, size(1, 8))), q_len, kv_len,
                          heads if most else kv_heads, kv_heads, dim, dtype, window=window, sinks=sinks, ragged=ragged)


def lengths(case):
    """The sequences' lengths (queries, keys): even where the batch is not ragged."""
    batch, q_len, kv_len = case["batch"], case["q_len"], case["kv_len"]
    cut = (kv_len * 5 // 8) if case["ragged"] else 0
    kv = [max(1, kv_len - b * cut // max(1, batch - 1)) for b in range(batch)]
    return [min(q_len, n) for n in kv], kv


def bucket_starts(buckets, max_distance):
    """First distance of each bucket: half the buckets hold one distance each, the others grow by
    an even ratio up to max_distance, and the last one holds everything from its start on. In whole
    numbers: bucket e + t starts at the least n with (n / e)^m >= (max_distance / e)^t, m = buckets - e."""
    e = buckets // 2
    m = buckets - e
    starts = list(range(e))
    for t in range(m):
        goal, n = max_distance ** t * e ** (m - t), starts[-1] + 1
        while n ** m < goal:
            n += 1
        starts.append(n)
    return tuple(starts)


# ------------------------------------------------------------------ inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=t):
        out = torch.empty(*shape, dtype=dtype, device="cuda")
        for part in (out if out.numel() > 1 << 28 else [out]):
            part.copy_(torch.randn(part.shape, generator=g, device="cuda") * scale)
        return out

    state = dict(case)
    if case["op"].startswith("bias"):
        pitch = -(-case["cols"] // 8) * 8
        shape = (case["batch"], case["heads"], case["rows"], pitch)
        state.update(starts=bucket_starts(case["buckets"], case["max_distance"]), scale=128 ** -0.5)
        if case["op"] == "bias_softmax":  # scores of 128-wide heads before their scale, and a trained table
            state["x"] = normal(*shape, scale=128 ** 0.5)
            state["table"] = normal(case["heads"], case["buckets"], dtype=torch.float32)
        else:  # saved probabilities and the gradient that reaches them
            state["p"] = torch.empty(shape, dtype=t, device="cuda")
            keep = positions_mask(case)
            for i in range(case["batch"]):
                z = torch.randn(shape[1:], generator=g, device="cuda") * 1.5
                z = torch.where(keep, z[:, :, :case["cols"]], -math.inf)
                e = torch.exp(z - z.amax(-1, keepdim=True).clamp_min(-1e30))
                e = e / e.sum(-1, keepdim=True).clamp_min(1e-30)
                state["p"][i].zero_()
                state["p"][i, :, :, :case["cols"]].copy_(e)
            state["dp"] = normal(*shape)
        return state
    b, q_len, kv_len, dim = case["batch"], case["q_len"], case["kv_len"], case["dim"]
    state["scale"] = dim ** -0.5
    state["q"] = normal(b, q_len, case["heads"], dim)
    state["k"] = normal(b, kv_len, case["kv_heads"], dim)
    state["v"] = normal(b, kv_len, case["kv_heads"], dim)
    if case["op"] == "step":
        state["dout"] = normal(b, q_len, case["heads"], dim)
    state["q_lens"] = state["kv_lens"] = None
    if case["ragged"]:
        state["q_lens"], state["kv_lens"] = (torch.tensor(n, dtype=torch.int32, device="cuda") for n in lengths(case))
    return state


# ------------------------------------------------------------------ plain forms

def sees(p, k, window, sinks):
    keep = k <= p
    return keep & ((p - k < window) | (k < sinks)) if window else keep


def positions_mask(case):
    r = torch.arange(case["rows"], device="cuda")[:, None] + case["row_offset"]
    return sees(r, torch.arange(case["cols"], device="cuda")[None, :], case["window"], case["sinks"])


def bucket_map(s):
    r = torch.arange(s["rows"], device="cuda")[:, None] + s["row_offset"]
    far = (r - torch.arange(s["cols"], device="cuda")[None, :]).clamp_min(0)
    return torch.bucketize(far, torch.tensor(s["starts"], device="cuda"), right=True) - 1


def plain_bias_softmax(s):
    cols, keep = s["cols"], positions_mask(s)
    z = s["x"][..., :cols].float() * s["scale"] + s["table"][:, bucket_map(s)]
    z = torch.where(keep, z, -math.inf)
    e = torch.exp(z - z.amax(-1, keepdim=True).clamp_min(-3e38))
    del z
    out = torch.zeros_like(s["x"])
    out[..., :cols] = (e / e.sum(-1, keepdim=True).clamp_min(1e-37)).to(out.dtype)
    return {"p": out}


def plain_bias_softmax_backward(s):
    cols, keep = s["cols"], positions_mask(s)
    p, dp = s["p"][..., :cols].float(), s["dp"][..., :cols].float()
    dz = torch.where(keep, p * (dp - (p * dp).sum(-1, keepdim=True)), 0.0)
    del p, dp
    ds = torch.zeros_like(s["p"])
    ds[..., :cols] = (dz * s["scale"]).to(ds.dtype)
    # Sums along the diagonals (one distance each): rows written one place further left from row to
    # row, so that a distance is a column; then the distances of a bucket together.
    heads, rows, dz = s["heads"], s["rows"], dz.sum(0)
    flat = torch.zeros(heads, rows * (rows + cols), device="cuda")
    flat.as_strided((heads, rows, cols), (flat.shape[1], rows + cols - 1, 1), rows - 1).copy_(dz)
    by_column = flat.reshape(heads, rows, rows + cols).sum(1, dtype=torch.float64)
    far = s["row_offset"] + rows - 1 - torch.arange(rows + cols, device="cuda")
    at = torch.bucketize(far.clamp_min(0), torch.tensor(s["starts"], device="cuda"), right=True) - 1
    table = torch.zeros(heads, s["buckets"], dtype=torch.float64, device="cuda")
    return {"ds": ds, "dtable": table.index_add_(1, at, by_column).float()}


def visible(s):
    """[batch, 1, 1, queries, keys] truth values, or without the batch where all lengths are whole."""
    i, k = torch.arange(s["q_len"], device="cuda"), torch.arange(s["kv_len"], device="cuda")
    if s["q_lens"] is None:
        return sees((i + s["kv_len"] - s["q_len"])[:, None], k[None, :], s["window"], s["sinks"])
    nq, nk = s["q_lens"][:, None, None], s["kv_lens"][:, None, None]
    p = i[None, :, None] + nk - nq
    keep = sees(p, k[None, None, :], s["window"], s["sinks"]) & (i[None, :, None] < nq) & (k < nk)
    return keep[:, None, None]


def plain_attention(s, keep_p=False):
    b, n, h, d = s["q"].shape
    hk = s["k"].shape[2]
    q = s["q"].float().reshape(b, n, hk, h // hk, d)
    z = torch.einsum("bqhgd,bkhd->bhgqk", q * s["scale"], s["k"].float())
    z.masked_fill_(~visible(s), -math.inf)
    m = z.amax(-1, keepdim=True).clamp_min(-3e38)
    e = z.sub_(m).exp_()
    total = e.sum(-1, keepdim=True)
    lse = (m + torch.log(total)).reshape(b, h, n)
    p = e.div_(total.clamp_min(1e-37))
    out = torch.einsum("bhgqk,bkhd->bqhgd", p, s["v"].float())
    if keep_p:
        return out, lse, p, q
    return {"out": out.reshape(b, n, h, d).to(s["q"].dtype), "lse": lse}


def plain_step(s):
    out, lse, p, q = plain_attention(s, keep_p=True)
    t = s["q"].dtype
    dout = s["dout"].float().reshape(out.shape)
    if s["q_lens"] is not None:  # rows behind a sequence's end are no part of it
        dout = dout * (torch.arange(s["q_len"], device="cuda")[None, :] < s["q_lens"][:, None])[:, :, None, None, None]
    dv = torch.einsum("bhgqk,bqhgd->bkhd", p, dout)
    dz = torch.einsum("bqhgd,bkhd->bhgqk", dout, s["v"].float())
    dz.sub_((dout * out).sum(-1).permute(0, 2, 3, 1)[..., None]).mul_(p).mul_(s["scale"])
    dq = torch.einsum("bhgqk,bkhd->bqhgd", dz, s["k"].float())
    dk = torch.einsum("bhgqk,bqhgd->bkhd", dz, q)
    shape = s["q"].shape
    return {"out": out.reshape(shape).to(t), "dq": dq.reshape(shape).to(t), "dk": dk.to(t), "dv": dv.to(t)}


def run(s):
    if own:
        cs = package()
        if s["op"] == "bias_softmax":
            return {"p": cs.bias_softmax(s["x"], s["table"], s["starts"], cols=s["cols"], scale=s["scale"],
                                         row_offset=s["row_offset"], window=s["window"], sinks=s["sinks"])}
        if s["op"] == "bias_softmax_backward":
            ds, dtable = cs.bias_softmax_backward(s["p"], s["dp"], s["starts"], cols=s["cols"], scale=s["scale"],
                                                  row_offset=s["row_offset"], window=s["window"], sinks=s["sinks"])
            return {"ds": ds, "dtable": dtable}
        how = dict(scale=s["scale"], window=s["window"], sinks=s["sinks"], q_lens=s["q_lens"], kv_lens=s["kv_lens"])
        out, lse = cs.attention(s["q"], s["k"], s["v"], return_lse=True, **how)
        if s["op"] == "attention":
            return {"out": out, "lse": lse}
        dq, dk, dv = cs.attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, **how)
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    return {"bias_softmax": plain_bias_softmax, "bias_softmax_backward": plain_bias_softmax_backward,
            "attention": plain_attention, "step": plain_step}[s["op"]](s)


# ------------------------------------------------------------------ what a pass cannot do without

def seen_by_row(p, window, sinks, keys):
    """How many of `keys` keys the queries at positions p see (an array)."""
    hi = np.minimum(p + 1, keys)
    if not window:
        return np.maximum(hi, 0)
    lo = np.maximum(p + 1 - window, 0)
    return np.maximum(hi - lo, 0) + np.minimum(sinks, np.clip(np.minimum(lo, hi), 0, None)) * (p >= 0)


def work(case):
    if case["op"].startswith("bias"):
        p = np.arange(case["rows"], dtype=np.int64) + case["row_offset"]
        seen = int(seen_by_row(p, case["window"], case["sinks"], case["cols"]).sum())
        n = case["batch"] * case["heads"]
        whole = case["rows"] * (-(-case["cols"] // 8) * 8)
        reads = 2 if case["op"] == "bias_softmax_backward" else 1
        return {"bytes": n * 2 * (reads * seen + whole) + 4 * case["heads"] * case["buckets"], "flops": n * seen * 6 * reads}
    pairs, keys = 0, 0
    for nq, nk in zip(*lengths(case)):
        p = np.arange(nk - nq, nk, dtype=np.int64)
        pairs += int(seen_by_row(p, case["window"], case["sinks"], nk).sum())
        first = max(0, nk - nq + 1 - case["window"]) if case["window"] else 0
        keys += nk - first + min(case["sinks"], first)
    b, rows, d = case["batch"], case["batch"] * case["q_len"], case["dim"]
    q, kv, all_kv = 2 * rows * case["heads"] * d, 2 * keys * case["kv_heads"] * d, 2 * b * case["kv_len"] * case["kv_heads"] * d
    moved, flops = 2 * q + 2 * kv + 4 * rows * case["heads"], 4 * d * pairs * case["heads"]
    if case["op"] == "step":  # dout in, dq out, dk and dv out whole; five products after the forward's two
        moved += 2 * q + 2 * all_kv
        flops += 10 * d * pairs * case["heads"]
    return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------ 64 bits

def exact_bias(s, backward):
    cols, rows, dev = s["cols"], s["rows"], "cuda"
    r = np.arange(rows)[:, None] + s["row_offset"]
    k = np.arange(cols)[None, :]
    far = np.maximum(r - k, 0)
    e = s["buckets"] // 2
    grown = e + np.floor(np.log(np.maximum(far, 1) / e) / math.log(s["max_distance"] / e) * (s["buckets"] - e) + 1e-9)
    at = torch.tensor(np.where(far < e, far, np.minimum(grown, s["buckets"] - 1)).astype(np.int64), device=dev)
    hidden = torch.tensor((k > r) | ((r - k >= s["window"]) & (k >= s["sinks"]) if s["window"] else k > r), device=dev)
    first = s["p"] if backward else s["x"]
    out = torch.zeros(first.shape, dtype=torch.float64, device=dev)
    table = torch.zeros(s["heads"], s["buckets"], dtype=torch.float64, device=dev)
    for b in range(s["batch"]):
        for h in range(s["heads"]):
            x = first[b, h, :, :cols].double()
            if backward:
                x = x.masked_fill(hidden, 0)
                g = s["dp"][b, h, :, :cols].double()
                g = x * (g - (x * g).sum(-1, keepdim=True))
                table[h] += torch.bincount(at.reshape(-1), weights=g.reshape(-1), minlength=s["buckets"])
                out[b, h, :, :cols] = g * s["scale"]
            else:
                x = (x * s["scale"] + s["table"][h].double()[at]).masked_fill(hidden, -math.inf)
                out[b, h, :, :cols] = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
    return {"ds": out, "dtable": table} if backward else {"p": out}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("bias"):
        return exact_bias(s, case["op"] != "bias_softmax")
    group = case["heads"] // case["kv_heads"]
    got = {n: torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in ("q", "k", "v")}
    out = torch.zeros_like(got["q"])
    lse = torch.full((case["batch"], case["heads"], case["q_len"]), -math.inf, dtype=torch.float64, device="cuda")
    for b, (nq, nk) in enumerate(zip(*lengths(case))):
        p = torch.arange(nk - nq, nk, device="cuda")[:, None]
        k_at = torch.arange(nk, device="cuda")[None, :]
        hidden = k_at > p
        if case["window"]:
            hidden = hidden | ((k_at <= p - case["window"]) & (k_at >= case["sinks"]))
        for h in range(case["heads"]):
            q, k, v = s["q"][b, :nq, h].double(), s["k"][b, :nk, h // group].double(), s["v"][b, :nk, h // group].double()
            z = ((q @ k.T) * s["scale"]).masked_fill_(hidden, -math.inf)
            lse[b, h, :nq] = torch.logsumexp(z, -1)
            w = torch.softmax(z, -1)
            o = w @ v
            out[b, :nq, h] = o
            if case["op"] == "step":
                g = s["dout"][b, :nq, h].double()
                got["v"][b, :nk, h // group] += w.T @ g
                w *= (g @ v.T) - (g * o).sum(-1, keepdim=True)
                w *= s["scale"]
                got["q"][b, :nq, h] = w @ k
                got["k"][b, :nk, h // group] += w.T @ q
    if case["op"] == "step":
        return {"out": out, "dq": got["q"], "dk": got["k"], "dv": got["v"]}
    return {"out": out, "lse": lse}
