"""Plain 64-bit forms of the operators beside the softmax, and the error bounds
that a correctly rounded 16-bit result has to keep. Test infrastructure (torch,
any device).

Bounds, with u the half step of the type (bf16 2^-8 ... torch.finfo(t).eps / 2)
and a result's fp32 arithmetic at 2^-24 per operation: a score is a sum of
head_dim products, so it is off by at most E = (dim + 8) 2^-24 scale max|q|.|k|
(plus the exponential's 2^-20), and a probability by the relative 2 E. What is
rounded to 16 bits on the way (probabilities before they meet the values, ds
before it meets q and k) adds u of each term's magnitude. Exponentials below
FLUSHED, the least normal fp32, count as zero. In fp16 the backward's
probabilities are held times 2^15, so those near zero are off by half a subnormal
step, 2^-25, over 2^15; ds is held times the power of two that brings its bound
2 max|d_o| max|v| (row norms over a kv head) to between 2^14 and 2^15, so it is
off by up to 2^-25 of that bound over 2^14.
"""
from __future__ import annotations

import math

import torch


FLUSHED = 2.0 ** -126


def half_step(t) -> float:
    return torch.finfo(t).eps / 2


def tiny(t) -> float:
    """Half a step among the type's subnormal numbers."""
    return torch.finfo(t).tiny * torch.finfo(t).eps / 2


def mask(positions, keys: int, window: int, sinks: int):
    """[len(positions), keys]: what a query at each position sees."""
    p = positions[:, None]
    k = torch.arange(keys, device=positions.device)[None, :]
    keep = k <= p
    if window:
        keep = keep & ((p - k < window) | (k < sinks))
    return keep


def buckets(positions, keys: int, starts):
    d = positions[:, None] - torch.arange(keys, device=positions.device)[None, :]
    return torch.bucketize(d.clamp_min(0), torch.tensor(starts, device=d.device), right=True) - 1


def softmax_rows(z):
    m = z.amax(-1, keepdim=True).clamp_min(-1e300)
    e = torch.exp(z - m)
    s = e.sum(-1, keepdim=True)
    return torch.where(s > 0, e / s, 0.0), m + torch.log(s)


def bias_softmax(x, table, starts, *, cols, scale, row_offset=0, window=0, sinks=0):
    """x [batch, heads, rows, pitch] -> (p, bound), in 64 bits."""
    rows = x.shape[2]
    pos = torch.arange(rows, device=x.device) + row_offset
    keep = mask(pos, cols, window, sinks)
    z = x[..., :cols].double() * scale + table.double()[:, buckets(pos, cols, starts)]
    z = torch.where(keep, z, -math.inf)
    p = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    p[..., :cols] = softmax_rows(z)[0]
    zmax = float(z.abs().masked_fill(~keep | z.isinf(), 0.0).max())  # infinite scores are exact
    return p, p * (half_step(x.dtype) + zmax * 2 ** -21 + 2 ** -19) + tiny(x.dtype)


def bias_backward(p, dp, starts, nbuckets, *, cols, scale, row_offset=0, window=0, sinks=0):
    """(ds, ds bound, dtable, dtable bound) in 64 bits."""
    rows = p.shape[2]
    pos = torch.arange(rows, device=p.device) + row_offset
    keep = mask(pos, cols, window, sinks)
    a = torch.where(keep, p[..., :cols].double(), 0.0)
    g = torch.where(keep, dp[..., :cols].double(), 0.0)
    dz = a * (g - (a * g).sum(-1, keepdim=True))
    # A row's sum of up to cols terms in fp32, a few per lane and a tree.
    size = a * (g.abs() + (a * g).abs().sum(-1, keepdim=True))
    ds, bound = (torch.zeros(p.shape, dtype=torch.float64, device=p.device) for _ in range(2))
    ds[..., :cols] = dz * scale
    bound[..., :cols] = scale * (dz.abs() * half_step(p.dtype) + size * 2 ** -18) + tiny(p.dtype)
    at = buckets(pos, cols, starts).reshape(-1)

    def by_bucket(t):
        out = torch.zeros(p.shape[1], nbuckets, dtype=torch.float64, device=p.device)
        return out.index_add_(1, at, t.sum(0).reshape(p.shape[1], -1))

    # Each term as above; rows added one after another, at most `rows` of them a sum.
    return ds, bound, by_bucket(dz), by_bucket(size) * 2 ** -18 + by_bucket(dz.abs()) * (rows + 64) * 2 ** -24


def _sequences(q, k, q_lens, kv_lens):
    for b in range(q.shape[0]):
        nq = q.shape[1] if q_lens is None else min(max(int(q_lens[b]), 0), q.shape[1])
        nk = k.shape[1] if kv_lens is None else min(max(int(kv_lens[b]), 0), k.shape[1])
        yield b, nq, nk


def attention(q, k, v, *, scale, window=0, sinks=0, q_lens=None, kv_lens=None):
    """(out, out bound, lse, lse bound) in 64 bits."""
    out, bound = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    lse = torch.full((q.shape[0], q.shape[2], q.shape[1]), -math.inf, dtype=torch.float64, device=q.device)
    lse_bound = torch.zeros_like(lse)
    group, u = q.shape[2] // k.shape[2], half_step(q.dtype)
    for b, nq, nk in _sequences(q, k, q_lens, kv_lens):
        if nq == 0 or nk == 0:
            continue
        keep = mask(torch.arange(nk - nq, nk, device=q.device), nk, window, sinks)
        seen = keep.any(0)
        for h in range(q.shape[2]):
            Q, K, V = q[b, :nq, h].double(), k[b, :nk, h // group].double(), v[b, :nk, h // group].double()
            K, V = torch.where(seen[:, None], K, 0.0), torch.where(seen[:, None], V, 0.0)
            p, l = softmax_rows(torch.where(keep, Q @ K.T * scale, -math.inf))
            e = float((Q.abs() @ K.abs().T).max()) * scale * (q.shape[3] + 8) * 2 ** -24 + 2 ** -20
            out[b, :nq, h] = p @ V
            bound[b, :nq, h] = u * (p @ V).abs() + (u + 2 * e) * (p @ V.abs()) + \
                FLUSHED * V.abs().sum(0) + tiny(q.dtype)
            lse[b, h, :nq] = l[:, 0]
            lse_bound[b, h, :nq] = e + l[:, 0].abs().nan_to_num(posinf=0) * 2 ** -22
    return out, bound, lse, lse_bound


def attention_backward(dout, q, k, v, *, scale, window=0, sinks=0, q_lens=None, kv_lens=None):
    """{name: (gradient, bound)} in 64 bits."""
    g = {n: tuple(torch.zeros(t.shape, dtype=torch.float64, device=q.device) for _ in range(2))
         for n, t in (("dq", q), ("dk", k), ("dv", v))}
    group, u, dim = q.shape[2] // k.shape[2], half_step(q.dtype), q.shape[3]
    for b, nq, nk in _sequences(q, k, q_lens, kv_lens):
        if nq == 0 or nk == 0:
            continue
        keep = mask(torch.arange(nk - nq, nk, device=q.device), nk, window, sinks)
        seen, sees = keep.any(0), keep.any(1)
        for h in range(q.shape[2]):
            hk = h // group
            Q, G = (torch.where(sees[:, None], t[b, :nq, h].double(), 0.0) for t in (q, dout))
            K, V = (torch.where(seen[:, None], t[b, :nk, hk].double(), 0.0) for t in (k, v))
            p, _ = softmax_rows(torch.where(keep, Q @ K.T * scale, -math.inf))
            e = float((Q.abs() @ K.abs().T).max()) * scale * (dim + 8) * 2 ** -24 + 2 ** -20
            O, dp = p @ V, G @ V.T
            ds = p * (dp - (G * O).sum(-1, keepdim=True))
            # ds: its own rounding, the probability's error, dp's sum in fp32 and the rounded out in the row's sum.
            off = (u + 4 * e) * ds.abs() + p * (u * (G * O).abs().sum(-1, keepdim=True) +
                                                (4 * e + (dim + 8) * 2 ** -24) * (G.abs() @ V.abs().T))
            small_p = 2.0 ** -40 if q.dtype == torch.float16 else 0.0
            group_g = torch.where(sees[:, None, None], dout[b, :nq, hk * group:(hk + 1) * group].double(), 0.0)
            off += keep * 2.0 ** 2 * small_p * group_g.norm(dim=-1).max() * V.norm(dim=-1).max()
            off += keep * FLUSHED * (dp.abs() + (G * O).sum(-1, keepdim=True).abs())
            g["dq"][0][b, :nq, h] = scale * ds @ K
            g["dq"][1][b, :nq, h] = scale * off @ K.abs()
            g["dk"][0][b, :nk, hk] += scale * ds.T @ Q
            g["dk"][1][b, :nk, hk] += scale * off.T @ Q.abs()
            g["dv"][0][b, :nk, hk] += p.T @ G
            g["dv"][1][b, :nk, hk] += (u + 4 * e) * (p.T @ G.abs()) + (FLUSHED + small_p) * G.abs().sum(0)
    return {n: (t, bound + u * t.abs() + 2 * tiny(q.dtype)) for n, (t, bound) in g.items()}
