"""Attention with a sliding window and sinks in 64 bits, sample by sample and head by head, with the error that the kernels may make.

Query i of n stands at place p = i + m - n of m keys and sees key j where |p - j| < window or j < sinks, and j <= p where causal. The
bounds count roundings as those of tests/plain_tokens.py do, with the keys (queries) that a row (key) sees in the place of all."""
import torch

from tests.plain_tokens import U32, half_step, samples


def seen(n, m, window, sinks, causal, device="cpu"):
    p = torch.arange(n, device=device)[:, None] + (m - n)
    j = torch.arange(m, device=device)[None, :]
    see = ((p - j).abs() < window) | (j < sinks)
    return see & (j <= p) if causal else see


def attention(q, k, v, offsets, kv_offsets=None, kv_lengths=None, causal=False, scale=None, window=1, sinks=0, grad=None):
    """{name: (value, bound)} of out and lse and, with ``grad``, of dq, dk and dv."""
    dtype = q.dtype
    u = half_step(dtype)
    u_part = u if dtype == torch.bfloat16 else 0.0  # p and ds may be rounded before they are multiplied
    scale = q.size(2) ** -0.5 if scale is None else scale
    h, hk, d = q.size(1), k.size(1), q.size(2)
    Q, K, V = q.double(), k.double(), v.double()
    G = None if grad is None else grad.double()
    out = {n: [torch.zeros_like(t), torch.zeros_like(t)] for n, t in (("out", Q), ("dq", Q), ("dk", K), ("dv", V))}
    lse = torch.full((h, q.size(0)), float("-inf"), dtype=torch.float64, device=q.device)
    e_lse = torch.zeros_like(lse)
    for rq, rk in samples(offsets, q.size(0), kv_offsets, kv_lengths):
        nq, nk = rq.stop - rq.start, rk.stop - rk.start
        if nq == 0 or nk == 0:
            continue
        see = seen(nq, nk, window, sinks, causal, q.device)
        keys, rows = int(see.sum(1).max()), int(see.sum(0).max())
        for i in range(h):
            j = i // (h // hk)
            a, b, c = Q[rq, i], K[rk, j], V[rk, j]
            s = (scale * (a @ b.T)).masked_fill(~see, float("-inf"))
            top = s.amax(1, keepdim=True)
            top = top.masked_fill(top == float("-inf"), 0)
            e = (s - top).exp()
            total = e.sum(1, keepdim=True)
            p = e / total.masked_fill(total == 0, 1)
            o = p @ c
            size = (abs(scale) * (a.abs() @ b.abs().T)).masked_fill(~see, 0)
            e_s = (2 * d + 8) * U32 * size + 4 * U32 * (s.masked_fill(~see, 0).abs() + top.abs())
            off = (2 * e_s.amax(1, keepdim=True) + (2 * keys + 64) * U32)
            pa = p @ c.abs()
            e_o = (off + u_part) * pa + (2 * keys + 64) * U32 * pa
            out["out"][0][rq, i] = o
            out["out"][1][rq, i] = e_o + (u + 4 * U32) * o.abs()
            lse[i, rq] = torch.where(total > 0, top + total.log(), float("-inf"))[:, 0]
            e_lse[i, rq] = (off + 8 * U32 * (top.abs() + 1))[:, 0]
            if G is None:
                continue
            g = G[rq, i]
            dp = g @ c.T
            delta = (g * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            e_delta = (g.abs() * (e_o + (u + 4 * U32) * o.abs())).sum(1, keepdim=True) + (d + 4) * U32 * (g * o).abs().sum(1, keepdim=True)
            e_dp = (2 * d + 8) * U32 * (g.abs() @ c.abs().T)
            e_ds = p * (e_dp + e_delta + (2 * off + 8 * U32) * (dp.abs() + delta.abs())) + u_part * ds.abs()
            n_q, n_k = (2 * keys + 64) * U32, (2 * rows * (h // hk) + 64) * U32
            dq = scale * (ds @ b)
            out["dq"][0][rq, i] = dq
            out["dq"][1][rq, i] = abs(scale) * (e_ds @ b.abs() + n_q * (ds.abs() @ b.abs())) + (u + 4 * U32) * dq.abs()
            out["dk"][0][rk, j] += scale * (ds.T @ a)
            out["dk"][1][rk, j] += abs(scale) * (e_ds.T @ a.abs() + n_k * (ds.abs().T @ a.abs()))
            out["dv"][0][rk, j] += p.T @ g
            out["dv"][1][rk, j] += ((off + u_part + n_k) * p).T @ g.abs()
    for n in ("dk", "dv"):
        out[n][1] += (u + 4 * U32) * out[n][0].abs()
    res = {n: tuple(t) for n, t in out.items() if grad is not None or n == "out"}
    res["lse"] = (lse, e_lse)
    return res
