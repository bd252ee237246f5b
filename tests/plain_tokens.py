"""Layer norm and packed attention in 64 bits, sample by sample and head by head, with the error that the kernels may make.

The bounds count roundings. u is half a step of the type, relative to the value: torch.finfo(type).eps / 2. A sum of n terms in fp32
is off by at most n u32 times the sum of the terms' sizes (tensor cores cut off instead of rounding: twice that)."""
import torch

U32 = torch.finfo(torch.float32).eps / 2


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def layer_norm(x, w, b, eps, dy=None):
    """{name: (value, bound)} of the output and, with ``dy``, of the gradients."""
    dtype, wtype = x.dtype, (w if w is not None else b if b is not None else x.float()).dtype
    x = x.double()
    n, c = x.shape
    w = torch.ones(c, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(c, dtype=torch.float64, device=x.device) if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    inv = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    xhat = (x - mean) * inv
    y = xhat * w + b
    # a thread adds at most 32 values, five shuffles and a block's five more follow; three roundings behind them
    adds = 45
    off = adds * U32 * inv * x.abs().amax(1, keepdim=True)          # of xhat, from the mean
    off_hat = 2 * off + (adds + 6) * U32 * (xhat.abs() + xhat.abs().amax(1, keepdim=True) * off)
    out = {"y": (y, off_hat * w.abs() + 3 * U32 * (y.abs() + b.abs()) + half_step(dtype) * y.abs())}
    if dy is None:
        return out
    dy = dy.double()
    g = dy * w
    a, m = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
    dx = inv * (g - a - xhat * m)
    e_a = (adds + 3) * U32 * g.abs().mean(1, keepdim=True)
    e_m = (adds + 3) * U32 * (g * xhat).abs().mean(1, keepdim=True) + (g.abs() * off_hat).mean(1, keepdim=True)
    e_dx = inv * (4 * U32 * (g.abs() + a.abs() + (xhat * m).abs()) + e_a + off_hat * m.abs() + xhat.abs() * e_m)
    e_dx = e_dx + dx.abs() * (adds + 6) * U32 + dx.abs() * off_hat.amax(1, keepdim=True)
    out["dx"] = (dx, e_dx + half_step(dtype) * dx.abs())
    dw, db = (dy * xhat).sum(0), dy.sum(0)
    # a thread's run of rows, the groups and warps of a block; the blocks are added in 64 bits
    run = n / 148 + 64
    e_dw = (run * U32 * (dy * xhat).abs()).sum(0) + (dy.abs() * off_hat).sum(0)
    out["dw"] = (dw, e_dw + (half_step(wtype) + U32) * dw.abs())
    out["db"] = (db, run * U32 * dy.abs().sum(0) + (half_step(wtype) + U32) * db.abs())
    return out


def samples(offsets, rows, kv_offsets=None, kv_lengths=None):
    """(query rows, key rows in use) of every sample, as slices."""
    o = offsets.tolist()
    ko = o if kv_offsets is None else kv_offsets.tolist()
    kl = [b - a for a, b in zip(ko, ko[1:])] if kv_lengths is None else kv_lengths.tolist()
    return [(slice(a, b), slice(k, k + n)) for a, b, k, n in zip(o, o[1:], ko, kl)]


def attention(q, k, v, offsets, kv_offsets=None, kv_lengths=None, causal=False, scale=None, grad=None, parts=True):
    """{name: (value, bound)} of out and lse and, with ``grad``, of dq, dk and dv. ``parts``: p and ds may be rounded to the
    tensors' type before they are multiplied (the tensor-core kernels do so)."""
    dtype = q.dtype
    u = half_step(dtype)
    u_part = u if parts and dtype == torch.bfloat16 else 0.0
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
        see = torch.ones(nq, nk, dtype=torch.bool, device=q.device)
        if causal:
            see = see.tril(nk - nq)
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
            # a score: d products and their sum, the scale; the exponential's argument and value, a few roundings of its size
            size = (abs(scale) * (a.abs() @ b.abs().T)).masked_fill(~see, 0)
            e_s = (2 * d + 8) * U32 * size + 4 * U32 * (s.masked_fill(~see, 0).abs() + top.abs())
            off = (2 * e_s.amax(1, keepdim=True) + (2 * nk + 64) * U32)    # relative, of p: its own and its sum's
            pa = p @ c.abs()
            e_o = (off + u_part) * pa + (2 * nk + 64) * U32 * pa
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
            # delta is made from the stored output
            e_delta = (g.abs() * (e_o + (u + 4 * U32) * o.abs())).sum(1, keepdim=True) + (d + 4) * U32 * (g * o).abs().sum(1, keepdim=True)
            e_dp = (2 * d + 8) * U32 * (g.abs() @ c.abs().T)
            e_ds = p * (e_dp + e_delta + (2 * off + 8 * U32) * (dp.abs() + delta.abs())) + u_part * ds.abs()
            n_q, n_k = (2 * nk + 64) * U32, (2 * nq * (h // hk) + 64) * U32
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


def check(got, want, what=""):
    """Every entry within its bound (an infinite value has to be the same infinity)."""
    value, bound = want
    got = got.detach().double()
    assert got.shape == value.shape, what
    same = (got == value) | (torch.isnan(got) & torch.isnan(value))
    off = torch.where(same, torch.zeros_like(value), (got - value).abs())
    bad = ~(off <= bound + 1e-30)
    if bool(bad.any()):
        i = int(torch.where(bad, off / (bound + 1e-30), torch.zeros_like(off)).flatten().nan_to_num(posinf=1e30, nan=1e30).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, worst at {i}: got {got.flatten()[i].item()}, "
                             f"want {value.flatten()[i].item()}, bound {bound.expand_as(value).flatten()[i].item()}")
