"""Rotary positions and norms of heads in 64 bits, with the error that the kernels may make.

The bounds count roundings; u is half a step of the type, relative to the value (tests/plain_tokens.py has ``check``). A turn is cut off at
2^-32 of it; frequency / 2 pi and this file's own angle are good to 2^-52 of the angle each. Sine and cosine: three roundings of an
argument below pi / 4, and five of a polynomial whose terms shrink, make fewer than eight in all."""
import math

import torch

from tests.plain_tokens import U32, half_step


def _turn(x, err, cos, sin, e_turn, interleaved):
    """The pairs of x [rows, heads, dim] turned, and the bound of the result where x is off by ``err``."""
    n = cos.size(1)
    cos, sin, e_turn = cos[:, None], sin[:, None], e_turn[:, None]
    rot = slice(0, 2 * n)
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    y, e = x.clone(), err.clone()
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    size = x[..., a].abs() + x[..., b].abs()
    # the other one's error comes in, too (|cos|, |sin| <= 1); two products and their sum
    off = err[..., a] + err[..., b] + size * (e_turn + 3 * U32)
    e[..., a], e[..., b] = off, off
    assert rot.stop <= x.size(2)
    return y, e


def rotary(q, k, positions, frequencies, sections, interleaved=False, norm=False, wq=None, wk=None, eps=1e-6, gq=None, gk=None):
    """{name: (value, bound)} of q, k (None: left out) and, with the outputs' gradients, of dq, dk, dwq, dwk."""
    dev, rows = q.device, q.size(0)
    if sum(sections):
        places = positions if positions.dim() == 2 else positions[:, None]
        axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device=dev)
        angle = places.double()[:, axis] * frequencies
        e_turn = 8 * U32 + 2 * math.pi * 2.0 ** -32 + angle.abs() * 2.0 ** -51
        cos, sin = torch.cos(angle), torch.sin(angle)
    else:
        cos = sin = e_turn = torch.zeros(rows, 0, dtype=torch.float64, device=dev)
    out = {}
    for name, x, w, g in (("q", q, wq, gq), ("k", k, wk, gk)):
        if x is None:
            continue
        dtype, h, d = x.dtype, x.size(1), x.size(2)
        u = half_step(dtype)
        X = x.double()
        W = torch.ones(d, dtype=torch.float64, device=dev) if w is None else w.double()
        if norm:
            inv = (X.square().mean(2, keepdim=True) + eps).rsqrt()
            e_inv = (d / 2 + 8) * U32   # relative: the sum of d squares, a root of it, a division
            hat = X * inv
            e_hat = (e_inv + U32) * hat.abs()
            y, e = hat * W, (e_hat + U32 * hat.abs()) * W.abs()
        else:
            y, e = X, torch.zeros_like(X)
        y, e = _turn(y, e, cos, sin, e_turn, interleaved)
        out[name] = (y, e + u * y.abs() + u * e)
        if g is None:
            continue
        G = g.double()
        b, e_b = _turn(G, torch.zeros_like(G), cos, -sin, e_turn, interleaved)
        if not norm:
            out["d" + name] = (b, e_b + u * b.abs() + u * e_b)
            continue
        # a thread adds the heads and rows that it visits (no fewer than 148 threads share them where there are as many), then 13 more sums
        run = rows * h / 148 + h + 16
        out["dw" + name] = ((b * hat).sum((0, 1)),
                            (e_b * hat.abs() + b.abs() * e_hat + (run * U32) * (b * hat).abs()).sum((0, 1)))
        value, bound = out["dw" + name]
        out["dw" + name] = (value, bound + (half_step(w.dtype if w is not None else torch.float32) + U32) * value.abs())
        a, e_a = b * W, e_b * W.abs() + U32 * (b * W).abs()
        dot = (a * hat).mean(2, keepdim=True)
        e_dot = (e_a * hat.abs() + a.abs() * e_hat + (d + 4) * U32 * (a * hat).abs()).mean(2, keepdim=True)
        dx = inv * (a - hat * dot)
        size = inv * (a.abs() + (hat * dot).abs())
        e_dx = inv * (e_a + e_hat * dot.abs() + hat.abs() * e_dot) + (e_inv + 4 * U32) * size
        out["d" + name] = (dx, e_dx + u * dx.abs() + u * e_dx)
    return out
