"""The operators of token networks on feature matrices, as a program that uses the C++ host layer (``riemann_cpp``) calls them:

* layer norm over the channels of every row, forward and forward + backward;
* attention within the samples of a batch: the rows of the samples lie one behind the other in one matrix ("packed"), every
  sample has a length of its own, several query heads may share a key head; full or causal, forward, forward + backward, and
  single query rows against long keys kept in a cache.

The plain forms are elementary torch operations in 32 bits over samples padded to one length; ``exact`` goes head by head and
sample by sample in 64 bits.
"""
import random

import torch

own = False

DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5


def listed():
    return [
        # the rows of one small object: what a call costs when latency is all there is
        {"name": "norm-object-f32", "op": "norm", "dtype": "f32", "rows": 1018, "channels": 32, "train": False},
        # the benchmark's eight rooms at its layer's width, in a training step
        {"name": "norm-rooms8-bf16-train", "op": "norm", "dtype": "bf16", "rows": 1_200_000, "channels": 64, "train": True},
        # a coarser map in fp32, ragged row count, channels that are no power of two, in a training step
        {"name": "norm-coarse-f32-train", "op": "norm", "dtype": "f32", "rows": 48_503, "channels": 96, "train": True},
        # wide token features, in a training step
        {"name": "norm-tokens-bf16-train", "op": "norm", "dtype": "bf16", "rows": 16_411, "channels": 1024, "train": True},
        # one small object, fp32 (the layers' default type): latency
        {"name": "attn-object-f32", "op": "attn", "dtype": "f32", "seqs": 1, "shortest": 203, "longest": 203, "heads": 4,
         "kv_heads": 4, "dim": 16, "causal": False, "train": False},
        # a few small clouds in fp32, in a training step
        {"name": "attn-clouds-f32-train", "op": "attn", "dtype": "f32", "seqs": 4, "shortest": 301, "longest": 1103,
         "heads": 4, "kv_heads": 4, "dim": 32, "causal": False, "train": True},
        # many windows of the rows of large scenes, few channels a head, in a training step
        {"name": "attn-windows-bf16-train", "op": "attn", "dtype": "bf16", "seqs": 96, "shortest": 17, "longest": 1024,
         "heads": 8, "kv_heads": 8, "dim": 32, "causal": False, "train": True},
        # clouds of very different lengths, causal, four query heads to a key head: a prompt
        {"name": "attn-clouds-bf16", "op": "attn", "dtype": "bf16", "seqs": 8, "shortest": 151, "longest": 5003, "heads": 8,
         "kv_heads": 2, "dim": 64, "causal": True, "train": False},
        # the same kind of batch in a training step
        {"name": "attn-clouds-bf16-train", "op": "attn", "dtype": "bf16", "seqs": 8, "shortest": 151, "longest": 4001,
         "heads": 8, "kv_heads": 4, "dim": 64, "causal": True, "train": True},
        # one long prompt
        {"name": "attn-long-bf16", "op": "attn", "dtype": "bf16", "seqs": 1, "shortest": 8192, "longest": 8192, "heads": 16,
         "kv_heads": 16, "dim": 128, "causal": True, "train": False},
        # two long samples in a training step
        {"name": "attn-long-bf16-train", "op": "attn", "dtype": "bf16", "seqs": 2, "shortest": 3989, "longest": 4600,
         "heads": 16, "kv_heads": 8, "dim": 128, "causal": True, "train": True},
        # one new token for each of sixteen samples against what the cache holds of them
        {"name": "attn-step-bf16", "op": "step", "dtype": "bf16", "seqs": 16, "shortest": 509, "longest": 30_011,
         "heads": 16, "kv_heads": 4, "dim": 128},
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over the logarithm."""
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def draw(rng):
    kind = rng.choice(("norm", "norm-train", "attn", "attn", "attn-train", "attn-train", "step"))
    if kind.startswith("norm"):
        channels = rng.choice((16, 32, 48, 64, 96, 128, 192, 256, 384, 512, 768, 1024, rng.randrange(7, 1025, 2)))
        rows = min(_spread(rng, 1, 1_200_000), 1_200_000 * 64 // channels)
        return {"op": "norm", "dtype": rng.choice(("f32", "bf16")), "rows": rows, "channels": channels,
                "train": kind == "norm-train"}
    dtype = rng.choice(("f32", "bf16", "bf16", "bf16"))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 1, 2, 4))
    if kind == "step":
        seqs = rng.randrange(1, 17)
        longest = _spread(rng, 16, 30_011)
        return {"op": "step", "dtype": dtype, "seqs": seqs, "shortest": max(1, longest // rng.randrange(1, 60)),
                "longest": longest, "heads": min(heads, 16), "kv_heads": min(kv_heads, 4) if heads > 16 else kv_heads,
                "dim": rng.choice((16, 32, 64, 96, 128))}
    train = kind == "attn-train"
    dim = rng.choice((16, 24, 32, 48, 64, 80, 96, 128))
    seqs = _spread(rng, 1, 64)
    most = int(((16 * 4600 ** 2 * 2) / (2 * heads * seqs)) ** 0.5)
    longest = _spread(rng, 2, max(2, min(most, 8192 if dtype == "bf16" else 2048)))
    return {"op": "attn", "dtype": dtype, "seqs": seqs, "shortest": max(1, longest // rng.randrange(1, 40)),
            "longest": longest, "heads": heads, "kv_heads": kv_heads, "dim": dim, "causal": rng.random() < 0.5,
            "train": train}


def _lengths(case):
    """The samples' lengths: spread over the logarithm between the two given ones, both among them, in mixed order."""
    rng = random.Random(case["seqs"] * 1_000_003 + case["longest"])
    n = case["seqs"]
    lengths = [_spread(rng, case["shortest"], case["longest"]) for _ in range(n)]
    lengths[0] = case["shortest"]
    lengths[-1] = case["longest"]
    rng.shuffle(lengths)
    return lengths


def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def _inputs(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "norm":
        n, c = case["rows"], case["channels"]
        # features behind a layer: channels with means and scales of their own
        mean, spread = _randn(gen, (c,), torch.float32), _randn(gen, (c,), torch.float32).abs() + 0.2
        x = (torch.randn((n, c), generator=gen, device=DEV) * spread + mean).to(dtype)
        s = {"x": x, "weight": _randn(gen, (c,), dtype, 0.2) + 1, "bias": _randn(gen, (c,), dtype, 0.2)}
        if case["train"]:
            s["grad"] = _randn(gen, (n, c), dtype, 0.1)
        return s
    lengths = _lengths(case)
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "step":
        # one slot a sample in the cache, a little longer than what it holds now
        slots = [n + 16 for n in lengths]
        rows_q, rows_k = len(lengths), sum(slots)
    else:
        slots, rows_q, rows_k = lengths, sum(lengths), sum(lengths)
    s = {"q": _randn(gen, (rows_q, h, d), dtype), "k": _randn(gen, (rows_k, hk, d), dtype),
         "v": _randn(gen, (rows_k, hk, d), dtype), "lengths": lengths, "slots": slots}
    if case.get("train"):
        s["grad"] = _randn(gen, (rows_q, h, d), dtype, 0.1)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["op"], s["train"] = case["op"], bool(case.get("train"))
    if case["op"] != "norm":
        starts = [0]
        for n in s["slots"]:
            starts.append(starts[-1] + n)
        s["kv_offsets"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
        s["kv_lengths"] = torch.tensor(s["lengths"], dtype=torch.int32, device=DEV)
        s["offsets"] = s["kv_offsets"]
        if case["op"] == "step":
            s["offsets"] = torch.arange(len(s["lengths"]) + 1, dtype=torch.int32, device=DEV)
        s["longest"], s["causal"] = max(s["lengths"]), bool(case.get("causal"))
    if s["train"]:
        for name in ("x", "weight", "bias") if case["op"] == "norm" else ("q", "k", "v"):
            s[name].requires_grad_(True)
    return s


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _plain_norm(state) if state["op"] == "norm" else _plain_attention(state)


def _run_own(s):
    from riemannengine_b200 import cpp
    host = cpp.load()
    if s["op"] == "norm":
        leaves = (s["x"], s["weight"], s["bias"])
        out = host.layer_norm(*leaves, eps=EPS)
    elif s["op"] == "step":
        return [host.packed_attention(s["q"], s["k"], s["v"], s["offsets"], kv_offsets=s["kv_offsets"],
                                      kv_lengths=s["kv_lengths"], causal=True)]
    else:
        leaves = (s["q"], s["k"], s["v"])
        out = host.packed_attention(*leaves, s["offsets"], causal=s["causal"])
    if not s["train"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, leaves, s["grad"])]


def _plain_norm(s):
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    centred = x - x.mean(1, keepdim=True)
    inv = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + EPS)
    xhat = centred * inv
    out = (xhat * w + b).to(s["x"].dtype)
    if not s["train"]:
        return [out]
    dy = s["grad"].float()
    g = dy * w
    dx = inv * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    dw, db = (dy * xhat).sum(0), dy.sum(0)
    return [out, dx.to(s["x"].dtype), dw.to(s["weight"].dtype), db.to(s["bias"].dtype)]


def _padded(x, offsets, longest):
    """[rows, heads, dim] -> [samples, heads, longest, dim] in 32 bits; places behind a sample's end hold some other row."""
    at = offsets[:-1, None].long() + torch.arange(longest, device=x.device)
    return x.float()[at.clamp_max(x.size(0) - 1)].transpose(1, 2)


def _plain_attention(s):
    q, k, v = s["q"], s["k"], s["v"]
    h, hk, d = q.size(1), k.size(1), q.size(2)
    group, samples = h // hk, s["kv_lengths"].numel()
    n_q = s["offsets"][1:] - s["offsets"][:-1]
    n_k = s["kv_lengths"]
    long_q = 1 if s["op"] == "step" else s["longest"]
    long_k = s["longest"]
    scale = d ** -0.5
    qp = _padded(q, s["offsets"], long_q).reshape(samples, hk, group * long_q, d)
    kp, vp = _padded(k, s["kv_offsets"], long_k), _padded(v, s["kv_offsets"], long_k)
    i = torch.arange(long_q, device=q.device)[None, :, None]
    j = torch.arange(long_k, device=q.device)[None, None, :]
    seen = (i < n_q[:, None, None]) & (j < n_k[:, None, None])
    if s["causal"]:
        seen = seen & (j <= i + (n_k - n_q)[:, None, None])
    hidden = ~seen[:, None, None]
    scores = (qp * scale) @ kp.transpose(2, 3)
    by_head = scores.view(samples, hk, group, long_q, long_k)
    by_head.masked_fill_(hidden, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    top = top.masked_fill_(top == float("-inf"), 0.0)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(total.masked_fill_(total == 0, 1.0))
    out = p @ vp
    # the rows that are a sample's, one behind the other again
    rows = torch.arange(q.size(0), device=q.device)
    sample = torch.searchsorted(s["offsets"][1:].long(), rows, right=True)
    place = rows - s["offsets"][:-1].long()[sample]

    def packed(x, length, dtype):
        return x.view(samples, -1, length, d)[sample, :, place].to(dtype)

    if not s["train"]:
        return [packed(out, long_q, q.dtype)]
    do = _padded(s["grad"], s["offsets"], long_q)
    do = (do * (i < n_q[:, None, None]).unsqueeze(1)).reshape(samples, hk, group * long_q, d)
    dv = p.transpose(2, 3) @ do
    ds = do @ vp.transpose(2, 3)
    ds = ds.sub_((do * out).sum(-1, keepdim=True)).mul_(p)
    dq = (ds @ kp) * scale
    dk = (ds.transpose(2, 3) @ qp) * scale
    return [packed(out, long_q, q.dtype), packed(dq, long_q, q.dtype), packed(dk, long_k, k.dtype), packed(dv, long_k, v.dtype)]


def _pairs(case):
    lengths = _lengths(case)
    if case["op"] == "step":
        return sum(lengths)
    return sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lengths)


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "norm":
        n, c = case["rows"], case["channels"]
        if case["train"]:  # x, dy in; y, dx out; weight, bias in, their gradients out
            return {"bytes": (4 * n * c + 4 * c) * size, "flops": 20 * n * c}
        return {"bytes": (2 * n * c + 2 * c) * size, "flops": 8 * n * c}
    rows_k = sum(_lengths(case))
    rows_q = case["seqs"] if case["op"] == "step" else rows_k
    numbers = 2 * rows_q * case["heads"] * case["dim"] + 2 * rows_k * case["kv_heads"] * case["dim"]
    products = 4 * case["dim"] * case["heads"] * _pairs(case)
    if case.get("train"):  # q, k, v, the output's gradient in; the output and three gradients out
        return {"bytes": 2 * numbers * size, "flops": 7 * products // 2}
    return {"bytes": numbers * size, "flops": products}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "norm":
        x, w, b = s["x"].double(), s["weight"].double(), s["bias"].double()
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        xhat = (x - mean) * torch.rsqrt(var + EPS)
        y = torch.addcmul(b, xhat, w)
        if not case["train"]:
            return [y]
        dy = s["grad"].double()
        g = dy * w
        c = x.size(1)
        dx = (c * g - g.sum(1, keepdim=True) - xhat * torch.einsum("nc,nc->n", g, xhat)[:, None]) * torch.rsqrt(var + EPS) / c
        return [y, dx, torch.einsum("nc,nc->c", dy, xhat), torch.einsum("nc->c", dy)]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    group, scale = h // hk, d ** -0.5
    q, k, v = (s[name].double() for name in ("q", "k", "v"))
    out = torch.zeros_like(q)
    train = bool(case.get("train"))
    do = s["grad"].double() if train else None
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    first_q = first_k = 0
    for n, slot in zip(s["lengths"], s["slots"]):
        n_q = 1 if case["op"] == "step" else n
        rq, rk = slice(first_q, first_q + n_q), slice(first_k, first_k + n)
        keep = torch.ones(n_q, n, dtype=torch.bool, device=DEV)
        if case.get("causal") or case["op"] == "step":
            keep = keep.tril(n - n_q)
        for head in range(h):
            kv = head // group
            logits = torch.where(keep, scale * torch.einsum("id,jd->ij", q[rq, head], k[rk, kv]), float("-inf"))
            p = torch.softmax(logits, 1)
            out[rq, head] = torch.einsum("ij,jd->id", p, v[rk, kv])
            if train:
                g = do[rq, head]
                dp = torch.einsum("id,jd->ij", g, v[rk, kv])
                ds = p * (dp - torch.einsum("ij,ij->i", p, dp)[:, None]) * scale
                dq[rq, head] = torch.einsum("ij,jd->id", ds, k[rk, kv])
                dk[rk, kv] += torch.einsum("ij,id->jd", ds, q[rq, head])
                dv[rk, kv] += torch.einsum("ij,id->jd", p, g)
        first_q, first_k = first_q + n_q, first_k + slot
    return [out, dq, dk, dv] if train else [out]
