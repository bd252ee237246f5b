"""What attention layers over the rows of a sparse tensor need around the product itself, as a program that uses the C++ host
layer (``riemann_cpp``) calls it:

* rotary positions with several axes: pairs of a head's channels turned by the row's coordinates (x, y, z of a voxel; time, height,
  width of a clip's tokens; one place in a text), forward and forward + backward;
* norms of queries and keys for each head with that rotation in the same pass, forward, forward + backward, and for single tokens;
* attention within packed samples with a sliding window and a few first rows that stay visible ("sinks"), forward, forward + backward,
  and single query rows against a cache.

The plain forms are elementary torch operations in 32 bits (the angles in 64), attention over samples padded to one length; ``exact``
goes head by head (and sample by sample) in 64 bits.
"""
import random

import torch

own = False

DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # the voxels of one small object: what a call costs when latency is all there is
        {"name": "rotary-object-f32", "op": "rotary", "dtype": "f32", "rows": 1018, "heads": 4, "dim": 32, "sections": "6,5,5",
         "layout": "voxels", "base": 100.0, "interleaved": False, "train": False},
        # the benchmark's eight rooms at its layer's width, in a training step
        {"name": "rotary-rooms8-bf16-train", "op": "rotary", "dtype": "bf16", "rows": 1_200_000, "heads": 4, "dim": 16,
         "sections": "4,2,2", "layout": "voxels", "base": 100.0, "interleaved": False, "train": True},
        # tokens of a clip: time, height and width, neighbouring channels as pairs, part of the channels without a position
        {"name": "rotary-clip-bf16", "op": "rotary", "dtype": "bf16", "rows": 65_536, "heads": 16, "dim": 80,
         "sections": "8,12,12", "layout": "clip", "base": 10_000.0, "interleaved": True, "train": False},
        # one new token for each of sixteen sequences, far into their contexts: latency
        {"name": "qknorm-step-bf16", "op": "qknorm", "dtype": "bf16", "rows": 16, "heads": 16, "kv_heads": 4, "dim": 128,
         "sections": "64", "layout": "text", "base": 1_000_000.0, "interleaved": False, "train": False},
        # wide token features with fewer key heads, in a training step
        {"name": "qknorm-tokens-bf16-train", "op": "qknorm", "dtype": "bf16", "rows": 16_411, "heads": 16, "kv_heads": 4, "dim": 128,
         "sections": "64", "layout": "text", "base": 1_000_000.0, "interleaved": False, "train": True},
        # a coarser map in fp32, ragged row count, heads that are no power of two, in a training step
        {"name": "qknorm-coarse-f32-train", "op": "qknorm", "dtype": "f32", "rows": 48_503, "heads": 4, "kv_heads": 4, "dim": 24,
         "sections": "4,4,4", "layout": "voxels", "base": 100.0, "interleaved": False, "train": True},
        # one small object's rows in serialised order, fp32: latency
        {"name": "window-object-f32", "op": "window", "dtype": "f32", "seqs": 1, "shortest": 203, "longest": 203, "heads": 4,
         "kv_heads": 4, "dim": 16, "causal": False, "window": 24, "sinks": 1, "train": False},
        # a few small clouds in fp32, in a training step
        {"name": "window-clouds-f32-train", "op": "window", "dtype": "f32", "seqs": 4, "shortest": 301, "longest": 2203,
         "heads": 4, "kv_heads": 4, "dim": 32, "causal": False, "window": 128, "sinks": 2, "train": True},
        # clouds of very different lengths, every row with its neighbours in serialised order, no sinks, in a training step
        {"name": "window-serial-bf16-train", "op": "window", "dtype": "bf16", "seqs": 8, "shortest": 511, "longest": 6007,
         "heads": 8, "kv_heads": 8, "dim": 32, "causal": False, "window": 65, "sinks": 0, "train": True},
        # a batch of texts in a training step, two query heads to a key head, a few first tokens always seen
        {"name": "window-texts-bf16-train", "op": "window", "dtype": "bf16", "seqs": 8, "shortest": 151, "longest": 4001,
         "heads": 8, "kv_heads": 4, "dim": 64, "causal": True, "window": 512, "sinks": 4, "train": True},
        # one long prompt
        {"name": "window-long-bf16", "op": "window", "dtype": "bf16", "seqs": 1, "shortest": 8192, "longest": 8192, "heads": 16,
         "kv_heads": 16, "dim": 128, "causal": True, "window": 1024, "sinks": 4, "train": False},
        # one new token for each of sixteen sequences against what the cache holds of them
        {"name": "window-step-bf16", "op": "step", "dtype": "bf16", "seqs": 16, "shortest": 509, "longest": 30_011, "heads": 16,
         "kv_heads": 4, "dim": 128, "causal": True, "window": 4096, "sinks": 4},
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over the logarithm."""
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def _sections(rng, pairs, axes):
    """Pairs dealt out over the axes: evenly, the first axes take what is left; sometimes a part of the pairs has no position."""
    used = pairs if rng.random() < 0.7 else max(axes, pairs * 3 // 4)
    return ",".join(str(used // axes + (i < used % axes)) for i in range(axes))


def draw(rng):
    kind = rng.choice(("rotary", "rotary-train", "qknorm", "qknorm-train", "window", "window", "window-train", "window-train", "step"))
    op, train = kind.split("-")[0], kind.endswith("-train")
    dtype = rng.choice(("f32", "bf16", "bf16"))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 1, 2, 4))
    if op in ("rotary", "qknorm"):
        dim = rng.choice((16, 24, 32, 48, 64, 80, 96, 128, 2 * rng.randrange(4, 65)))
        axes = rng.randrange(1, 4)
        size = 2 if dtype == "bf16" else 4
        # no more bytes than the benchmark's rooms in a training step
        most = 1_200_000 * 64 * 2 // ((heads + (kv_heads if op == "qknorm" else 0)) * dim * size)
        case = {"op": op, "dtype": dtype, "rows": _spread(rng, 1, max(2, most)), "heads": heads, "dim": dim,
                "sections": _sections(rng, dim // 2, axes), "layout": ("text", "clip", "voxels")[axes - 1] if axes != 2 else "voxels",
                "base": rng.choice((100.0, 10_000.0, 1_000_000.0)), "interleaved": rng.random() < 0.3, "train": train}
        if op == "qknorm":
            case["kv_heads"] = kv_heads
        return case
    sinks = rng.choice((0, 0, 1, 2, 4, 16, 130))
    if op == "step":
        seqs = rng.randrange(1, 17)
        longest = _spread(rng, 16, 30_011)
        return {"op": "step", "dtype": dtype, "seqs": seqs, "shortest": max(1, longest // rng.randrange(1, 60)),
                "longest": longest, "heads": min(heads, 16), "kv_heads": min(kv_heads, 4) if heads > 16 else kv_heads,
                "dim": rng.choice((16, 32, 64, 96, 128)), "causal": True, "window": _spread(rng, 8, 4096), "sinks": sinks}
    seqs = _spread(rng, 1, 32)
    most = int(((16 * 4600 ** 2 * 2) / (2 * heads * seqs)) ** 0.5)
    longest = _spread(rng, 16, max(16, min(most, 8192 if dtype == "bf16" else 2203)))
    return {"op": "window", "dtype": dtype, "seqs": seqs, "shortest": max(1, longest // rng.randrange(1, 40)), "longest": longest,
            "heads": heads, "kv_heads": kv_heads, "dim": rng.choice((16, 24, 32, 48, 64, 80, 96, 128)),
            "causal": rng.random() < 0.5, "window": _spread(rng, 8, max(9, min(1024, longest))), "sinks": sinks, "train": train}


def _lengths(case):
    """The samples' lengths: spread over the logarithm between the two given ones, both among them, in mixed order."""
    rng = random.Random(case["seqs"] * 1_000_003 + case["longest"])
    n = case["seqs"]
    lengths = [_spread(rng, case["shortest"], case["longest"]) for _ in range(n)]
    lengths[0] = case["shortest"]
    lengths[-1] = case["longest"]
    rng.shuffle(lengths)
    return lengths


def _pairs_of(case):
    return [int(n) for n in case["sections"].split(",")]


def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def _positions(case, gen):
    """int32 [rows, axes]; of voxels a view of their coordinates [rows, 1 + axes], whose first column is the sample."""
    n, axes = case["rows"], len(_pairs_of(case))
    if case["layout"] == "voxels":
        coords = torch.randint(-512, 512, (n, 1 + axes), generator=gen, device=DEV, dtype=torch.int32)
        coords[:, 0] = 0
        return coords[:, 1:]
    if case["layout"] == "clip":
        i = torch.arange(n, device=DEV)
        side = 32
        return torch.stack([i // (side * side), i // side % side, i % side], 1).to(torch.int32)
    if n <= 64:  # new tokens, each at the end of a context of its own
        return torch.randint(500, 1_000_000, (n, 1), generator=gen, device=DEV, dtype=torch.int32)
    return torch.arange(n, device=DEV, dtype=torch.int32)[:, None] + 100_000


def _frequencies(case):
    """Radians a unit of position, float64, one for each pair: of a clip over all pairs together, else axis by axis."""
    pairs, out = _pairs_of(case), []
    for n in pairs:
        start, whole = (len(out), sum(pairs)) if case["layout"] == "clip" else (0, n)
        out += [case["base"] ** (-(start + i) / whole) for i in range(n)]
    return torch.tensor(out, dtype=torch.float64, device=DEV)


def _inputs(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dtype, h, d = DTYPES[case["dtype"]], case["heads"], case["dim"]
    if case["op"] in ("rotary", "qknorm"):
        n, hk = case["rows"], case.get("kv_heads", 0)
        # the heads of one projection behind a layer: channels with scales of their own
        spread = _randn(gen, (d,), torch.float32).abs() + 0.3
        both = (torch.randn((n, h + hk, d), generator=gen, device=DEV) * spread).to(dtype)
        s = {"x": both[:, :h], "positions": _positions(case, gen), "frequencies": _frequencies(case)}
        if hk:
            s["k"] = both[:, h:]
            s["wq"], s["wk"] = (_randn(gen, (d,), dtype, 0.2) + 1 for _ in range(2))
        if case["train"]:
            s["grad"] = _randn(gen, (n, h, d), dtype, 0.1)
            if hk:
                s["grad_k"] = _randn(gen, (n, hk, d), dtype, 0.1)
        return s
    lengths, hk = _lengths(case), case["kv_heads"]
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
    if s["op"] in ("rotary", "qknorm"):
        s["sections"], s["interleaved"] = _pairs_of(case), case["interleaved"]
        leaves = ("x", "k", "wq", "wk") if s["op"] == "qknorm" else ("x",)
    else:
        starts = [0]
        for n in s["slots"]:
            starts.append(starts[-1] + n)
        s["kv_offsets"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
        s["kv_lengths"] = torch.tensor(s["lengths"], dtype=torch.int32, device=DEV)
        s["offsets"] = s["kv_offsets"]
        if case["op"] == "step":
            s["offsets"] = torch.arange(len(s["lengths"]) + 1, dtype=torch.int32, device=DEV)
        s["longest"], s["causal"], s["window"], s["sinks"] = max(s["lengths"]), case["causal"], case["window"], case["sinks"]
        leaves = ("q", "k", "v")
    if s["train"]:
        for name in leaves:
            s[name] = s[name].detach().requires_grad_(True)
    return s


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _plain_rotary(state) if state["op"] in ("rotary", "qknorm") else _plain_attention(state)


def _run_own(s):
    from riemannengine_b200 import cpp
    host = cpp.load()
    if s["op"] == "rotary":
        out = host.rotary_positions(s["x"], s["positions"], s["frequencies"], s["sections"], interleaved=s["interleaved"])
        if not s["train"]:
            return [out]
        return [out.detach(), *torch.autograd.grad(out, (s["x"],), s["grad"])]
    if s["op"] == "qknorm":
        q, k = host.qk_norm_rotary(s["x"], s["k"], s["wq"], s["wk"], s["positions"], s["frequencies"], s["sections"], eps=EPS,
                                   interleaved=s["interleaved"])
        if not s["train"]:
            return [q, k]
        leaves = (s["x"], s["k"], s["wq"], s["wk"])
        return [q.detach(), k.detach(), *torch.autograd.grad((q, k), leaves, (s["grad"], s["grad_k"]))]
    if s["op"] == "step":
        return [host.packed_attention(s["q"], s["k"], s["v"], s["offsets"], kv_offsets=s["kv_offsets"],
                                      kv_lengths=s["kv_lengths"], causal=True, window=s["window"], sinks=s["sinks"])]
    leaves = (s["q"], s["k"], s["v"])
    out = host.packed_attention(*leaves, s["offsets"], causal=s["causal"], window=s["window"], sinks=s["sinks"])
    if not s["train"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, leaves, s["grad"])]


def _turn(x, cos, sin, interleaved):
    """The pairs of the first channels turned, the others as they are."""
    pairs = cos.size(-1)
    cos, sin = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., 2 * pairs:]), -1)


def _plain_rotary(s):
    axis = torch.tensor([a for a, n in enumerate(s["sections"]) for _ in range(n)], device=DEV)
    angle = s["positions"].double()[:, axis] * s["frequencies"]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    outs, grads, weights = [], [], []
    for name, weight, grad in (("x", "wq", "grad"), ("k", "wk", "grad_k")):
        if name not in s:
            continue
        x = s[name].float()
        hat, w = x, None
        if weight in s:
            w = s[weight].float()
            inv = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
            hat = x * inv
        outs.append(_turn(hat if w is None else hat * w, cos, sin, s["interleaved"]).to(s[name].dtype))
        if not s["train"]:
            continue
        g = _turn(s[grad].float(), cos, -sin, s["interleaved"])
        if w is not None:
            weights.append((g * hat).sum((0, 1)).to(s[weight].dtype))
            g = g * w
            g = inv * (g - hat * (g * hat).mean(-1, keepdim=True))
        grads.append(g.to(s[name].dtype))
    return outs + grads + weights


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
    place = i + (n_k - n_q)[:, None, None]
    seen = (i < n_q[:, None, None]) & (j < n_k[:, None, None])
    seen = seen & (((place - j).abs() < s["window"]) | (j < s["sinks"]))
    if s["causal"]:
        seen = seen & (j <= place)
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
    at = rows - s["offsets"][:-1].long()[sample]

    def packed(x, length, dtype):
        return x.view(samples, -1, length, d)[sample, :, at].to(dtype)

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


def _seen(p, m, case):
    """How many of m keys the query at place p sees."""
    first = max(0, p - case["window"] + 1)  # (below end: p is a key's place)
    end = min(m, p + 1 if case["causal"] else p + case["window"])
    sinks = min(case["sinks"], m, p + 1 if case["causal"] else m)
    return end - first + min(sinks, first) + max(0, sinks - end)


def _visible(case):
    """(query, key) pairs of one head, and the key rows that some query sees."""
    pairs = keys = 0
    for m in _lengths(case):
        if case["op"] == "step":
            pairs, keys = pairs + _seen(m - 1, m, case), keys + _seen(m - 1, m, case)
            continue
        # rows near the ends one by one, those between see the same number of keys
        edge = case["window"] + case["sinks"]
        if m <= 2 * edge:
            pairs += sum(_seen(p, m, case) for p in range(m))
        else:
            pairs += sum(_seen(p, m, case) for p in (*range(edge), *range(m - edge, m))) + (m - 2 * edge) * _seen(edge, m, case)
        keys += m
    return pairs, keys


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] in ("rotary", "qknorm"):
        pairs, heads = _pairs_of(case), case["heads"] + case.get("kv_heads", 0)
        n, numbers = case["rows"], case["rows"] * heads * case["dim"]
        small = n * 4 * len(pairs) + 8 * sum(pairs) + (2 * case["dim"] * size if case["op"] == "qknorm" else 0)
        flops = n * sum(pairs) * (6 * heads + 20) + (4 * numbers if case["op"] == "qknorm" else 0)
        if not case["train"]:
            return {"bytes": 2 * numbers * size + small, "flops": flops}
        # a rotation alone needs no x again for its gradient
        more = 4 if case["op"] == "qknorm" else 3 + 1
        return {"bytes": more * numbers * size + small + (2 * case["dim"] * size if case["op"] == "qknorm" else 0), "flops": 3 * flops}
    pairs, rows_k = _visible(case)
    rows_q = case["seqs"] if case["op"] == "step" else rows_k
    numbers = 2 * rows_q * case["heads"] * case["dim"] + 2 * rows_k * case["kv_heads"] * case["dim"]
    products = 4 * case["dim"] * case["heads"] * pairs
    if case.get("train"):  # q, k, v, the output's gradient in; the output and three gradients out
        return {"bytes": 2 * numbers * size, "flops": 7 * products // 2}
    return {"bytes": numbers * size, "flops": products}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] in ("rotary", "qknorm"):
        return _exact_rotary(case, s)
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
        ones = torch.ones(n_q, n, dtype=torch.bool, device=DEV)
        keep = ones.triu(n - n_q - case["window"] + 1) & ones.tril(n - n_q + case["window"] - 1)
        keep[:, :case["sinks"]] = True
        if case["causal"]:
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


def _exact_rotary(case, s):
    """A pair as a complex number, turned by exp(i angle), head by head."""
    pairs = _pairs_of(case)
    total, places = sum(pairs), s["positions"].double()
    angle = torch.cat([places[:, a:a + 1] * f for a, f in enumerate(s["frequencies"].split(pairs))], 1)
    turn = torch.polar(torch.ones_like(angle), angle)
    order = torch.arange(2 * total, device=DEV)
    order = order.view(total, 2) if case["interleaved"] else order.view(2, total).T

    def turned(x, by):
        y = x.clone()
        z = torch.complex(x[:, order[:, 0]], x[:, order[:, 1]]) * by
        y[:, order[:, 0]], y[:, order[:, 1]] = z.real, z.imag
        return y

    outs, grads, weights = [], [], []
    for x, w, g in ((s["x"], s.get("wq"), s.get("grad")), (s.get("k"), s.get("wk"), s.get("grad_k"))):
        if x is None:
            continue
        out, dx = (torch.empty(x.shape, dtype=torch.float64, device=DEV) for _ in range(2))
        dw = torch.zeros(case["dim"], dtype=torch.float64, device=DEV)
        for head in range(x.size(1)):
            a = x[:, head].double()
            inv = torch.ones_like(a[:, :1]) if w is None else (a.square().mean(1, keepdim=True) + EPS).rsqrt()
            out[:, head] = turned(a * inv * (1.0 if w is None else w.double()), turn)
            if g is None:
                continue
            b = turned(g[:, head].double(), turn.conj())
            if w is None:
                dx[:, head] = b
                continue
            dw += torch.einsum("nd,nd->d", b, a * inv)
            b = b * w.double()
            dx[:, head] = b * inv - a * inv ** 3 * torch.einsum("nd,nd->n", a, b)[:, None] / case["dim"]
        outs.append(out)
        if g is not None:
            grads.append(dx)
            if w is not None:
                weights.append(dw)
    return outs + grads + weights
