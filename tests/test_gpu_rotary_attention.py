"""Norms of heads, rotary positions and attention with a window run together, as a network and as a loop over single tokens run them:
the layer on sparse tensors against 64 bits, its gradients against the formula's, and a captured step over a cache against the same."""
import pytest
import torch

from tests import plain_rotary as R
from tests import plain_window as W
from tests.plain_tokens import U32, check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _host(name):
    if name == "cpp":
        from riemannengine_b200 import cpp
        return cpp.load()
    from riemannengine_b200 import engine
    return engine


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _turned(x, positions, frequencies, sections):
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    angle = (positions.double()[:, axis] * frequencies)[:, None]
    n = len(axis)
    a, b = x[..., :n], x[..., n:2 * n]
    return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), x[..., 2 * n:]], 2)


@pytest.mark.parametrize("host", ["python", "cpp"])
@pytest.mark.parametrize("rotary,norm,window,sinks,causal", [(100.0, True, 9, 2, True), (100.0, False, 5, 0, False),
                                                             (None, True, None, 0, True), (50.0, True, None, 0, False),
                                                             (None, False, 1, 1, True)])
def test_layer(host, rotary, norm, window, sinks, causal):
    H = _host(host)
    coords = torch.tensor([[7, 3 * i, -i, 2] for i in range(60)] + [[3, i, 1, -i * i] for i in range(90)], dtype=torch.int32, device=DEV)
    x = torch.randn(150, 64, generator=_gen(11), device=DEV)
    tensor = H.SparseTensor(x.requires_grad_(True), coords)
    torch.manual_seed(5)
    layer = H.RiemannSelfAttention(64, 4, 2, causal=causal, rotary_base=rotary, qk_norm=norm, window=window, sinks=sinks)
    layer.to(DEV)
    p = dict(layer.named_parameters().items()) if host == "cpp" else dict(layer.named_parameters())
    assert ("q_norm" in p) == ("k_norm" in p) == norm
    if norm:
        with torch.no_grad():
            p["q_norm"].copy_(1 + torch.rand(16, generator=_gen(2), device=DEV))
            p["k_norm"].copy_(1 + torch.rand(16, generator=_gen(3), device=DEV))
    y = layer(tensor)
    y.F.square().sum().backward()
    leaves = {k: v.detach().double().requires_grad_(True) for k, v in p.items()}
    X = x.detach().double().requires_grad_(True)
    q, k, v = (X @ leaves["qkv.weight"].T + leaves["qkv.bias"]).view(150, 8, 16).split([4, 2, 2], 1)
    if norm:
        q, k = (t * (t.square().mean(2, keepdim=True) + 1e-6).rsqrt() * leaves[w] for t, w in ((q, "q_norm"), (k, "k_norm")))
    if rotary:
        sections = H.rotary_sections(16, 3)
        assert sum(sections) == 8
        frequencies = H.rotary_frequencies(sections, rotary).to(DEV)
        q, k = (_turned(t, coords[:, 1:], frequencies, sections) for t in (q, k))
    rows = []
    for a, b in ((0, 60), (60, 150)):
        s = torch.einsum("ihd,jhd->hij", q[a:b], k[a:b].repeat_interleave(2, 1)) / 4
        s = s.masked_fill(~W.seen(b - a, b - a, 1 << 20 if window is None else window, sinks, causal, DEV), float("-inf"))
        rows.append(torch.einsum("hij,jhd->ihd", s.softmax(-1), v[a:b].repeat_interleave(2, 1)).reshape(b - a, 64))
    want = torch.cat(rows) @ leaves["projection.weight"].T + leaves["projection.bias"]
    want.square().sum().backward()
    # four products of 64 terms and one of up to 90 behind one another, each off by its terms times u of values of order 1 ... 10; a norm
    # divides by a root of a mean square of no less than 1 / 10
    tol = 10 * 64 * 5 * U32 * (10 if norm else 1)
    assert (y.F.double() - want).abs().max() <= tol
    for name, got in [("x", x), *p.items()]:
        ref = X.grad if name == "x" else leaves[name].grad
        assert (got.grad.double() - ref).abs().max() <= 4 * tol * ref.abs().max() + 150 * tol, name


@pytest.mark.parametrize("host", ["python", "cpp"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tokens_one_by_one(host, dtype):
    """Three sequences, fed whole for some tokens and then one token at a time by a captured step over a cache; rows of the cache behind
    a sequence's length are NaN."""
    H = _host(host)
    h, hk, d, room, window, sinks, steps = 4, 2, 64, 80, 12, 3, 6
    lengths = [1, 17, 64]
    sections = H.rotary_sections(d, 1)
    frequencies = H.rotary_frequencies(sections).to(DEV)
    wq, wk = (1 + torch.rand(d, generator=_gen(s), device=DEV).to(dtype) for s in (1, 2))
    rows = sum(lengths)
    cache_k, cache_v = (torch.full((3 * room, hk, d), float("nan"), device=DEV, dtype=dtype) for _ in range(2))
    starts = torch.tensor([0, room, 2 * room, 3 * room], dtype=torch.int32, device=DEV)
    offsets = torch.tensor([0, 1, 18, 82], dtype=torch.int32, device=DEV)
    held = torch.tensor(lengths, dtype=torch.int32, device=DEV)

    def fresh(n, seed):
        g = _gen(seed)
        return [torch.randn(n, heads, d, generator=g, device=DEV).to(dtype) for heads in (h, hk, hk)]

    def attend(q, k, v, positions, slots, rows_of):
        q, k = H.qk_norm_rotary(q, k, wq, wk, positions, frequencies, sections)
        cache_k.index_copy_(0, slots, k)
        cache_v.index_copy_(0, slots, v)
        return q, H.packed_attention(q, cache_k, cache_v, rows_of, starts, held, True, None, window, sinks)

    def verify(raw, positions, q, out, slots, rows_of, name):
        want = R.rotary(raw[0], raw[1], positions, frequencies, sections, norm=True, wq=wq, wk=wk)
        check(q, want["q"], name + " q")
        check(cache_k[slots], want["k"], name + " k")
        seen = W.attention(q, cache_k.nan_to_num(), cache_v.nan_to_num(), rows_of, starts, held, True, None, window, sinks)
        check(out, seen["out"], name + " out")

    with torch.no_grad():
        raw = fresh(rows, 10)
        place = torch.cat([torch.arange(n, device=DEV) for n in lengths])
        slots = torch.cat([room * i + torch.arange(n, device=DEV) for i, n in enumerate(lengths)])
        positions = place.int()[:, None]
        q, out = attend(*raw, positions, slots, offsets)
        verify(raw, positions, q, out, slots, offsets, "whole")

        one = torch.arange(4, dtype=torch.int32, device=DEV)
        static = fresh(3, 0)
        slot = torch.zeros(3, dtype=torch.int64, device=DEV)
        kept_k, kept_v, kept_held = cache_k.clone(), cache_v.clone(), held.clone()

        def step():
            positions = held[:, None].clone()
            slot.copy_(starts[:3] + held)
            held.add_(1)
            return positions, *attend(*static, positions, slot, one)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            positions, q, out = step()
        cache_k.copy_(kept_k), cache_v.copy_(kept_v), held.copy_(kept_held)
        for i in range(steps):
            raw = fresh(3, 20 + i)
            for there, now in zip(static, raw):
                there.copy_(now)
            graph.replay()
            assert held.tolist() == [n + i + 1 for n in lengths]
            verify(raw, positions, q, out, slot, one, "step %d" % i)


@pytest.mark.parametrize("host", ["python", "cpp"])
def test_layer_refusals(host):
    H = _host(host)
    for arguments in (dict(channels=12, num_heads=4, rotary_base=100.0), dict(channels=12, num_heads=4, qk_norm=True),
                      dict(channels=1032, num_heads=4, qk_norm=True), dict(channels=64, num_heads=4, rotary_base=0.0),
                      dict(channels=64, num_heads=4, sinks=2), dict(channels=64, num_heads=4, window=0),
                      dict(channels=64, num_heads=4, window=4, sinks=-1)):
        with pytest.raises((RuntimeError, ValueError)):
            H.RiemannSelfAttention(**arguments)
