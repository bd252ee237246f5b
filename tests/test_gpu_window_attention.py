"""Attention with a sliding window and sinks: both hosts against 64 bits, forward and backward, at the lengths, windows, masks and
offsets where it can go wrong."""
import ctypes

import pytest
import torch

from tests import plain_window as W
from tests.plain_tokens import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _host(name):
    if name == "cpp":
        from riemannengine_b200 import cpp
        return cpp.load().packed_attention
    from riemannengine_b200 import engine
    return engine.packed_attention


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _offsets(lengths, first=0):
    o = [first]
    for n in lengths:
        o.append(o[-1] + n)
    return torch.tensor(o, dtype=torch.int32, device=DEV)


def _inputs(rows_q, rows_k, h, hk, d, dtype, seed=0):
    g = _gen(seed * 1009 + rows_q * 13 + rows_k * 7 + h * 3 + d)
    r = lambda n, m: torch.randn(n, m, d, generator=g, device=DEV).to(dtype)  # noqa: E731
    return r(rows_q, h), r(rows_k, hk), r(rows_k, hk), r(rows_q, h)


def _check(host, q, k, v, grad, offsets, window, sinks, kv_offsets=None, kv_lengths=None, causal=False, scale=None, what="", clean=None):
    """clean: keys and values with what is never read replaced, for the bounds."""
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    f = _host(host)
    out = f(*leaves, offsets, kv_offsets, kv_lengths, causal, scale, window=window, sinks=sinks)
    assert out.is_contiguous() and out.dtype == q.dtype
    grads = torch.autograd.grad(out, leaves, grad)
    want = W.attention(q, *(clean or (k, v)), offsets, kv_offsets, kv_lengths, causal, scale, window, sinks, grad)
    what = f"{what} window {window} sinks {sinks} causal {causal}"
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        check(got, want[name], f"{name} {what}")
    with torch.no_grad():
        again = f(q, k, v, offsets, kv_offsets, kv_lengths, causal, scale, window=window, sinks=sinks)
    check(again, want["out"], f"inference {what}")
    return out, *grads


LENGTHS = {"one": [1], "short": [1, 0, 2, 31, 33], "tiles": [63, 64, 65], "wide": [127, 128, 129, 1], "long": [300, 0, 520, 17],
           "longer": [1100]}
# windows of one key, around a tile, longer than the samples; sinks that meet the window, end inside a tile, fill tiles, pass the sample
WINDOWS = [(1, 0), (1, 3), (2, 1), (17, 4), (63, 0), (64, 64), (65, 1), (100, 130), (128, 4), (129, 128), (200, 0), (257, 257), (5000, 2),
           (2**31 - 1, 0), (3, 2**30 - 1)]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("h,hk,d", [(2, 2, 32), (4, 1, 64), (2, 1, 128)])
def test_windows(lengths, h, hk, d, dtype, causal):
    lens = LENGTHS[lengths]
    q, k, v, grad = _inputs(sum(lens), sum(lens), h, hk, d, TYPES[dtype])
    for window, sinks in WINDOWS:
        _check("cpp", q, k, v, grad, _offsets(lens), window, sinks, causal=causal)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [1, 8, 20, 24, 33, 48, 72, 96, 112, 130, 256])
def test_head_sizes(d, dtype):
    lens = [70, 340]
    q, k, v, grad = _inputs(410, 410, 4, 2, d, TYPES[dtype])
    _check("cpp", q, k, v, grad, _offsets(lens), 50, 5, causal=True)
    _check("cpp", q, k, v, grad, _offsets(lens), 90, 1, causal=False)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("h,hk,d", [(3, 1, 64), (6, 1, 128), (16, 2, 64), (32, 2, 40), (11, 1, 16)])
def test_many_query_heads_to_a_key_head(h, hk, d, dtype, causal):
    lens = [40, 0, 557, 130]
    q, k, v, grad = _inputs(727, 727, h, hk, d, TYPES[dtype])
    _check("cpp", q, k, v, grad, _offsets(lens), 70, 6, causal=causal)


@pytest.mark.parametrize("host", ["python", "cpp"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_views(host, dtype):
    """Parts of one projection, aligned and not; heads first, channels that are not adjacent, one head for all."""
    t, h, hk, d, lens = TYPES[dtype], 4, 2, 64, [150, 3, 300]
    n = sum(lens)
    g = _gen(d)
    for extra, first in ((0, 0), (8, 8), (3, 1)):
        whole = torch.randn(n, (h + 2 * hk) * d + extra, generator=g, device=DEV).to(t)
        q, k, v = whole[:, first:first + (h + 2 * hk) * d].unflatten(1, (h + 2 * hk, d)).split([h, hk, hk], 1)
        grad = torch.randn(h, n, d, generator=g, device=DEV).to(t).transpose(0, 1)
        _check(host, q, k, v, grad, _offsets(lens), 40, 3, causal=True, what=f"first {first}")
    q = torch.randn(h, n, d, generator=g, device=DEV).to(t).transpose(0, 1)
    k = torch.randn(n, d, hk, generator=g, device=DEV).to(t).transpose(1, 2)
    v = torch.randn(n, 1, d, generator=g, device=DEV).to(t).expand(n, hk, d)
    grad = torch.randn(1, 1, d, generator=g, device=DEV).to(t).expand(n, h, d)
    _check(host, q, k, v, grad, _offsets(lens), 40, 3, what="expanded")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_keys_of_their_own_in_a_cache_with_room(dtype, causal, d):
    """Other key rows than query rows (fewer and more), slots longer than what is in use, NaN behind it; rows before the first sample and
    behind the last, which are zeros; rows that see nothing."""
    nq, nk, slots = [3, 1, 0, 200, 40, 7, 300], [130, 1, 64, 77, 0, 300, 900], [150, 4, 64, 90, 10, 301, 1000]
    t = TYPES[dtype]
    q, k, v, grad = _inputs(sum(nq) + 12, sum(slots) + 9, 4, 2, d, t)
    offsets, kv_offsets = _offsets(nq, 5), _offsets(slots, 4)
    kv_lengths = torch.tensor(nk, dtype=torch.int32, device=DEV)
    clean = [k.clone(), v.clone()]
    unused = torch.ones(k.size(0), dtype=torch.bool, device=DEV)
    for a, n in zip(kv_offsets.tolist(), nk):
        unused[a:a + n] = False
    k[unused], v[unused] = float("nan"), float("inf")
    for c in clean:
        c[unused] = 0
    for window, sinks in ((1, 0), (30, 2), (128, 64), (400, 200)):
        out, dq, dk, dv = _check("cpp", q, k, v, grad, offsets, window, sinks, kv_offsets, kv_lengths, causal, clean=clean)
        for rows in (out, dq):
            assert not rows[:5].any() and not rows[5 + sum(nq):].any() and not rows[5 + 204:5 + 244].any()
        assert not dk[unused].any() and not dv[unused].any()
        if causal:
            assert not out[5 + 4:5 + 4 + 123].any()  # 200 queries, 77 keys
        elif sinks == 0:
            assert not out[5 + 4:5 + 4 + 123 - window + 1].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("h,hk,d", [(4, 4, 32), (8, 2, 64), (16, 4, 128), (4, 1, 96)])
def test_few_new_rows_against_a_cache(h, hk, d, dtype):
    """One and a few new rows a sample, keys from one to thousands, NaN wherever no key is to be read."""
    t = TYPES[dtype]
    nk = [1, 5, 64, 65, 700, 3001, 130, 0, 2048, 90]
    slots = [n + 7 for n in nk]
    for rows in (1, 2, 5):
        nq = [rows] * len(nk)
        q, k, v, _ = _inputs(sum(nq), sum(slots), h, hk, d, t)
        offsets, kv_offsets = _offsets(nq), _offsets(slots)
        kv_lengths = torch.tensor(nk, dtype=torch.int32, device=DEV)
        for window, sinks, causal in ((1, 0, True), (20, 4, True), (64, 0, True), (500, 130, True), (4096, 4, True), (64, 3, False)):
            K, V = k.clone(), v.clone()
            for a, n, s in zip(kv_offsets.tolist(), nk, slots):
                K[a + n:a + s], V[a + n:a + s] = float("nan"), float("nan")
            got = _host("cpp")(q, K, V, offsets, kv_offsets, kv_lengths, causal, window=window, sinks=sinks)
            want = W.attention(q, k, v, offsets, kv_offsets, kv_lengths, causal, None, window, sinks)["out"]
            check(got, want, f"{rows} rows, window {window} sinks {sinks}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_samples(dtype):
    """More samples than are counted one by one, of uneven lengths."""
    g = torch.Generator().manual_seed(4)
    lens = torch.randint(0, 90, (500,), generator=g).tolist()
    n = sum(lens)
    q, k, v, grad = _inputs(n, n, 4, 2, 32, TYPES[dtype])
    _check("cpp", q, k, v, grad, _offsets(lens), 12, 2, causal=True)
    _check("cpp", q, k, v, grad, _offsets(lens), 70, 0, causal=False)


@pytest.mark.parametrize("samples", [29, 30, 31, 33, 383, 385])
def test_numbers_of_samples(samples):
    """Up to as many as a warp counts, as a block counts, and beyond; samples of no rows, rows before the first and behind the last, and
    one sample long enough for parts of its sinks' gradients."""
    lens = [(7 * i) % 5 * (i % 3) for i in range(samples)]
    lens[samples // 2] = 700
    n = sum(lens) + 9
    q, k, v, grad = _inputs(n, n, 4, 2, 48, torch.bfloat16)
    _check("cpp", q, k, v, grad, _offsets(lens, 4), 33, 2, causal=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_sinks_of_long_samples(dtype, d, causal):
    """Sinks that thousands of queries see, with one, several and many query heads to a key head; other samples beside them."""
    lens = [2500, 3, 1700, 513]
    n = sum(lens)
    for h, hk in ((2, 2), (4, 1)):
        q, k, v, grad = _inputs(n, n, h, hk, d, TYPES[dtype])
        for window, sinks in ((130, 4), (64, 129), (40, 700)):
            _check("cpp", q, k, v, grad, _offsets(lens), window, sinks, causal=causal)


def test_a_window_over_everything_is_no_window():
    """The same sums as without a window, up to roundings: sinks of all keys, or a window that reaches them."""
    lens = [300, 130]
    for dtype in TYPES.values():
        q, k, v, grad = _inputs(430, 430, 4, 2, 64, dtype)
        for causal in (False, True):
            want = W.attention(q, k, v, _offsets(lens), None, None, causal, None, 1000, 0, grad)
            for window, sinks in ((300, 0), (1, 300)):
                leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
                out = _host("cpp")(*leaves, _offsets(lens), causal=causal, window=window, sinks=sinks)
                for name, got in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, grad))):
                    check(got, want[name], name)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_same_bits_every_time_on_any_stream(dtype):
    lens = [900, 1300, 77]
    n = sum(lens)
    q, k, v, grad = _inputs(n, n, 8, 2, 64, TYPES[dtype])
    offsets = _offsets(lens)

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = _host("cpp")(*leaves, offsets, causal=True, window=100, sinks=4)
        return [out, *torch.autograd.grad(out, leaves, grad)]

    first = step()
    side = torch.cuda.Stream()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            second = step()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, second))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_captured_and_replayed(dtype):
    """A training step and a step of new rows in graphs, replayed over new inputs, offsets and lengths."""
    t, most = TYPES[dtype], 700
    q, k, v, grad = _inputs(most, most, 4, 2, 64, t)
    offsets = _offsets([300, 400])
    lengths = torch.tensor([300, 400], dtype=torch.int32, device=DEV)
    ones = _offsets([1, 1])
    f = _host("cpp")

    def step():
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out = f(*leaves, offsets, causal=True, window=50, sinks=3)
        new = f(q[:2], k, v, ones, offsets, lengths, True, window=50, sinks=3)
        return [out, *torch.autograd.grad(out, leaves, grad), new]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed, lens in ((1, [690, 10]), (2, [0, 700]), (3, [350, 350])):
        for x, n in zip((q, k, v, grad), _inputs(most, most, 4, 2, 64, t, seed)):
            x.copy_(n)
        offsets.copy_(_offsets(lens))
        lengths.copy_(torch.tensor([max(0, n - 5) for n in lens], dtype=torch.int32))
        graph.replay()
        want = W.attention(q, k, v, offsets, None, None, True, None, 50, 3, grad)
        for name, got in zip(("out", "dq", "dk", "dv"), outs):
            check(got, want[name], f"{name} {lens}")
        check(outs[4], W.attention(q[:2], k, v, ones, offsets, lengths, True, None, 50, 3)["out"], f"new {lens}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_offsets_that_make_no_sense_are_reported(dtype):
    """They are clamped on the device, and the status word says so."""
    from riemannengine_b200 import capi
    t, lib = TYPES[dtype], capi.lib()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.rmn_device_status(stream) == capi.OK
    for bad in ([0, 300, 100], [-50, 100, 200], [0, 100, 5000], [200, 100, 0]):
        q, k, v, grad = _inputs(200, 200, 2, 1, 64, t)
        offsets = torch.tensor(bad, dtype=torch.int32, device=DEV)
        leaves = [x.requires_grad_(True) for x in (q, k, v)]
        for causal in (False, True):
            out = _host("cpp")(*leaves, offsets, causal=causal, window=20, sinks=2)
            torch.autograd.grad(out, leaves, grad)
            assert lib.rmn_device_status(stream) == capi.ERR_BAD_ARG, bad
            assert lib.rmn_device_status(stream) == capi.OK
        with torch.no_grad():
            _host("cpp")(q[:2], k, v, torch.arange(3, dtype=torch.int32, device=DEV), offsets, causal=True, window=20, sinks=2)
        assert lib.rmn_device_status(stream) == capi.ERR_BAD_ARG, bad
    # and calls that make sense work behind it
    q, k, v, grad = _inputs(200, 200, 2, 1, 64, t)
    _check("cpp", q, k, v, grad, _offsets([150, 50]), 20, 2, causal=True)


@pytest.mark.parametrize("host", ["python", "cpp"])
def test_refusals_and_second_derivatives(host):
    f = _host(host)
    q, k, v, _ = _inputs(10, 10, 2, 2, 16, torch.float32)
    o = _offsets([10])
    for window, sinks, text in ((0, 0, "window must be"), (-3, 0, "window must be"), (2**31, 0, "window must be"), (4, -1, "window must be"),
                                (4, 2**30, "window must be"), (None, 2, "sinks need")):
        with pytest.raises(RuntimeError, match=text):
            f(q, k, v, o, window=window, sinks=sinks)
    q.requires_grad_(True)
    grad = torch.autograd.grad(f(q, k, v, o, window=3, sinks=1).sum(), q, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="packed_attention is differentiable once only"):
        grad.sum().backward()


def test_gradients_against_differences():
    """The loss along a direction, by differences of the 64-bit form, against the kernels' gradients."""
    lens = [60, 41]
    q, k, v, grad = _inputs(101, 101, 4, 2, 32, torch.float32)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    g = _gen(9)
    steps = [torch.randn(t.shape, generator=g, device=DEV).double() for t in leaves]
    for causal in (False, True):
        out = _host("cpp")(*leaves, _offsets(lens), causal=causal, window=15, sinks=2)
        grads = torch.autograd.grad(out, leaves, grad)

        def loss(by):
            a = [t.detach().double() + by * s for t, s in zip(leaves, steps)]
            return (W.attention(*a, _offsets(lens), None, None, causal, None, 15, 2)["out"][0] * grad.double()).sum().item()

        e = 1e-4
        slope = (loss(e) - loss(-e)) / (2 * e)
        terms = [(a.double() * s) for a, s in zip(grads, steps)]
        # differences: e^2 / 6 of a third derivative, of the size of the terms here; gradients: 2^-20 of the terms' sizes
        assert abs(slope - sum(t.sum() for t in terms).item()) <= sum(t.abs().sum() for t in terms).item() * (2.0 ** -20 + 1e-6)
