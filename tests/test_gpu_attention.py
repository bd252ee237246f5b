"""Attention within packed samples: both hosts against 64 bits, forward and backward, at the lengths, strides, masks and offsets
where it can go wrong."""
import ctypes

import pytest
import torch

from tests import plain_tokens as P

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


def _check(host, q, k, v, grad, offsets, kv_offsets=None, kv_lengths=None, causal=False, scale=None, what="", bound_k=None, bound_v=None):
    """bound_k, bound_v: the keys and values with what is never read replaced, for the bounds."""
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = _host(host)(*leaves, offsets, kv_offsets, kv_lengths, causal, scale)
    assert out.is_contiguous() and out.dtype == q.dtype
    dq, dk, dv = torch.autograd.grad(out, leaves, grad)
    want = P.attention(q, k if bound_k is None else bound_k, v if bound_v is None else bound_v, offsets, kv_offsets, kv_lengths,
                       causal, scale, grad)
    for name, got in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        P.check(got, want[name], f"{name} {what}")
    with torch.no_grad():  # without the backward pass's needs
        again = _host(host)(q, k, v, offsets, kv_offsets, kv_lengths, causal, scale)
    P.check(again, want["out"], f"inference {what}")
    return out, dq, dk, dv


LENGTHS = {"one": [1], "few": [5], "short": [1, 0, 2, 31, 33], "tiles": [63, 64, 65], "wide": [127, 128, 129, 1],
           "long": [300, 0, 520, 17]}


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("h,hk,d", [(2, 2, 32), (4, 1, 64), (3, 3, 128), (4, 2, 16)])
def test_packed_samples(lengths, h, hk, d, dtype, causal):
    lens = LENGTHS[lengths]
    n = sum(lens)
    q, k, v, grad = _inputs(n, n, h, hk, d, TYPES[dtype])
    _check("cpp", q, k, v, grad, _offsets(lens), causal=causal)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [1, 3, 8, 20, 24, 33, 40, 48, 72, 80, 96, 100, 112, 120, 130, 192, 256])
def test_head_sizes(d, dtype):
    lens = [70, 140]
    q, k, v, grad = _inputs(210, 210, 4, 2, d, TYPES[dtype])
    _check("cpp", q, k, v, grad, _offsets(lens), causal=True, what=f"dim {d}")


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("h,hk,d", [(3, 1, 64), (6, 1, 128), (5, 1, 32), (16, 2, 64), (14, 2, 80), (32, 2, 40), (11, 1, 16), (22, 2, 128)])
def test_many_query_heads_to_a_key_head(h, hk, d, dtype, causal):
    """Groups of every kind: that divide into up to eight blocks, and (11 heads) that do not."""
    lens = [40, 0, 257, 130]
    q, k, v, grad = _inputs(427, 427, h, hk, d, TYPES[dtype])
    _check("cpp", q, k, v, grad, _offsets(lens), causal=causal)


@pytest.mark.parametrize("host", ["python", "cpp"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_views_of_one_projection(host, dtype, d):
    """q, k and v as parts of one matrix, with a gradient whose heads come first, and unaligned ones."""
    t, h, hk, lens = TYPES[dtype], 4, 2, [150, 3, 200]
    n = sum(lens)
    g = _gen(d)
    for extra, first in ((0, 0), (8, 8), (3, 1)):
        whole = torch.randn(n, (h + 2 * hk) * d + extra, generator=g, device=DEV).to(t)
        parts = whole[:, first:first + (h + 2 * hk) * d].unflatten(1, (h + 2 * hk, d))
        q, k, v = parts.split([h, hk, hk], 1)
        grad = torch.randn(h, n, d, generator=g, device=DEV).to(t).transpose(0, 1)
        _check(host, q, k, v, grad, _offsets(lens), causal=True, what=f"first {first}")
    # heads first, channels not adjacent, one head for all
    q = torch.randn(h, n, d, generator=g, device=DEV).to(t).transpose(0, 1)
    k = torch.randn(n, d, hk, generator=g, device=DEV).to(t).transpose(1, 2)
    v = torch.randn(n, 1, d, generator=g, device=DEV).to(t).expand(n, hk, d)
    grad = torch.randn(1, 1, d, generator=g, device=DEV).to(t).expand(n, h, d)
    _check(host, q, k, v, grad, _offsets(lens), what="expanded")


@pytest.mark.parametrize("host", ["python", "cpp"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
def test_keys_of_their_own_in_a_cache_with_room(host, dtype, causal):
    """Other key rows than query rows, slots longer than what is in use; what lies behind is NaN and must not be seen. More queries
    than keys: the first rows see nothing (causal)."""
    nq, nk, slots = [3, 1, 0, 200, 40, 7], [130, 1, 64, 77, 0, 300], [150, 4, 64, 90, 10, 301]
    t = TYPES[dtype]
    q, k, v, grad = _inputs(sum(nq), sum(slots), 4, 2, 64, t)
    offsets, kv_offsets = _offsets(nq), _offsets(slots)
    kv_lengths = torch.tensor(nk, dtype=torch.int32, device=DEV)
    clean_k, clean_v = k.clone(), v.clone()
    for a, n, s in zip(kv_offsets.tolist(), nk, slots):
        k[a + n:a + s] = float("nan")
        v[a + n:a + s] = float("inf")
        clean_k[a + n:a + s] = 0
        clean_v[a + n:a + s] = 0
    out, dq, dk, dv = _check(host, q, k, v, grad, offsets, kv_offsets, kv_lengths, causal, bound_k=clean_k, bound_v=clean_v)
    first = offsets[4].item()
    assert not out[first:first + 40].any() and not dq[first:first + 40].any()  # no keys at all
    if causal:
        first = offsets[3].item()
        assert not out[first:first + 123].any() and out[first + 123:first + 200].any(1).all()
    for a, n, s in zip(kv_offsets.tolist(), nk, slots):
        assert not dk[a + n:a + s].any() and not dv[a + n:a + s].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("h,hk,d", [(4, 4, 32), (16, 4, 128), (8, 1, 64), (6, 2, 40), (1, 1, 16), (32, 2, 128)])
def test_single_queries_against_long_keys(dtype, h, hk, d):
    """One new row for each sample: the form that serves token by token."""
    nk = [1, 700, 33, 2500, 64, 0, 129]
    slots = [n + 5 for n in nk]
    q, k, v, _ = _inputs(len(nk), sum(slots), h, hk, d, TYPES[dtype])
    kv_offsets, kv_lengths = _offsets(slots), torch.tensor(nk, dtype=torch.int32, device=DEV)
    offsets = torch.arange(len(nk) + 1, dtype=torch.int32, device=DEV)
    want = P.attention(q, k, v, offsets, kv_offsets, kv_lengths, True)["out"]
    for host in ("python", "cpp"):
        P.check(_host(host)(q, k, v, offsets, kv_offsets, kv_lengths, True), want)
        P.check(_host(host)(q, k, v, offsets, kv_offsets, kv_lengths, False), want)
    k[kv_offsets[-1].item() - 5:] = float("nan")
    v[kv_offsets[-1].item() - 5:] = float("nan")
    P.check(_host("cpp")(q, k, v, offsets, kv_offsets, kv_lengths, True), want)
    # none, several and many new rows in one call
    nq = [1, 3, 0, 9, 1, 2, 129]
    q = _inputs(sum(nq), 1, h, hk, d, TYPES[dtype])[0]
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    for causal in (False, True):
        want = P.attention(q, k, v, _offsets(nq), kv_offsets, kv_lengths, causal)["out"]
        P.check(_host("cpp")(q, k, v, _offsets(nq), kv_offsets, kv_lengths, causal), want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_of_no_sample_are_zero(dtype):
    """Rows before the first sample and behind the last, which may hold anything; no sample at all."""
    t = TYPES[dtype]
    q, k, v, grad = _inputs(400, 400, 2, 2, 64, t)
    offsets = _offsets([100, 150], first=30)
    clean = [x.clone() for x in (q, k, v, grad)]
    for x in (q, k, v, grad):
        x[:30] = float("nan")
        x[280:] = float("nan")
    for x in clean:
        x[:30] = 0
        x[280:] = 0
    for causal in (False, True):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out = _host("cpp")(*leaves, offsets, causal=causal)
        grads = torch.autograd.grad(out, leaves, grad)
        want = P.attention(*clean[:3], offsets, causal=causal, grad=clean[3])
        for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
            P.check(got, want[name], name)
            assert not got[:30].any() and not got[280:].any()
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out = _host("cpp")(*leaves, none)
    grads = torch.autograd.grad(out, leaves, grad)
    assert not out.any() and not any(g.any() for g in grads)


@pytest.mark.parametrize("host", ["python", "cpp"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_empty_calls(host, dtype):
    t = TYPES[dtype]
    q, k, v, grad = _inputs(0, 0, 2, 1, 32, t)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    out = _host(host)(*leaves, _offsets([0, 0]))
    grads = torch.autograd.grad(out, leaves, grad)
    assert out.shape == (0, 2, 32) and [g.shape for g in grads] == [q.shape, k.shape, v.shape]
    q, k, v, grad = _inputs(6, 0, 2, 1, 32, t)  # queries without any key row
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    out = _host(host)(*leaves, _offsets([2, 4]), _offsets([0, 0]))
    grads = torch.autograd.grad(out, leaves, grad)
    assert not out.any() and not grads[0].any()
    q, k, v, grad = _inputs(0, 7, 2, 1, 32, t)  # keys that no query sees
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    out = _host(host)(*leaves, _offsets([0, 0]), _offsets([3, 4]))
    grads = torch.autograd.grad(out, leaves, grad)
    assert out.numel() == 0 and not grads[1].any() and not grads[2].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_large_and_equal_scores(dtype):
    """Scores of hundreds: the running maximum has to move; equal ones: plain means."""
    t = TYPES[dtype]
    lens = [257, 300]
    n = sum(lens)
    q, k, v, grad = _inputs(n, n, 2, 2, 64, t)
    k = (k.float() * torch.linspace(0.1, 6, n, device=DEV)[:, None, None]).to(t)  # later keys score higher
    _check("cpp", q, k, v, grad, _offsets(lens), scale=1.0, what="rising")
    _check("cpp", q, k.flip(0).contiguous(), v, grad, _offsets(lens), scale=1.0, what="falling")
    _check("cpp", q, torch.zeros_like(k), v, grad, _offsets(lens), what="equal")
    _check("cpp", q, k, v, grad, _offsets(lens), scale=-0.3, what="negative scale")
    _check("cpp", q, k, v, grad, _offsets(lens), scale=0.0, what="no scale")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_non_finite_sample_stays_alone(dtype):
    t = TYPES[dtype]
    lens = [90, 100, 130]
    q, k, v, grad = _inputs(320, 320, 2, 1, 64, t)
    offsets = _offsets(lens)
    clean = P.attention(q, k, v, offsets, grad=grad, causal=True)
    for x in (q, k, v, grad):
        x[90:190] = float("nan")
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out = _host("cpp")(*leaves, offsets, causal=True)
    grads = torch.autograd.grad(out, leaves, grad)
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        value, bound = clean[name]
        for rows in (slice(0, 90), slice(190, 320)):
            P.check(got[rows], (value[rows], bound[rows]), name)
        assert torch.isnan(got[100:190].float()).any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradient_against_differences(dtype):
    lens = [40, 90]
    q, k, v, grad = _inputs(130, 130, 4, 2, 32, TYPES[dtype])
    offsets = _offsets(lens)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    grads = torch.autograd.grad(_host("cpp")(*leaves, offsets, causal=True), leaves, grad)
    want = P.attention(q.detach(), k.detach(), v.detach(), offsets, causal=True, grad=grad)
    gen = _gen(3)
    step = 1e-4
    for i, name in enumerate(("dq", "dk", "dv")):
        way = torch.randn(grads[i].shape, generator=gen, device=DEV, dtype=torch.float64)
        value = []
        for s in (step, -step):
            args = [x.detach().double() for x in (q, k, v)]
            args[i] = args[i] + s * way
            value.append((P.attention(*args, offsets, causal=True)["out"][0] * grad.double()).sum().item())
        slope = (value[0] - value[1]) / (2 * step)
        # the kernel's own bound along the way, and the step's square times the third derivatives
        room = (want[name][1] * way.abs()).sum().item() + 1e-6 * (want[name][0] * way).abs().sum().item()
        assert abs((grads[i].double() * way).sum().item() - slope) <= room


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_same_bits_every_time(dtype):
    lens = [500, 700, 3]
    n = sum(lens)
    q, k, v, grad = _inputs(n, n, 8, 2, 64, TYPES[dtype])
    first = None
    for _ in range(3):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out = _host("cpp")(*leaves, _offsets(lens), causal=True)
        got = (out, *torch.autograd.grad(out, leaves, grad))
        if first is None:
            first = got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_samples(dtype):
    """More samples than a block has threads, some empty."""
    lens = [(i * 7) % 23 for i in range(700)]
    n = sum(lens)
    q, k, v, grad = _inputs(n, n, 2, 1, 32, TYPES[dtype])
    _check("cpp", q, k, v, grad, _offsets(lens), causal=True)
    nk = [(i * 5) % 41 for i in range(700)]
    q, k, v, _ = _inputs(700, sum(nk), 4, 2, 64, TYPES[dtype])
    offsets = torch.arange(701, dtype=torch.int32, device=DEV)
    P.check(_host("cpp")(q, k, v, offsets, _offsets(nk), causal=True), P.attention(q, k, v, offsets, _offsets(nk), causal=True)["out"])


@pytest.mark.parametrize("samples", [383, 384, 385, 1100])
def test_samples_counted_and_searched_for(samples):
    """Rows before the first sample and behind the last, slots longer than what is in use, samples without rows."""
    lens = [(i * 7) % 13 if i % 50 else 140 for i in range(samples)]
    slots = [(i * 5) % 17 if i % 40 else 150 for i in range(samples)]
    used = torch.tensor([max(0, n - i % 3) for i, n in enumerate(slots)], dtype=torch.int32, device=DEV)
    offsets, kv_offsets = _offsets(lens, 9), _offsets(slots, 300)
    q, _, _, grad = _inputs(sum(lens) + 9 + 260, 1, 1, 1, 40, torch.bfloat16)
    k, v = _inputs(sum(slots) + 300 + 5, sum(slots) + 300 + 5, 1, 1, 40, torch.bfloat16)[1:3]
    out, dq, dk, dv = _check("cpp", q, k, v, grad, offsets, kv_offsets, used, True)
    for t, a, b in ((out, 9, offsets[-1]), (dq, 9, offsets[-1]), (dk, 300, kv_offsets[-1]), (dv, 300, kv_offsets[-1])):
        assert not t[:a].any() and not t[b:].any()
    x = [t.float() for t in (q, k, v, grad)]
    _check("cpp", *x, offsets, kv_offsets, used, True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_offsets_that_leave_the_tensors_are_reported(dtype):
    from riemannengine_b200 import capi
    lib = capi.lib()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.rmn_device_status(stream) == capi.OK
    q, k, v, grad = _inputs(100, 100, 2, 1, 64, TYPES[dtype])
    single = _inputs(3, 1, 2, 1, 64, TYPES[dtype])[0]
    for bad in ([0, 50, 101], [0, 60, 50], [-5, 50, 100], [0, 1 << 30, 100], [7, -(1 << 31), (1 << 31) - 1]):
        offsets = torch.tensor(bad, dtype=torch.int32, device=DEV)
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out = _host("cpp")(*leaves, offsets, causal=True)
        torch.autograd.grad(out, leaves, grad)
        assert lib.rmn_device_status(stream) == capi.ERR_BAD_ARG, bad
        assert lib.rmn_device_status(stream) == capi.OK
        one = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
        _host("cpp")(single, k, v, one, offsets, None, True)
        assert lib.rmn_device_status(stream) == capi.ERR_BAD_ARG, bad
    for lengths in ([51, 50], [-1, 50], [(1 << 31) - 1, 3]):
        _host("cpp")(single, k, v, torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV), _offsets([50, 50]),
                     torch.tensor(lengths, dtype=torch.int32, device=DEV), True)
        assert lib.rmn_device_status(stream) == capi.ERR_BAD_ARG, lengths
    # and the device serves on
    _check("cpp", q, k, v, grad, _offsets([40, 60]))
    assert lib.rmn_device_status(stream) == capi.OK


def test_two_streams_at_once_and_captured():
    lens = [300, 500]
    n = sum(lens)
    offsets = _offsets(lens)
    f = _host("cpp")
    sets = [_inputs(n, n, 4, 2, 64, torch.bfloat16, seed=s) for s in (1, 2)]
    wants = [P.attention(*s[:3], offsets, causal=True, grad=s[3]) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        got = []
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                leaves = [x.detach().requires_grad_(True) for x in s[:3]]
                out = f(*leaves, offsets, causal=True)
                got.append((out, *torch.autograd.grad(out, leaves, s[3])))
    torch.cuda.synchronize()
    for g, want in zip(got, wants):
        for name, t in zip(("out", "dq", "dk", "dv"), g):
            P.check(t, want[name], name)
    # captured: other inputs and other offsets of the same sizes at replay
    q, k, v, grad = (x.clone() for x in sets[0])
    live = offsets.clone()
    for x in (q, k, v):
        x.requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(f(q, k, v, live, causal=True), (q, k, v), grad)
        f(q[:2].detach(), k.detach(), v.detach(), live[:3] * 0 + torch.arange(3, dtype=torch.int32, device=DEV), live, causal=True)
    torch.cuda.current_stream().wait_stream(side)
    ones = torch.arange(3, dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f(q, k, v, live, causal=True)
        grads = torch.autograd.grad(out, (q, k, v), grad)
        step = f(q[:2].detach(), k.detach(), v.detach(), ones, live, causal=True)
    for s, ends in ((sets[1], lens), (sets[0], [17, 783]), (sets[1], [800, 0])):
        with torch.no_grad():
            for t, new in zip((q, k, v), s[:3]):
                t.copy_(new)
            grad.copy_(s[3])
            live.copy_(_offsets(ends))
        graph.replay()
        want = P.attention(*s[:3], live, causal=True, grad=s[3])
        for name, t in zip(("out", "dq", "dk", "dv"), (out, *grads)):
            P.check(t, want[name], name)
        P.check(step, P.attention(s[0][:2], s[1], s[2], ones, live, causal=True)["out"])


@pytest.mark.parametrize("host", ["python", "cpp"])
def test_refusals(host):
    f = _host(host)
    q, k, v, _ = _inputs(10, 10, 4, 2, 32, torch.float32)
    o = _offsets([4, 6])
    for args in ((q[0], k, v, o), (q, k, v[:, :1], o), (q, k[:, :, :16], v[:, :, :16], o), (q[:, :3], k, v, o), (q, k.bfloat16(), v, o),
                 (q.half(), k.half(), v.half(), o), (q, k, v, o.long()), (q, k, v, o.cpu()), (q, k, v, o[None]), (q, k, v, o[:0]),
                 (q[:9], k, v, o), (q, k, v, o, o[:2]), (q, k, v, o, o, o), (q.cpu(), k.cpu(), v.cpu(), o),
                 (q, k, v, torch.zeros(6, dtype=torch.int32, device=DEV)[::2])):
        with pytest.raises((RuntimeError, TypeError)):
            f(*args)
    with pytest.raises(RuntimeError, match="bad argument"):
        f(q, k, v, o, scale=float("nan"))
    wide = torch.zeros(10, 1, 257, device=DEV)
    with pytest.raises(RuntimeError, match="unsupported"):
        f(wide, wide, wide, o)
    a = q.clone().requires_grad_(True)
    w = torch.ones_like(q, requires_grad=True)
    with pytest.raises(RuntimeError, match="once|differentiate twice"):
        (g,) = torch.autograd.grad(f(a, k, v, o), a, w, create_graph=True)
        g.sum().backward()


@pytest.mark.parametrize("host", ["python", "cpp"])
def test_sizes_that_do_not_fit_are_refused(host):
    f = _host(host)
    q, o = torch.zeros(1, 1, 8, device=DEV), _offsets([1])
    for many in (q.expand(2**32 + 1, 1, 8), q.expand(1, 2**32 + 1, 8)):
        with pytest.raises(RuntimeError, match="2\\^31"):
            f(many, q, q, o, o)
        with pytest.raises(RuntimeError, match="2\\^31"):
            f(q, many, many, o, o)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("h,hk,d", [(4, 4, 32), (4, 2, 128), (16, 2, 64)])
def test_uneven_new_rows_against_long_keys(dtype, h, hk, d):
    """Few new rows on average, many of some samples, whose keys several blocks share; and fewer tiles of keys than blocks."""
    nq, nk = [150, 0, 7, 20] + [1] * 60, [3000, 700, 2500, 1000] + [64, 1, 130] * 20
    slots = [n + 3 for n in nk]
    q, k, v, _ = _inputs(sum(nq), sum(slots), h, hk, d, TYPES[dtype], seed=3)
    offsets, kv_offsets = _offsets(nq), _offsets(slots)
    few = [0] * len(nk)
    few[0], few[2], few[3] = 200, 130, 64
    for used in (nk, few):
        lengths = torch.tensor(used, dtype=torch.int32, device=DEV)
        for causal in (False, True):
            want = P.attention(q, k, v, offsets, kv_offsets, lengths, causal)["out"]
            for host in ("python", "cpp"):
                P.check(_host(host)(q, k, v, offsets, kv_offsets, lengths, causal), want, f"{used[:4]} {causal} {host}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_hundreds_of_heads(dtype):
    """More key heads than the GPU has places for blocks of one each."""
    q, k, v, grad = _inputs(70, 70, 320, 320, 16, TYPES[dtype])
    _check("cpp", q, k, v, grad, _offsets([20, 50]), causal=True)
    one = torch.arange(3, dtype=torch.int32, device=DEV)
    want = P.attention(q[:2], k, v, one, _offsets([20, 50]), None, True)["out"]
    P.check(_host("cpp")(q[:2], k, v, one, _offsets([20, 50]), None, True), want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths_without_offsets_of_their_own(dtype, causal):
    lens, used = [40, 200, 1, 130, 9], [40, 33, 0, 129, 1]
    q, k, v, grad = _inputs(sum(lens), sum(lens), 4, 2, 64, TYPES[dtype])
    lengths = torch.tensor(used, dtype=torch.int32, device=DEV)
    for host in ("python", "cpp"):
        _check(host, q, k, v, grad, _offsets(lens), None, lengths, causal)


@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("f32", 32), ("f32", 30)])
def test_a_cache_of_more_than_2_31_elements(dtype, d):
    """The samples at the very end of it: prompts with their gradients, and new rows."""
    lens = [300, 77]
    rows = (1 << 31) // d + 5000
    cache = torch.zeros(rows, 1, d, dtype=TYPES[dtype], device=DEV)
    q, k, _, grad = _inputs(sum(lens), sum(lens), 2, 1, d, TYPES[dtype])
    cache[-sum(lens):] = k
    offsets, kv_offsets = _offsets(lens), _offsets(lens, rows - sum(lens))
    want = P.attention(q, k, k, offsets, causal=True, grad=grad)
    leaves = [q.requires_grad_(True), cache.requires_grad_(True)]
    out = _host("cpp")(q, cache, cache.detach(), offsets, kv_offsets, None, True)
    dq, dk = torch.autograd.grad(out, leaves, grad)
    for name, got in (("out", out), ("dq", dq), ("dk", dk[-sum(lens):])):
        P.check(got, want[name], name)
    assert not dk[:5000].any() and not dk[rows - sum(lens) - 5000:rows - sum(lens)].any()
    del dq, dk, out
    one = torch.arange(3, dtype=torch.int32, device=DEV)
    with torch.no_grad():
        got = _host("cpp")(q[:2], cache, cache, one, kv_offsets, None, True)
    P.check(got, P.attention(q[:2].detach(), k, k, one, offsets, None, True)["out"])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("h,hk,d", [(4, 4, 32), (4, 2, 128), (3, 3, 80)])
def test_uneven_new_rows_against_a_thousand_keys(dtype, h, hk, d):
    nq, nk = [60, 0, 7, 20] + [1] * 12, [3000, 700, 2500, 1000] + [900, 1000, 30] * 4
    q, k, v, _ = _inputs(sum(nq), sum(nk), h, hk, d, TYPES[dtype], seed=5)
    for causal in (False, True):
        want = P.attention(q, k, v, _offsets(nq), _offsets(nk), None, causal)["out"]
        P.check(_host("cpp")(q, k, v, _offsets(nq), _offsets(nk), None, causal), want)


def test_offsets_that_give_rows_to_many_samples():
    """2^17 samples that each claim all rows: more tiles than 32 bits count. The call reports it and touches only its tensors."""
    from riemannengine_b200 import capi
    lib = capi.lib()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    n = 1 << 21
    offsets = torch.tensor([0, n], dtype=torch.int32, device=DEV).repeat(1 << 16)
    lengths = torch.zeros(offsets.numel() - 1, dtype=torch.int32, device=DEV)
    for heads in (1, 4):
        q = torch.zeros(n, heads, 8, dtype=torch.bfloat16, device=DEV)
        out = _host("cpp")(q, q[:, :1], q[:, :1], offsets, None, lengths, True)
        assert lib.rmn_device_status(stream) == capi.ERR_BAD_ARG
        del out
    assert lib.rmn_device_status(stream) == capi.OK


@pytest.mark.parametrize("n,runs", [(0, 0), (1, 1), (255, 3), (1000, 1000), (300_001, 7), (300_001, 100_000), (2_000_000, 1_999_999)])
def test_sample_offsets(n, runs):
    from riemannengine_b200 import ops
    g = _gen(n + runs)
    starts = torch.sort(torch.randperm(max(n - 1, 0), generator=g, device=DEV)[:max(runs - 1, 0)] + 1).values
    batch = torch.zeros(n, dtype=torch.int32, device=DEV)
    batch[starts] = 1
    coords = torch.zeros(n, 4, dtype=torch.int32, device=DEV)
    coords[:, 0] = batch.cumsum(0) * 37 % 65521  # neighbours differ
    coords[:, 1] = torch.randint(0, 9, (n,), generator=g, device=DEV)
    first = torch.cat([torch.zeros(min(n, 1), dtype=torch.int64, device=DEV), starts]).tolist()
    for room in sorted({runs, max(runs - 1, 0), runs + 3}):
        want = (first + [n] * 3)[:room] + [n, runs]
        assert ops.sample_offsets(coords, room).tolist() == want


def _cloud(host, order):
    """Two samples of 60 and 90 rows, batch indices 7 and 3; `order` shuffles the rows across samples."""
    coords = torch.tensor([[7, i, 0, 0] for i in range(60)] + [[3, i, 1, 0] for i in range(90)], dtype=torch.int32, device=DEV)
    x = torch.randn(150, 64, generator=_gen(11), device=DEV)
    return coords[order].contiguous(), x[order].contiguous()


@pytest.mark.parametrize("host", ["python", "cpp"])
def test_layers_on_sparse_tensors(host):
    """Norm, self-attention and the sum with the input, as a network runs them, against 64 bits; and sample_offsets."""
    if host == "cpp":
        from riemannengine_b200 import cpp
        H = cpp.load()
    else:
        from riemannengine_b200 import engine as H
    coords, x = _cloud(H, torch.arange(150, device=DEV))
    tensor = H.SparseTensor(x.requires_grad_(True), coords)
    norm, attend = H.RiemannLayerNorm(64), H.RiemannSelfAttention(64, 4, 2, causal=True)
    for layer in (norm, attend):
        layer.to(DEV)
    offsets = tensor.coordinate_manager.sample_offsets(tensor.coordinate_map_key)
    assert offsets.tolist() == [0, 60, 150] and offsets.dtype == torch.int32
    y = attend(norm(tensor)) + tensor
    y.F.square().sum().backward()
    p = {**{"n." + k: v for k, v in norm.named_parameters().items()}, **dict(attend.named_parameters())} if host == "cpp" else \
        {**{"n." + k: v for k, v in norm.named_parameters()}, **dict(attend.named_parameters())}
    leaves = {k: v.detach().double().requires_grad_(True) for k, v in p.items()}
    X = x.detach().double().requires_grad_(True)
    hat = torch.nn.functional.layer_norm(X, (64,), leaves["n.normalization.weight"], leaves["n.normalization.bias"])
    qkv = hat @ leaves["qkv.weight"].T + leaves["qkv.bias"]
    q, k, v = qkv.view(150, 8, 16).split([4, 2, 2], 1)
    rows = []
    for a, b in ((0, 60), (60, 150)):
        s = torch.einsum("ihd,jhd->hij", q[a:b], k[a:b].repeat_interleave(2, 1)) / 4
        s = s.masked_fill(~torch.ones(b - a, b - a, dtype=torch.bool, device=DEV).tril(), float("-inf"))
        rows.append(torch.einsum("hij,jhd->ihd", s.softmax(-1), v[a:b].repeat_interleave(2, 1)).reshape(b - a, 64))
    want = torch.cat(rows) @ leaves["projection.weight"].T + leaves["projection.bias"] + X
    want.square().sum().backward()
    # four products of 64 terms and one of up to 90 behind one another, each off by its terms times u of values of order 1 ... 10
    tol = 10 * 64 * 5 * P.U32
    assert (y.F.double() - want).abs().max() <= tol
    for name, got in [("x", x), *p.items()]:
        ref = X.grad if name == "x" else leaves[name].grad
        assert (got.grad.double() - ref).abs().max() <= 4 * tol * ref.abs().max() + 150 * tol, name
    # rows of a sample that are not adjacent
    coords, x = _cloud(H, torch.randperm(150, generator=_gen(1), device=DEV))
    mixed = H.SparseTensor(x, coords)
    with pytest.raises(RuntimeError, match="adjacent"):
        mixed.coordinate_manager.sample_offsets(mixed.coordinate_map_key)
    with pytest.raises(RuntimeError, match="adjacent"):
        attend(mixed)
    with pytest.raises(RuntimeError, match="channel count"):
        attend(H.SparseTensor(x[:, :32], coords))


@pytest.mark.parametrize("host", ["python", "cpp"])
def test_second_derivatives_are_refused_where_the_first_is_of_a_sum(host):
    """As one of several terms, too, whose derivative would lack it without an error."""
    q, k, v, _ = _inputs(20, 20, 2, 1, 32, torch.float32)
    offsets = _offsets([8, 12])
    for wanted in ((0,), (1,), (2,), (0, 1, 2)):
        leaves = [t.clone().requires_grad_(i in wanted) for i, t in enumerate((q, k, v))]
        some = [leaves[i] for i in wanted]
        loss = _host(host)(*leaves, offsets).sum()
        grads = torch.autograd.grad(loss, some, create_graph=True)
        want = P.attention(q, k, v, offsets, grad=torch.ones_like(q))
        for i, g in zip(wanted, grads):
            P.check(g, want[("dq", "dk", "dv")[i]])
        for grad in (lambda: (loss + grads[0].square().sum()).backward(retain_graph=True),
                     lambda: torch.autograd.grad(loss + grads[0].square().sum(), some, retain_graph=True)):
            with pytest.raises(RuntimeError, match="packed_attention is differentiable once only"):
                grad()


def _unaligned(x):
    """The same values one element off 16 bytes: only the multiply-add kernels of whole tiles take them."""
    y = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view(x.shape)
    return y.copy_(x)


@pytest.mark.parametrize("sign", ["either", "one"])
@pytest.mark.parametrize("keys", [500, 30_000])
@pytest.mark.parametrize("rows,h,hk,d", [(1, 4, 4, 32), (1, 8, 2, 64), (1, 16, 2, 128), (5, 4, 2, 64), (12, 1, 1, 128)])
def test_few_rows_in_fp32_are_as_exact_as_whole_tiles(rows, h, hk, d, keys, sign):
    """What a batch's averages decide is the time, not how exact fp32 is: the error (root of the mean square) against 64 bits is not above
    that of the kernel of whole tiles but for the last rounding of every output, half a step of its size."""
    nk = [keys, keys // 3 + 1]
    q, k, v, _ = _inputs(2 * rows, sum(nk), h, hk, d, torch.float32, seed=keys)
    if sign == "one":
        q, k, v = q.abs() * 0.2, k.abs(), v.abs()
    offsets, kv_offsets = _offsets([rows, rows]), _offsets(nk)
    want = P.attention(q, k, v, offsets, kv_offsets, None, True)["out"][0]
    rms = lambda t: t.square().mean().sqrt().item()  # noqa: E731
    for host in ("python", "cpp"):
        few = rms(_host(host)(q, k, v, offsets, kv_offsets, None, True).double() - want)
        whole = rms(_host(host)(_unaligned(q), k, v, offsets, kv_offsets, None, True).double() - want)
        assert few <= whole + P.U32 * rms(want), (few, whole, rms(want))


@pytest.mark.parametrize("rows,h,hk,d", [(1, 4, 4, 32), (1, 8, 2, 64), (1, 16, 2, 128), (12, 1, 1, 64)])
def test_infinite_and_largest_values_with_few_rows_in_fp32(rows, h, hk, d):
    """Keys that are infinitely or as far off as numbers go have no weight; an infinite value with a weight makes the output infinite,
    a largest one does not, as in the kernel of whole tiles."""
    n, lowest = 700, torch.finfo(torch.float32).min
    q, k, v, _ = _inputs(rows, n, h, hk, d, torch.float32)
    q[..., 0] = q[..., 0].abs() + 0.1
    offsets, kv_offsets = _offsets([rows]), _offsets([n])
    keep = torch.ones(n, dtype=torch.bool, device=DEV)
    k[100, :, 0], k[300, :, 0], k[650, :, 0] = float("-inf"), lowest, lowest
    keep[[100, 300, 650]] = False
    want = P.attention(q, k[keep], v[keep], offsets, _offsets([n - 3]))["out"]
    f = _host("cpp")
    for x in (q, _unaligned(q)):
        P.check(f(x, k, v, offsets, kv_offsets), want)
    # (a weight of a few thousandths of what is largest: no sum leaves the numbers)
    v[7, :, 3], v[8, :, 5], v[9, :, 6] = float("inf"), float("-inf"), torch.finfo(torch.float32).max
    for x in (q, _unaligned(q)):
        out = f(x, k, v, offsets, kv_offsets)
        assert (out[..., 3] == float("inf")).all() and (out[..., 5] == float("-inf")).all() and torch.isfinite(out[..., 6]).all()
        rest = [c for c in range(d) if c not in (3, 5, 6)]
        P.check(out[..., rest], tuple(t[..., rest] for t in want))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("h,hk,d", [(2, 1, 64), (16, 4, 128), (4, 4, 40)])
def test_few_rows_with_descending_offsets_are_zero(dtype, h, hk, d):
    """The call is reported, and what was in the outputs' memory does not come back as a result."""
    from riemannengine_b200 import capi, ops
    lib, p = capi.lib(), lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    q, k, v, _ = _inputs(3, 900, h, hk, d, TYPES[dtype])
    offsets = _offsets([1, 1, 1])
    for bad in ([0, 500, 200, 900], [300, 0, 400, 900], [0, 901, 1, 900]):
        kv_offsets = torch.tensor(bad, dtype=torch.int32, device=DEV)  # (the problem holds its address only)
        problem = ops._attention(q, k, v, offsets, kv_offsets, None, True, None)
        nbytes = lib.rmn_attention_forward_workspace_bytes(ctypes.byref(problem))
        assert nbytes > 0  # few query rows
        ws = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
        out, low, lse = torch.full_like(q, 7), torch.full_like(q, 7), torch.full((h, 3), 7.0, device=DEV)
        assert lib.rmn_attention_forward(ctypes.byref(problem), p(out), p(low), p(lse), p(ws), nbytes, stream) == capi.OK
        assert lib.rmn_device_status(stream) == capi.ERR_BAD_ARG, bad
        assert not out.any() and (lse == float("-inf")).all()
        assert not low.any() if dtype == "bf16" else (low == 7).all()


def _grids(call):
    """Blocks of every kernel that `call` launches on the current stream, in order: from the nodes of a captured graph."""
    class Params(ctypes.Structure):  # CUDA_KERNEL_NODE_PARAMS_v2 of the driver's interface
        _fields_ = ([("func", ctypes.c_void_p)] + [(f"{what}{axis}", ctypes.c_uint) for what in ("grid", "block") for axis in "xyz"]
                    + [("smem", ctypes.c_uint), ("args", ctypes.c_void_p), ("extra", ctypes.c_void_p), ("kern", ctypes.c_void_p),
                       ("ctx", ctypes.c_void_p)])
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    cu, raw, n = ctypes.CDLL("libcuda.so.1"), ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t()
    assert cu.cuGraphGetNodes(raw, None, ctypes.byref(n)) == 0
    nodes = (ctypes.c_void_p * n.value)()
    assert cu.cuGraphGetNodes(raw, nodes, ctypes.byref(n)) == 0
    grids = []
    for node in nodes:
        kind, p = ctypes.c_int(), Params()
        assert cu.cuGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(kind)) == 0
        if kind.value == 0:
            assert cu.cuGraphKernelNodeGetParams_v2(ctypes.c_void_p(node), ctypes.byref(p)) == 0
            grids.append(p.gridx * p.gridy * p.gridz)
    return grids


@pytest.mark.parametrize("samples,rows,h,hk,d,clusters", [(4096, 4, 8, 1, 64, False), (700, 60, 8, 2, 128, False), (64, 130, 8, 1, 64, True),
                                                          (2, 700, 8, 2, 128, True)])
def test_key_heads_are_shared_by_clusters_where_there_are_few_tiles(samples, rows, h, hk, d, clusters):
    """Every sample has a tile of its own at least: many short ones fill the GPU without clusters."""
    from riemannengine_b200 import ops
    n = samples * rows
    q, k, v, grad = _inputs(n, n, h, hk, d, torch.bfloat16)
    offsets = _offsets([rows] * samples)
    out, low, lse = ops.attention_forward(q, k, v, offsets, want_stats=True)
    grids = _grids(lambda: ops.attention_backward(grad, q, k, v, out, low, lse, offsets))
    blocks = (n // 128 + samples + 2) * hk  # one for every tile of keys that there may be, and key head
    assert len(grids) == 2 and grids[1] == blocks * (h // hk if clusters else 1), (grids, blocks)
    got = ops.attention_backward(grad, q, k, v, out, low, lse, offsets)
    few = slice(0, 3 * rows)
    want = P.attention(q[few], k[few], v[few], offsets[:4] if samples > 2 else offsets, grad=grad[few]) if samples > 2 else \
        P.attention(q, k, v, offsets, grad=grad)
    for name, t in zip(("dq", "dk", "dv"), got):
        P.check(t[few] if samples > 2 else t, want[name], name)


@pytest.mark.parametrize("host", ["python", "cpp"])
@pytest.mark.parametrize("d", [32, 128])
def test_broadcast_and_unaligned_gradients_stay_on_the_tensor_cores(host, d):
    from riemannengine_b200 import capi
    h, hk, lens = 4, 2, [150, 3, 200]
    n = sum(lens)
    q, k, v, grad = _inputs(n, n, h, hk, d, torch.bfloat16)
    offsets = _offsets(lens)
    gradients = {"a mean over rows": grad[:1].expand(n, h, d), "a mean over heads": grad[:, :1].expand(n, h, d), "unaligned": _unaligned(grad),
                 "rows apart": torch.zeros(n, h * d + 4, dtype=grad.dtype, device=DEV)[:, 4:].unflatten(1, (h, d)).copy_(grad)}
    for what, g in gradients.items():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = _host(host)(*leaves, offsets)
        before = capi.lib().rmn_tensor_core_launch_count()
        grads = torch.autograd.grad(out, leaves, g)
        assert capi.lib().rmn_tensor_core_launch_count() == before + 2, what
        want = P.attention(q, k, v, offsets, grad=g)
        for name, t in zip(("dq", "dk", "dv"), grads):
            P.check(t, want[name], f"{name} {what}")
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    before = capi.lib().rmn_tensor_core_launch_count()
    _host(host)(*leaves, offsets).mean(0).square().sum().backward()
    assert capi.lib().rmn_tensor_core_launch_count() == before + 3


def _check_statistics(q, k, v, offsets, kv_offsets=None, kv_lengths=None, causal=False):
    """lse, and what is stored of the output with what rounding took from it: it differs from the value by the roundings of the weights and
    of fp32, no more by the output's own."""
    from riemannengine_b200 import ops
    out, low, lse = ops.attention_forward(q, k, v, offsets, kv_offsets, kv_lengths, causal, want_stats=True)
    want = P.attention(q, k, v, offsets, kv_offsets, kv_lengths, causal)
    assert lse.dtype == torch.float32 and lse.shape == want["lse"][0].shape
    P.check(lse, want["lse"], "lse")
    P.check(out, want["out"], "out")
    if q.dtype == torch.float32:
        assert low is None
    else:
        u = P.half_step(q.dtype)
        value, bound = want["out"]
        # (low is rounded, too: u of what is at most u of the output)
        P.check(out.double() + low.double(), (value, bound - u * value.abs() + 2 * u * u * value.abs()), "out and low")
    return want["lse"][0]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("h,hk,d", [(4, 2, 32), (4, 1, 64), (3, 3, 128), (2, 2, 20), (2, 1, 192)])
def test_statistics_of_packed_samples(dtype, h, hk, d, causal):
    """Rows before the first sample and behind the last, samples of no rows, more queries than keys: -infinity where nothing is seen."""
    t, lens = TYPES[dtype], [70, 0, 140, 1, 300]
    q, k, v, _ = _inputs(sum(lens) + 14, sum(lens) + 14, h, hk, d, t)
    lse = _check_statistics(q, k, v, _offsets(lens, 9), causal=causal)
    assert (lse[:, :9] == float("-inf")).all() and (lse[:, -5:] == float("-inf")).all() and torch.isfinite(lse[:, 9:-5]).all()
    nk = [30, 12, 150, 0, 300]
    k, v = _inputs(sum(nk), sum(nk), h, hk, d, t)[1:3]
    lse = _check_statistics(q, k, v, _offsets(lens, 9), _offsets(nk), causal=causal)
    assert (lse[:, 9 + 210] == float("-inf")).all()  # no key at all
    assert torch.equal(lse[:, 9:9 + 40] == float("-inf"), torch.full_like(lse[:, 9:9 + 40], float(causal)) > 0)


FEW_ROWS = {"single": ([1] * 7, [1, 700, 33, 2500, 64, 0, 129]), "several": ([1, 3, 0, 4, 1, 2, 5], [1, 700, 33, 2500, 64, 0, 129]),
            "uneven": ([60, 0, 7, 20] + [1] * 12, [3000, 700, 2500, 1000] + [900, 1000, 30] * 4), "one": ([1], [20_000]), "two": ([2], [5000])}


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("which", FEW_ROWS)
@pytest.mark.parametrize("h,hk,d", [(4, 4, 32), (8, 1, 64), (16, 4, 128), (6, 2, 40)])
def test_statistics_and_gradients_of_few_rows(which, dtype, h, hk, d):
    """The form for few query rows leaves what a backward pass needs, also where several blocks have pieces of a sample."""
    nq, nk = FEW_ROWS[which]
    slots = [n + 3 for n in nk]
    q, k, v, grad = _inputs(sum(nq), sum(slots), h, hk, d, TYPES[dtype], seed=len(nq))
    kv_lengths = torch.tensor(nk, dtype=torch.int32, device=DEV)
    for causal in (False, True):
        _check_statistics(q, k, v, _offsets(nq), _offsets(slots), kv_lengths, causal)
        _check("cpp", q, k, v, grad, _offsets(nq), _offsets(slots), kv_lengths, causal)


def test_samples_without_rows_among_thousands_of_one_row():
    """More samples than rows: the tiles there may be are those of the rows."""
    from riemannengine_b200 import ops
    lens, h, d = [i % 2 for i in range(4096)], 8, 64
    n = sum(lens)
    q, k, v, grad = _inputs(n, n, h, 1, d, torch.bfloat16)
    offsets = _offsets(lens)
    out, low, lse = ops.attention_forward(q, k, v, offsets, want_stats=True)
    grids = _grids(lambda: ops.attention_backward(grad, q, k, v, out, low, lse, offsets))
    assert grids[1] == n // 128 + 4096 + 2, grids
    got = ops.attention_backward(grad, q, k, v, out, low, lse, offsets)
    want = P.attention(q[:20], k[:20], v[:20], offsets[:41], grad=grad[:20])
    for name, t in zip(("dq", "dk", "dv"), got):
        P.check(t[:20], want[name], name)
