"""Rotary positions, and norms of queries and keys with them: both hosts against 64 bits, forward and backward, at the sizes, strides
and positions where it can go wrong."""
import pytest
import torch

from tests import plain_rotary as R
from tests.plain_tokens import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


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


def _frequencies(sections, base=10000.0):
    return torch.tensor([base ** (-i / n) for n in sections for i in range(n)], dtype=torch.float64, device=DEV)


def _positions(rows, axes, g, low=-1000, high=1000):
    return torch.randint(low, high, (rows, axes), generator=g, device=DEV, dtype=torch.int32)


def _check(host, q, k, positions, sections, interleaved, wq=None, wk=None, gq=None, gk=None, base=10000.0, norm=True, eps=1e-6, what=""):
    f = _frequencies(sections, base)
    H = _host(host)
    args = (positions, f, sections)
    if not norm:
        x = q.detach().requires_grad_(True)
        y = H.rotary_positions(x, *args, interleaved=interleaved)
        assert y.is_contiguous() and y.dtype == q.dtype
        want = R.rotary(q, None, positions, f, sections, interleaved, gq=gq)
        check(y, want["q"], f"out {what}")
        if gq is not None:
            check(torch.autograd.grad(y, x, gq)[0], want["dq"], f"dx {what}")
        with torch.no_grad():
            assert torch.equal(H.rotary_positions(q, *args, interleaved=interleaved), y)
        return y
    leaves = {n: t.detach().requires_grad_(True) for n, t in (("q", q), ("k", k), ("wq", wq), ("wk", wk)) if t is not None}
    yq, yk = H.qk_norm_rotary(leaves["q"], leaves["k"], leaves.get("wq"), leaves.get("wk"), *args, eps=eps, interleaved=interleaved)
    want = R.rotary(q, k, positions, f, sections, interleaved, True, wq, wk, eps, gq, gk)
    check(yq, want["q"], f"q {what}")
    check(yk, want["k"], f"k {what}")
    if gq is not None:
        grads = torch.autograd.grad((yq, yk), list(leaves.values()), (gq, gk))
        for n, g in zip(leaves, grads):
            assert g.dtype == leaves[n].dtype
            check(g, want["d" + n], f"d{n} {what}")
    with torch.no_grad():
        again = H.qk_norm_rotary(q, k, wq, wk, *args, eps=eps, interleaved=interleaved)
    assert torch.equal(again[0], yq) and torch.equal(again[1], yk)
    return yq, yk


def _data(rows, h, hk, d, dtype, seed=0):
    g = _gen(seed * 7919 + rows + 31 * h + 17 * d)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    return (r(rows, h, d).to(dtype), r(rows, hk, d).to(dtype), (r(d) * 0.3 + 1).to(dtype), (r(d) * 0.3 + 1).to(dtype),
            r(rows, h, d).to(dtype), r(rows, hk, d).to(dtype), g)


# channels, pairs of each axis: whole heads and parts of them, sections that cut through a 16-byte load, one pair, odd numbers of pairs
SIZES = [(2, [1]), (6, [1, 1, 1]), (10, [5]), (16, [4, 2, 2]), (24, [4, 4, 4]), (32, [6, 5, 5]), (40, [20]), (48, [0, 24]), (64, [11, 11, 10]),
         (66, [33]), (80, [8, 12, 12]), (80, [30]), (96, [16, 16, 16]), (112, [3, 5]), (128, [64]), (128, [16, 24, 24]), (130, [20, 20, 25]),
         (192, [1, 2, 3, 4, 5, 6, 7, 8]), (256, [128]), (254, [100])]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d,sections", SIZES, ids=lambda v: str(v))
def test_sizes(d, sections, dtype, interleaved):
    t = TYPES[dtype]
    for rows, h, hk in ((1, 1, 1), (7, 3, 1), (37, 4, 2), (300, 5, 5)):
        q, k, wq, wk, gq, gk, g = _data(rows, h, hk, d, t)
        positions = _positions(rows, len(sections), g)
        _check("cpp", q, k, positions, sections, interleaved, wq, wk, gq, gk, what=f"{rows} {h} {hk}")
        _check("cpp", q, None, positions, sections, interleaved, gq=gq, norm=False, what=f"{rows} {h}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,h,hk,d", [(1, 64, 8, 128), (16, 16, 4, 128), (5000, 2, 2, 16), (40_000, 4, 1, 32), (3001, 12, 3, 64),
                                         (70_001, 1, 1, 8)])
def test_row_counts(rows, h, hk, d, dtype):
    """From one row, whose heads are dealt out, to more than the blocks of the backward pass take at a time."""
    t = TYPES[dtype]
    q, k, wq, wk, gq, gk, g = _data(rows, h, hk, d, t)
    sections = [d // 2 - d // 8, d // 8]
    positions = _positions(rows, 2, g)
    _check("cpp", q, k, positions, sections, False, wq, wk, gq, gk)
    _check("cpp", q, None, positions, sections, False, gq=gq, norm=False)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d,sections", [(12, [6]), (20, [3, 4]), (24, [12]), (40, [16]), (48, [8, 8, 8]), (72, [36]), (80, [8, 12, 12]),
                                        (88, [40]), (112, [20, 20]), (136, [4]), (200, [100]), (240, [64, 3])], ids=lambda v: str(v))
def test_lanes_and_heads(d, sections, dtype):
    """Heads over any number of lanes, several of a row and several rows in a warp, some of its lanes idle; what turns ends inside a lane's
    share, and lanes have nothing that turns. Channels that do not turn are not finite."""
    t = TYPES[dtype]
    for rows, h in ((1, 64), (130, 9), (131, 16), (67, 24), (3001, 7)):
        q, _, _, _, gq, _, g = _data(rows, h, 1, d, t)
        positions = _positions(rows, len(sections), g)
        for interleaved in (False, True):
            _check("cpp", q, None, positions, sections, interleaved, gq=gq, norm=False, what=f"{rows} {h} {interleaved}")
        turned = 2 * sum(sections)
        if turned < d:
            x = q.clone()
            x[..., turned] = float("inf")
            x[..., turned + 1:] = float("nan")
            y = _host("cpp").rotary_positions(x, positions, _frequencies(sections), sections)
            assert torch.equal(y[..., turned:].nan_to_num(), x[..., turned:].nan_to_num())
            want = R.rotary(q[..., :turned], None, positions, _frequencies(sections), sections)["q"]
            check(y[..., :turned], want, "beside what is not finite")


@pytest.mark.parametrize("host", ["python", "cpp"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_views(host, dtype):
    """Parts of one projection, aligned and not; heads first; broadcast rows and heads; channels that are not adjacent; positions as the
    columns of coordinates, one for all rows, one axis as a vector."""
    t, h, hk, d, n, sections = TYPES[dtype], 4, 2, 48, 77, [8, 8, 8]
    g = _gen(5)
    coords = torch.randint(-300, 300, (n, 4), generator=g, device=DEV, dtype=torch.int32)
    wq, wk = ((torch.randn(d, generator=g, device=DEV) * 0.2 + 1).to(t) for _ in range(2))
    gq = torch.randn(h, n, d, generator=g, device=DEV).to(t).transpose(0, 1)
    gk = torch.randn(1, 1, d, generator=g, device=DEV).to(t).expand(n, hk, d)
    for extra, first in ((0, 0), (8, 8), (4, 4), (3, 1)):
        whole = torch.randn(n, (h + hk) * d + extra, generator=g, device=DEV).to(t)
        q, k = whole[:, first:first + (h + hk) * d].unflatten(1, (h + hk, d)).split([h, hk], 1)
        _check(host, q, k, coords[:, 1:], sections, False, wq, wk, gq, gk, what=f"first {first}")
        _check(host, q, None, coords[:, 1:], sections, True, gq=gq, norm=False, what=f"first {first}")
    q = torch.randn(n, d, h, generator=g, device=DEV).to(t).transpose(1, 2)
    k = torch.randn(1, 1, d, generator=g, device=DEV).to(t).expand(n, hk, d)
    one = coords[:1, 1:].expand(n, 3)
    _check(host, q, k, one, sections, False, wq, wk, gq, gk, what="expanded")
    _check(host, q, k, coords[:, 2], [24], False, wq.float() if t == torch.bfloat16 else wq.bfloat16(),
           wk.float() if t == torch.bfloat16 else wk.bfloat16(), gq, gk, what="weights of the other type")
    _check(host, q, k, coords[:, 2], [24], False, None, wk, gq, gk, what="no q_weight")
    _check(host, q, k, coords[:, 2], [24], False, None, None, gq, gk, what="no weights")


@pytest.mark.parametrize("host", ["python", "cpp"])
def test_norm_alone_and_rotation_without_pairs(host):
    q, k, wq, wk, gq, gk, g = _data(50, 4, 2, 40, torch.float32)
    H = _host(host)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
    out = H.qk_norm_rotary(*leaves, eps=1e-3)
    want = R.rotary(q, k, None, None, [], False, True, wq, wk, 1e-3, gq, gk)
    for n, got in zip(("q", "k", "dq", "dk", "dwq", "dwk"), (*out, *torch.autograd.grad(out, leaves, (gq, gk)))):
        check(got, want[n], n)
    positions, none = _positions(50, 2, g), torch.empty(0, dtype=torch.float64, device=DEV)
    assert torch.equal(H.rotary_positions(q, positions, none, [0, 0]), q)
    # one of the outputs alone, and gradients of the weights alone
    out = H.qk_norm_rotary(*leaves, eps=1e-3)
    check(torch.autograd.grad(out[0], leaves[2], gq)[0], want["dwq"])
    out = H.qk_norm_rotary(q, k, leaves[2], wk, eps=1e-3)
    check(torch.autograd.grad(out[0], leaves[2], gq)[0], want["dwq"])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_far_positions_are_as_exact_as_near_ones(dtype):
    ends = [0, 1, -1, 12345, -99999, 10_000_000, 2**31 - 1, -2**31, 2**30 + 7, 1 << 24]
    positions = torch.tensor([[a, b] for a in ends for b in reversed(ends)], dtype=torch.int32, device=DEV)
    q, _, _, _, gq, _, _ = _data(len(positions), 3, 1, 64, TYPES[dtype])
    for base in (10000.0, 1.0, 1_000_000.0):
        _check("cpp", q, None, positions, [16, 16], False, gq=gq, norm=False, base=base)
    # eighths, quarters and whole turns
    f = torch.tensor([2 * torch.pi * i / 16 for i in range(-32, 32)], dtype=torch.float64, device=DEV)
    x = torch.randn(9, 2, 128, generator=_gen(3), device=DEV).to(TYPES[dtype])
    places = torch.arange(-4, 5, device=DEV, dtype=torch.int32)
    check(_host("cpp").rotary_positions(x, places, f, [64]), R.rotary(x, None, places, f, [64])["q"])


def test_rotation_leaves_the_other_channels_and_heads_alone():
    """What is not finite in channels behind the pairs, or in one head, stays there."""
    x = torch.randn(6, 3, 64, generator=_gen(1), device=DEV)
    positions = torch.arange(6, dtype=torch.int32, device=DEV)
    f = _frequencies([20])
    clean = _host("cpp").rotary_positions(x, positions, f, [20])
    assert torch.equal(clean[..., 40:], x[..., 40:])
    y = x.clone()
    y[2, 1, 40:] = float("inf")
    y[3, 0] = float("nan")
    got = _host("cpp").rotary_positions(y, positions, f, [20])
    assert torch.equal(got[2], torch.cat((clean[2, :, :40], y[2, :, 40:]), 1)) and got[3, 0].isnan().all()
    assert torch.equal(got[3, 1:], clean[3, 1:]) and torch.equal(got[4:], clean[4:])


@pytest.mark.parametrize("host", ["python", "cpp"])
def test_no_rows(host):
    H = _host(host)
    x = torch.zeros(0, 4, 32, device=DEV, requires_grad=True)
    w = torch.ones(32, device=DEV, requires_grad=True)
    positions, f = torch.zeros(0, 1, dtype=torch.int32, device=DEV), _frequencies([16])
    y = H.rotary_positions(x, positions, f, [16])
    assert y.shape == x.shape and torch.autograd.grad(y.sum(), x)[0].shape == x.shape
    q, k = H.qk_norm_rotary(x, x, w, w, positions, f, [16])
    assert q.shape == x.shape and not torch.autograd.grad(q.sum() + k.sum(), w)[0].any()


def test_gradients_against_differences():
    """The loss along a direction, by differences of the 64-bit form, against the kernels' gradients."""
    q, k, wq, wk, gq, gk, g = _data(40, 4, 2, 32, torch.float32)
    positions, sections = _positions(40, 2, g), [9, 5]
    f = _frequencies(sections)
    leaves = [t.requires_grad_(True) for t in (q, k, wq, wk)]
    out = _host("cpp").qk_norm_rotary(*leaves, positions, f, sections)
    grads = torch.autograd.grad(out, leaves, (gq, gk))
    steps = [torch.randn(t.shape, generator=g, device=DEV) for t in leaves]

    def loss(by):
        a = [t.detach().double() + by * s.double() for t, s in zip(leaves, steps)]
        want = R.rotary(a[0], a[1], positions, f, sections, False, True, a[2], a[3])
        return ((want["q"][0] * gq.double()).sum() + (want["k"][0] * gk.double()).sum()).item()

    e = 1e-4
    slope = (loss(e) - loss(-e)) / (2 * e)
    got = sum((a.double() * s.double()).sum().item() for a, s in zip(grads, steps))
    # differences: e^2 / 6 of a third derivative, of the size of the terms here; gradients: 2^-20 of the terms' sizes
    size = sum((a.double() * s.double()).abs().sum().item() for a, s in zip(grads, steps))
    assert abs(slope - got) <= size * (2.0 ** -20 + 1e-6)


def test_same_bits_every_time_and_on_another_stream():
    q, k, wq, wk, gq, gk, g = _data(20_000, 8, 2, 64, torch.bfloat16)
    positions, f = _positions(20_000, 3, g), _frequencies([11, 11, 10])
    leaves = [t.requires_grad_(True) for t in (q, k, wq, wk)]
    H = _host("cpp")

    def step():
        out = H.qk_norm_rotary(*leaves, positions, f, [11, 11, 10])
        return [*out, *torch.autograd.grad(out, leaves, (gq, gk))]

    first = step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_captured_and_replayed():
    """A forward pass of new tokens, and a training step, in graphs that are replayed over new inputs."""
    H = _host("cpp")
    q, k, wq, wk, gq, gk, g = _data(33, 4, 2, 64, torch.float32)
    positions, sections = _positions(33, 1, g, 0, 100_000), [32]
    f = _frequencies(sections)
    leaves = [t.requires_grad_(True) for t in (q, k, wq, wk)]

    def step():
        out = H.qk_norm_rotary(*leaves, positions, f, sections)
        return [*out, *torch.autograd.grad(out, leaves, (gq, gk))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in (1, 2):
        new = _data(33, 4, 2, 64, torch.float32, seed)
        with torch.no_grad():
            for t, n in zip((q, k, wq, wk, gq, gk), new):
                t.copy_(n)
            positions.copy_(_positions(33, 1, new[6], -50_000, 50_000))
        graph.replay()
        want = R.rotary(q.detach(), k.detach(), positions, f, sections, False, True, wq.detach(), wk.detach(), 1e-6, gq, gk)
        for n, got in zip(("q", "k", "dq", "dk", "dwq", "dwk"), outs):
            check(got, want[n], n)


def test_more_than_2_31_elements():
    rows, d = (1 << 31) // 128 + 1000, 128
    x = torch.empty(rows, 1, d, dtype=torch.bfloat16, device=DEV)
    x.view(-1, 8).copy_(torch.randn(8, generator=_gen(1), device=DEV))
    positions, f = torch.arange(rows, dtype=torch.int32, device=DEV), _frequencies([64])
    y = _host("cpp").rotary_positions(x, positions, f, [64])
    for part in (slice(0, 300), slice(rows // 2, rows // 2 + 300), slice(rows - 300, rows)):
        check(y[part], R.rotary(x[part], None, positions[part], f, [64])["q"])


@pytest.mark.parametrize("host", ["python", "cpp"])
def test_second_derivatives(host):
    """A rotation keeps lengths: the squares of what it makes have the gradient 2 x, and that one 2. The norm's are refused."""
    H = _host(host)
    x = torch.randn(5, 2, 16, device=DEV, requires_grad=True)
    w = torch.ones(16, device=DEV, requires_grad=True)
    positions, f = torch.arange(5, dtype=torch.int32, device=DEV), _frequencies([8])
    v = torch.randn(5, 2, 16, device=DEV)
    first = torch.autograd.grad(H.rotary_positions(x, positions, f, [8]).square().sum(), x, create_graph=True)[0]
    second = torch.autograd.grad(first, x, v)[0]
    # two rotations, each off by 12 roundings of |a| + |b|, no more than twice the largest channel: 48
    for got, want in ((first, 2 * x), (second, 2 * v)):
        assert ((got - want).abs() <= 48 * R.U32 * want.abs().amax(2, keepdim=True)).all()
    grad = torch.autograd.grad(sum(t.sum() for t in H.qk_norm_rotary(x, x, w, w, positions, f, [8])), x, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="qk_norm_rotary is differentiable once only"):
        grad.square().sum().backward()
