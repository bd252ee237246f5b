"""Layer norm over the channels of every row: both hosts against 64 bits, forward and backward."""
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
        return cpp.load().layer_norm
    from riemannengine_b200 import engine
    return engine.layer_norm


def _inputs(n, c, dtype, ptype=None, seed=0, shift=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 7919 + n * 31 + c)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    ptype = dtype if ptype is None else ptype
    x = (r(n, c) * (r(c).abs() + 0.2) + shift * r(c)).to(dtype)
    return x, (1 + 0.3 * r(c)).to(ptype), (0.3 * r(c)).to(ptype), r(n, c).to(dtype)


def _run(host, x, w, b, dy, eps=1e-5):
    leaves = [t.detach().clone().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    y = _host(host)(*leaves, eps)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    return y, grads


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,c", [(1, 1), (1, 64), (2, 7), (37, 16), (5, 24), (300, 32), (257, 33), (1000, 64), (129, 96), (64, 100),
                                 (33, 128), (9, 130), (50, 256), (17, 384), (21, 512), (16, 513), (10, 1000), (7, 1024), (5, 2048),
                                 (3, 4096), (3, 20480), (2, 16384)])
def test_against_64_bits(dtype, n, c):
    if dtype == "f32" and c == 20480:
        pytest.skip("beyond what a block's registers hold in fp32")
    x, w, b, dy = _inputs(n, c, TYPES[dtype])
    want = P.layer_norm(x, w, b, 1e-5, dy)
    y, (dx, dw, db) = _run("cpp", x, w, b, dy)
    for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        assert got.dtype == TYPES[dtype]
        P.check(got, want[name], f"{name} {n}x{c}")


@pytest.mark.parametrize("host", ["python", "cpp"])
@pytest.mark.parametrize("dtype,ptype", [("f32", "f32"), ("bf16", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
def test_parameters_of_either_type_present_or_not(host, dtype, ptype):
    x, w, b, dy = _inputs(70, 40, TYPES[dtype], TYPES[ptype])
    for ww, bb in ((w, b), (w, None), (None, b), (None, None)):
        want = P.layer_norm(x, ww, bb, 1e-3, dy)
        y, grads = _run(host, x, ww, bb, dy, 1e-3)
        P.check(y, want["y"])
        names = ["dx"] + (["dw"] if ww is not None else []) + (["db"] if bb is not None else [])
        for name, got in zip(names, grads):
            P.check(got, want[name], name)
            assert got.dtype == (TYPES[dtype] if name == "dx" else TYPES[ptype])


@pytest.mark.parametrize("host", ["python", "cpp"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_rows(host, dtype):
    """More rows than one round of all blocks; the sums over them and the last ragged group."""
    x, w, b, dy = _inputs(60_001, 64, TYPES[dtype])
    want = P.layer_norm(x, w, b, 1e-5, dy)
    y, (dx, dw, db) = _run(host, x, w, b, dy)
    for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        P.check(got, want[name], name)
    again = _run(host, x, w, b, dy)
    assert torch.equal(again[1][1], dw) and torch.equal(again[1][2], db)  # no order of atomics in the sums


@pytest.mark.parametrize("host", ["python", "cpp"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_alignment(host, dtype):
    t = TYPES[dtype]
    x, w, b, dy = _inputs(100, 64, t)
    wide = torch.zeros(100, 200, dtype=t, device=DEV)
    for first in (0, 8, 1, 3):  # rows apart, aligned and not
        view = wide[:, first:first + 64]
        view.copy_(x)
        want = P.layer_norm(x, w, b, 1e-5, dy)
        leaf = view.detach().requires_grad_(True)
        y = _host(host)(leaf, w, b, 1e-5)
        assert y.is_contiguous()
        P.check(y, want["y"], f"first {first}")
        (dx,) = torch.autograd.grad(y, leaf, dy)
        P.check(dx, want["dx"], f"first {first}")
    # transposed features, an expanded gradient, parameters that are no contiguous vectors
    xt = x.t().contiguous().t().requires_grad_(True)
    row = dy[:1].expand(100, 64)
    w2 = torch.stack([w, w], 1)[:, 0].requires_grad_(True)
    assert w2.stride(0) == 2
    want = P.layer_norm(x, w, b, 1e-5, row)
    y = _host(host)(xt, w2, b, 1e-5)
    dx, dw = torch.autograd.grad(y, (xt, w2), row)
    P.check(y, want["y"])
    P.check(dx, want["dx"])
    P.check(dw, want["dw"])
    y = _host(host)(xt, w2, b, 1e-5)
    (dx,) = torch.autograd.grad(y.sum(), xt)  # a gradient with no strides at all
    P.check(dx, P.layer_norm(x, w, b, 1e-5, torch.ones_like(x))["dx"])


@pytest.mark.parametrize("host", ["python", "cpp"])
def test_empty_constant_far_and_non_finite_rows(host):
    f = _host(host)
    w = torch.ones(32, device=DEV, requires_grad=True)
    b = torch.zeros(32, device=DEV, requires_grad=True)
    x = torch.zeros(0, 32, device=DEV, requires_grad=True)
    y = f(x, w, b, 1e-5)
    assert y.shape == (0, 32)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros(0, 32, device=DEV))
    assert dx.shape == (0, 32) and not dw.any() and not db.any()
    # a row of one value is that of the bias; far from zero its own spread still counts
    x = torch.full((3, 32), 1e4, device=DEV)
    x[1] += torch.arange(32, device=DEV) * 0.25
    x[2, 5] = float("nan")
    y = f(x, w, b, 1e-5)
    assert not y[0].any() and torch.isnan(y[2]).all()
    P.check(y[:2], P.layer_norm(x[:2], w.detach(), b.detach(), 1e-5)["y"])
    x[2, 5] = float("inf")
    assert torch.isnan(f(x, w, b, 1e-5)[2]).all() and torch.isfinite(f(x, w, b, 1e-5)[:2]).all()


@pytest.mark.parametrize("host", ["python", "cpp"])
def test_gradient_against_differences(host):
    x, w, b, dy = _inputs(23, 48, torch.float32)
    _, grads = _run(host, x, w, b, dy)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(5)
    step = 1e-5
    for i, t in enumerate((x, w, b)):
        way = torch.randn(t.shape, generator=gen, device=DEV, dtype=torch.float64)
        value = []
        for s in (step, -step):
            args = [a.double() for a in (x, w, b)]
            args[i] = args[i] + s * way
            value.append((P.layer_norm(*args, 1e-5)["y"][0] * dy.double()).sum().item())
        slope = (value[0] - value[1]) / (2 * step)
        got = (grads[i].double() * way).sum().item()
        size = (grads[i].double() * way).abs().sum().item()
        # fp32 gradients: a thousand roundings of the terms at most; differences: step^2 times the third derivative
        assert abs(got - slope) <= 1000 * P.U32 * size + 1e-7 * size


def test_layers_of_both_hosts_agree_with_the_function():
    from riemannengine_b200 import cpp, engine
    host = cpp.load()
    coords = torch.tensor([[s, i, 0, 0] for s in range(2) for i in range(40)], dtype=torch.int32, device=DEV)
    x, w, b, _ = _inputs(80, 48, torch.float32)
    want = P.layer_norm(x, w, b, 1e-5)["y"]
    for layer, tensor in ((host.RiemannLayerNorm(48), host.SparseTensor(x, coords)),
                          (engine.RiemannLayerNorm(48), engine.SparseTensor(x, coords))):
        layer.to(torch.device(DEV) if isinstance(layer, torch.nn.Module) else DEV)
        params = dict(layer.named_parameters())
        assert set(params) == {"normalization.weight", "normalization.bias"}
        with torch.no_grad():
            params["normalization.weight"].copy_(w)
            params["normalization.bias"].copy_(b)
        y = layer(tensor)
        P.check(y.F, want)
        assert y.F.requires_grad and y.coordinate_map_key == tensor.coordinate_map_key
        with pytest.raises(RuntimeError, match="channel count"):
            layer(type(tensor)(x[:, :32], coords))


@pytest.mark.parametrize("host", ["python", "cpp"])
def test_on_a_stream_and_captured(host):
    f = _host(host)
    x, w, b, dy = _inputs(2000, 64, torch.bfloat16)
    for t in (x, w, b):
        t.requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(f(x, w, b, 1e-5), (x, w, b), dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = f(x, w, b, 1e-5)
        grads = torch.autograd.grad(y, (x, w, b), dy)
    for seed in (1, 2):
        x2, w2, b2, dy2 = _inputs(2000, 64, torch.bfloat16, seed=seed)
        with torch.no_grad():
            for t, new in ((x, x2), (w, w2), (b, b2)):
                t.copy_(new)
            dy.copy_(dy2)
        graph.replay()
        want = P.layer_norm(x2, w2, b2, 1e-5, dy2)
        for name, got in (("y", y), ("dx", grads[0]), ("dw", grads[1]), ("db", grads[2])):
            P.check(got, want[name], name)


@pytest.mark.parametrize("host", ["python", "cpp"])
def test_sizes_that_do_not_fit_are_refused(host):
    with pytest.raises(RuntimeError, match="2\\^31"):
        _host(host)(torch.zeros(1, 8, device=DEV).expand(2**32 + 1, 8), None, None, 1e-5)


def test_more_than_2_31_elements():
    """The last rows of a tensor of 4 GB, forward and backward; the others are zero."""
    n, c, last = (1 << 31) // 64 + 1000, 64, 500
    x, w, b, dy = _inputs(last, c, torch.bfloat16)
    many, grad = (torch.zeros(n, c, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    many[-last:], grad[-last:] = x, dy
    want = P.layer_norm(x, w, b, 1e-5, dy)
    y, (dx, dw, db) = _run("cpp", many, w, b, grad)
    for name, got in (("y", y[-last:]), ("dx", dx[-last:]), ("dw", dw), ("db", db)):
        P.check(got, want[name], name)
    assert torch.equal(y[:1000], b.expand(1000, c)) and not dx[:1000].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,c", [(5, 3), (1000, 64), (300, 1024), (7, 5000)])
def test_in_place(dtype, n, c):
    """The C calls may write over x and over dy."""
    from riemannengine_b200 import capi, ops
    x, w, b, dy = _inputs(n, c, TYPES[dtype])
    want = P.layer_norm(x, w, b, 1e-5, dy)
    code, pcode = (capi.F32 if t.dtype == torch.float32 else capi.BF16 for t in (x, w))
    lib, p = capi.lib(), lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    y, stats = x.clone(), torch.empty(2, n, device=DEV)
    assert lib.rmn_layer_norm_forward(p(y), c, n, c, p(w), p(b), pcode, 1e-5, p(y), p(stats[0]), p(stats[1]), code, stream) == 0
    P.check(y, want["y"], "y")
    dx, dw, db = dy.clone(), torch.empty_like(w), torch.empty_like(b)
    nbytes = lib.rmn_layer_norm_backward_workspace_bytes(n, c)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
    assert lib.rmn_layer_norm_backward(p(dx), c, p(x), c, n, c, p(w), pcode, p(stats[0]), p(stats[1]), p(dx), p(dw), p(db), code,
                                       p(ws), nbytes, stream) == 0
    for name, got in (("dx", dx), ("dw", dw), ("db", db)):
        P.check(got, want[name], name)


@pytest.mark.parametrize("host", ["python", "cpp"])
def test_refusals(host):
    f = _host(host)
    x = torch.randn(8, 32, device=DEV)
    w = torch.ones(32, device=DEV)
    for args in ((x[0], w, w), (x, w[:31], w), (x, w, torch.ones(32, 1, device=DEV)), (x, w, w.bfloat16()), (x.half(), w, w),
                 (x.double(), w, w), (x, w.half(), w.half()), (x.cpu(), w, w), (x, w.cpu(), w)):
        with pytest.raises(RuntimeError):
            f(*args, 1e-5)
    with pytest.raises(RuntimeError):
        f(x, w, w, -1.0)
    with pytest.raises(RuntimeError, match="unsupported"):
        f(torch.zeros(2, 40_000, device=DEV), None, None, 1e-5)
    # differentiable once
    a = x.clone().requires_grad_(True)
    dy = torch.ones_like(x, requires_grad=True)
    with pytest.raises(RuntimeError, match="once|differentiate twice"):
        (g,) = torch.autograd.grad(f(a, w, w, 1e-5), a, dy, create_graph=True)
        g.sum().backward()


@pytest.mark.parametrize("host", ["python", "cpp"])
def test_second_derivatives_are_refused_where_the_first_is_of_a_sum(host):
    x, w, b, _ = _inputs(9, 32, torch.float32)
    for wanted in ((0,), (1,), (0, 1, 2)):
        leaves = [t.clone().requires_grad_(i in wanted) for i, t in enumerate((x, w, b))]
        some = [leaves[i] for i in wanted]
        loss = _host(host)(*leaves, 1e-5).sum()
        grads = torch.autograd.grad(loss, some, create_graph=True)
        want = P.layer_norm(x, w, b, 1e-5, torch.ones_like(x))
        for i, g in zip(wanted, grads):
            P.check(g, want[("dx", "dw", "db")[i]])
        for grad in (lambda: (loss + grads[0].square().sum()).backward(retain_graph=True),
                     lambda: torch.autograd.grad(loss + grads[0].square().sum(), some, retain_graph=True)):
            with pytest.raises(RuntimeError, match="layer norm is differentiable once only"):
                grad()


@pytest.mark.parametrize("host", ["python", "cpp"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_wide_rows_at_any_alignment(host, dtype):
    """Rows beyond what is read one channel at a time: features and gradients that are parts of wider matrices (as behind a concatenation)."""
    t, c = TYPES[dtype], 5000
    x, w, b, dy = _inputs(5, c, t)
    want = P.layer_norm(x, w, b, 1e-5, dy)
    for first, room in ((1, 1), (8, 11), (0, 1)):
        whole, grads = (torch.zeros(5, first + c + room, dtype=t, device=DEV) for _ in range(2))
        view, dview = whole[:, first:first + c], grads[:, first:first + c]
        view.copy_(x)
        dview.copy_(dy)
        leaf, ww, bb = view.detach().requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)
        y = _host(host)(leaf, ww, bb, 1e-5)
        got = (y, *torch.autograd.grad(y, (leaf, ww, bb), dview))
        for name, value in zip(("y", "dx", "dw", "db"), got):
            P.check(value, want[name], f"{name} {first} {room}")
    one = _host(host)(view[2:3], w, b, 1e-5)
    P.check(one, tuple(v[2:3] for v in want["y"]))


@pytest.mark.parametrize("host", ["python", "cpp"])
def test_the_widest_rows_with_parameter_gradients_are_refused_by_the_forward_pass(host):
    x, w, b, dy = _inputs(2, 32768, torch.bfloat16)
    f = _host(host)
    for leaves in ((x, w.clone().requires_grad_(True), b), (x, None, b.clone().requires_grad_(True))):
        with pytest.raises(RuntimeError, match="25600"):
            f(*leaves, 1e-5)
        with torch.no_grad():
            f(*leaves, 1e-5)
    leaf = x.clone().requires_grad_(True)  # without them the widest rows have a backward pass
    y = f(leaf, w, b, 1e-5)
    want = P.layer_norm(x, w, b, 1e-5, dy)
    P.check(y, want["y"])
    P.check(torch.autograd.grad(y, leaf, dy)[0], want["dx"])
