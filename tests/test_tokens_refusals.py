"""Layer norm and packed attention: what the C ABI refuses before it touches a GPU, and what the hosts refuse of CPU tensors."""
import ctypes

import pytest
import torch

from riemannengine_b200 import capi, engine


def test_layer_norm_arguments():
    lib = capi.lib()
    p = ctypes.c_void_p(16)  # never read: every call below is refused or has nothing to do
    ok = dict(x=p, ld=64, n=4, c=64, g=p, b=p, pt=0, eps=1e-5, out=p, mean=None, inv=None, dt=0)

    def forward(**change):
        a = {**ok, **change}
        return lib.rmn_layer_norm_forward(a["x"], a["ld"], a["n"], a["c"], a["g"], a["b"], a["pt"], a["eps"], a["out"], a["mean"],
                                          a["inv"], a["dt"], None)

    for change in (dict(c=0), dict(c=65537), dict(dt=2), dict(pt=7), dict(x=None), dict(out=None), dict(mean=p), dict(inv=p),
                   dict(ld=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(n=1 << 31)):
        assert forward(**change) == capi.ERR_BAD_ARG, change
    assert forward(n=0, x=None, out=None) == capi.OK
    assert forward(c=40_000) == capi.ERR_UNSUPPORTED
    assert forward(c=4097, ld=4097) == capi.ERR_UNSUPPORTED
    assert lib.rmn_layer_norm_backward_workspace_bytes(10, 64) == 10 * 2 * 64 * 4
    assert lib.rmn_layer_norm_backward_workspace_bytes(1 << 20, 64) == 592 * 2 * 64 * 4

    def backward(dy=p, x=p, n=4, c=64, mean=p, inv=p, dx=p, dg=p, db=p, ws=p, nbytes=1 << 20, dt=0):
        return lib.rmn_layer_norm_backward(dy, 64, x, 64, n, c, p, 0, mean, inv, dx, dg, db, dt, ws, nbytes, None)

    assert backward(dy=None) == backward(x=None) == backward(mean=None) == backward(inv=None) == capi.ERR_BAD_ARG
    assert backward(ws=None) == backward(ws=ctypes.c_void_p(20)) == backward(dt=3) == capi.ERR_BAD_ARG
    assert backward(nbytes=100) == capi.ERR_ALLOC
    assert backward(dx=None, dg=None, db=None) == capi.OK


def _problem(**change):
    p = capi.Attention()
    for name in ("q", "k", "v", "offsets"):
        setattr(p, name, 16)
    p.q_row = p.k_row = p.v_row = 128
    p.q_head = p.k_head = p.v_head = 32
    p.rows_q = p.rows_k = 10
    p.sequences, p.heads, p.kv_heads, p.dim, p.scale = 2, 4, 4, 32, 0.1
    for name, value in change.items():
        setattr(p, name, value)
    return p


def test_attention_arguments():
    lib = capi.lib()
    p = ctypes.c_void_p(16)
    bad = (dict(heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(heads=65537), dict(dim=0), dict(dtype=2), dict(offsets=None),
           dict(q=None), dict(k=None), dict(v=None), dict(q_row=-1), dict(v_head=-3), dict(rows_k=11), dict(scale=float("nan")),
           dict(rows_q=1 << 31), dict(rows_k=1 << 31), dict(sequences=(1 << 32) - 1))
    for change in bad:
        problem = _problem(**change)
        assert lib.rmn_attention_forward(ctypes.byref(problem), p, None, None, p, 1 << 30, None) == capi.ERR_BAD_ARG, change
        assert lib.rmn_attention_backward(ctypes.byref(problem), p, None, p, p, 128, 32, p, p, p, p, 1 << 30, None) == capi.ERR_BAD_ARG
    assert lib.rmn_attention_forward(None, p, None, None, p, 0, None) == capi.ERR_BAD_ARG
    # few query rows a sample ask for scratch
    few = _problem(rows_q=2, rows_k=100_000, kv_offsets=16)
    need = lib.rmn_attention_forward_workspace_bytes(ctypes.byref(few))
    assert need > 0
    assert lib.rmn_attention_forward(ctypes.byref(few), p, None, None, None, need, None) == capi.ERR_BAD_ARG
    assert lib.rmn_attention_forward(ctypes.byref(few), p, None, None, ctypes.c_void_p(20), need, None) == capi.ERR_BAD_ARG
    assert lib.rmn_attention_forward(ctypes.byref(few), p, None, None, p, need - 1, None) == capi.ERR_ALLOC
    assert lib.rmn_attention_forward_workspace_bytes(ctypes.byref(_problem(rows_q=10_000, rows_k=10_000))) == 0
    assert lib.rmn_attention_forward(ctypes.byref(_problem(dim=257)), p, None, None, p, 1 << 30, None) == capi.ERR_UNSUPPORTED


def test_sample_offsets_arguments():
    lib = capi.lib()
    p = ctypes.c_void_p(16)
    nbytes = lib.rmn_sample_offsets_workspace_bytes(3)
    assert lib.rmn_sample_offsets(p, 5, 1, 3, p, p, nbytes, None) == capi.ERR_BAD_ARG
    assert lib.rmn_sample_offsets(None, 5, 4, 3, p, p, nbytes, None) == capi.ERR_BAD_ARG
    assert lib.rmn_sample_offsets(p, 5, 4, 3, None, p, nbytes, None) == capi.ERR_BAD_ARG
    assert lib.rmn_sample_offsets(p, 5, 4, 3, p, None, nbytes, None) == capi.ERR_BAD_ARG
    assert lib.rmn_sample_offsets(p, 5, 4, 3, p, p, nbytes - 1, None) == capi.ERR_ALLOC


def _hosts():
    from riemannengine_b200 import cpp
    return (engine, cpp.load())


def test_hosts_refuse_cpu_tensors_and_bad_layers():
    x, o = torch.zeros(4, 2, 8), torch.tensor([0, 4], dtype=torch.int32)
    for host in _hosts():
        with pytest.raises(RuntimeError, match="CUDA"):
            host.layer_norm(torch.zeros(3, 8))
        with pytest.raises(RuntimeError, match="CUDA"):
            host.packed_attention(x, x, x, o)
        with pytest.raises(RuntimeError, match="multiple"):
            host.RiemannSelfAttention(30, 4)
        with pytest.raises(RuntimeError, match="multiple"):
            host.RiemannSelfAttention(32, 4, 3)
        layer = host.RiemannSelfAttention(32, 4, 2)
        assert tuple(dict(layer.named_parameters())["qkv.weight"].shape) == (64, 32)


def _layer_norm_on_the_cpu(monkeypatch):
    """engine.layer_norm with torch's arithmetic in the place of the kernels (which leave no graph either)."""
    def forward(x, weight=None, bias=None, eps=1e-5, want_stats=False):
        with torch.no_grad():
            out, mean, inv = torch.native_layer_norm(x, x.shape[1:], weight, bias, eps)
        return (out, mean, inv) if want_stats else (out, None, None)

    def backward(grad_out, x, weight, mean, inv, want_input=True, want_weight=True, want_bias=True, param_dtype=None):
        bias = torch.zeros(x.size(1))
        with torch.no_grad():
            return torch.ops.aten.native_layer_norm_backward(grad_out.contiguous(), x, x.shape[1:], mean, inv, weight, bias,
                                                             [want_input, want_weight, want_bias])

    monkeypatch.setattr(engine.ops, "layer_norm_forward", forward)
    monkeypatch.setattr(engine.ops, "layer_norm_backward", backward)


def test_second_derivatives_are_refused_where_the_first_is_of_a_sum(monkeypatch):
    """The gradient of a sum comes in without a graph; what is made of the layer's own gradient has to be refused all the same, also
    as one of several terms, whose derivative would lack it otherwise."""
    _layer_norm_on_the_cpu(monkeypatch)
    x, w, b = torch.randn(5, 8), torch.randn(8), torch.randn(8)
    for wanted in ((0,), (1,), (0, 1, 2)):
        leaves = [t.clone().requires_grad_(i in wanted) for i, t in enumerate((x, w, b))]
        some = [leaves[i] for i in wanted]
        loss = engine.layer_norm(*leaves).sum()
        grads = torch.autograd.grad(loss, some, create_graph=True)
        for grad in (lambda: (loss + grads[0].square().sum()).backward(retain_graph=True),
                     lambda: torch.autograd.grad(loss + grads[0].square().sum(), some, retain_graph=True)):
            with pytest.raises(RuntimeError, match="layer norm is differentiable once only"):
                grad()
    # a gradient kept with its graph is a tensor like others
    x = x.clone().requires_grad_(True)
    engine.layer_norm(x, w, b).square().sum().backward(create_graph=True)
    want = torch.autograd.grad(torch.nn.functional.layer_norm(x, (8,), w, b).square().sum(), x)[0]
    assert torch.allclose(x.grad, want, atol=1e-5)
    torch.optim.SGD([x], lr=0.1).zero_grad(set_to_none=False)
    assert not x.grad.any() and not x.grad.requires_grad


def test_without_gradients_nothing_is_kept_for_them(monkeypatch):
    """Parameters and features that require gradients, under no_grad: the kernels are not asked for what a backward pass needs."""
    asked = []

    def norm(x, weight=None, bias=None, eps=1e-5, want_stats=False):
        asked.append(want_stats)
        return x.detach().clone(), (x.new_zeros(x.size(0)) if want_stats else None), (x.new_zeros(x.size(0)) if want_stats else None)

    def attention(q, k, v, offsets, kv_offsets=None, kv_lengths=None, causal=False, scale=None, want_stats=False):
        asked.append(want_stats)
        return q.detach().clone(), None, (q.new_zeros(q.size(1), q.size(0)) if want_stats else None)

    monkeypatch.setattr(engine.ops, "layer_norm_forward", norm)
    monkeypatch.setattr(engine.ops, "attention_forward", attention)
    x, w = torch.zeros(4, 8, requires_grad=True), torch.ones(8, requires_grad=True)
    q, o = torch.zeros(4, 2, 8, requires_grad=True), torch.tensor([0, 4], dtype=torch.int32)
    calls = (lambda: engine.layer_norm(x, w), lambda: engine.layer_norm(x.detach(), w), lambda: engine.packed_attention(q, q, q, o),
             lambda: engine.packed_attention(q.detach(), q, q.detach(), o))
    for call in calls:
        assert call().requires_grad
    with torch.no_grad():
        for call in calls:
            assert not call().requires_grad
    assert not engine.layer_norm(x.detach(), w.detach()).requires_grad
    assert asked == [True] * 4 + [False] * 5
