"""Rotary positions: what the C ABI refuses before it touches a GPU, what the hosts refuse, and the helpers that need none."""
import ctypes

import pytest
import torch

from riemannengine_b200 import capi, engine


def _problem(sections=(8, 8), **change):
    p = capi.Rotary()
    for name in ("q", "k", "positions", "frequencies", "q_weight", "k_weight"):
        setattr(p, name, 16)  # never read: every call below is refused or has nothing to do
    p.q_row, p.q_head, p.k_row, p.k_head = 128, 32, 64, 32
    p.rows, p.heads, p.kv_heads, p.dim = 5, 4, 2, 32
    p.position_row, p.position_axis = 2, 1
    p.sections, p.axes = (ctypes.c_int * max(1, len(sections)))(*sections), len(sections)
    p.norm, p.eps = 1, 1e-6
    for name, value in change.items():
        setattr(p, name, value)
    return p


def test_arguments():
    lib, p = capi.lib(), ctypes.c_void_p(16)

    def forward(problem, q=p, k=p):
        return lib.rmn_rotary_forward(ctypes.byref(problem), q, k, None)

    def backward(problem, gq=p, gk=p, dq=p, dk=p, dwq=p, dwk=p, ws=p, nbytes=1 << 30, strides=(128, 32, 64, 32)):
        return lib.rmn_rotary_backward(ctypes.byref(problem), gq, strides[0], strides[1], gk, strides[2], strides[3], dq, dk, dwq, dwk, ws,
                                       nbytes, None)

    bad = [dict(rows=1 << 31), dict(heads=0), dict(kv_heads=-1), dict(heads=65537), dict(dim=0), dict(dim=31), dict(dtype=2), dict(axes=-1),
           dict(axes=9), dict(q=None), dict(k=None), dict(positions=None), dict(frequencies=None), dict(frequencies=20), dict(q_row=-1),
           dict(k_head=-2), dict(position_row=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(weight_dtype=3), dict(sections=(8, 9)),
           dict(sections=(-1, 8)), dict(sections=(2**31 - 1, 2**31 - 1))]
    for change in bad:
        assert forward(_problem(**change)) == capi.ERR_BAD_ARG, change
        assert backward(_problem(**change)) == capi.ERR_BAD_ARG, change
    assert lib.rmn_rotary_forward(None, p, p, None) == capi.ERR_BAD_ARG
    assert lib.rmn_rotary_backward(None, p, 1, 1, p, 1, 1, p, p, p, p, p, 1 << 20, None) == capi.ERR_BAD_ARG
    assert forward(_problem(), q=None) == forward(_problem(), k=None) == capi.ERR_BAD_ARG
    assert forward(_problem(dim=258)) == capi.ERR_UNSUPPORTED
    assert forward(_problem(rows=0, q=None, k=None, positions=None), q=None, k=None) == capi.OK
    for change in (dict(gq=None), dict(gk=None), dict(dq=None), dict(dk=None), dict(ws=None), dict(ws=ctypes.c_void_p(24)),
                   dict(strides=(-1, 32, 64, 32)), dict(strides=(128, 32, 64, -32))):
        assert backward(_problem(), **change) == capi.ERR_BAD_ARG, change
    need = lib.rmn_rotary_backward_workspace_bytes(ctypes.byref(_problem()))
    assert need == 296 * 2 * 32 * 4 and backward(_problem(), nbytes=need - 1) == capi.ERR_ALLOC
    # without a norm there are no weights
    assert lib.rmn_rotary_backward_workspace_bytes(ctypes.byref(_problem(norm=0))) == 0
    assert backward(_problem(norm=0)) == capi.ERR_BAD_ARG
    assert backward(_problem(norm=0, rows=0), dwq=None, dwk=None) == capi.OK
    assert backward(_problem(kv_heads=0)) == capi.ERR_BAD_ARG


def _hosts():
    from riemannengine_b200 import cpp
    return (engine, cpp.load())


def test_hosts_refuse_cpu_tensors():
    x, places, f, w = torch.zeros(4, 2, 8), torch.zeros(4, 1, dtype=torch.int32), torch.zeros(4, dtype=torch.float64), torch.ones(8)
    for host in _hosts():
        with pytest.raises(RuntimeError, match="CUDA"):
            host.rotary_positions(x, places, f, [4])
        with pytest.raises(RuntimeError, match="CUDA"):
            host.qk_norm_rotary(x, x, w, w, places, f, [4])


def test_sections_and_frequencies():
    for host in _hosts():
        assert list(host.rotary_sections(64, 3)) == [11, 11, 10] and list(host.rotary_sections(128, 1)) == [64]
        for bad in ((63, 1), (0, 1), (64, 0), (64, 9)):
            with pytest.raises(RuntimeError, match="even number"):
                host.rotary_sections(*bad)
        f = host.rotary_frequencies([2, 3], 100.0)
        assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1, 0.1, 1, 100 ** (-1 / 3), 100 ** (-2 / 3)], dtype=torch.float64),
                                                           rtol=1e-15, atol=0)
        f = host.rotary_frequencies([2, 3], 32.0, whole=True)
        assert torch.allclose(f, torch.tensor([1, 0.5, 0.25, 0.125, 0.0625], dtype=torch.float64), rtol=1e-15, atol=0)
        assert host.rotary_frequencies([]).numel() == 0
        with pytest.raises(RuntimeError, match="positive base"):
            host.rotary_frequencies([2], 0.0)
        with pytest.raises(RuntimeError, match="not negative"):
            host.rotary_frequencies([-2])


@pytest.mark.gpu
def test_hosts_refuse_what_does_not_fit():
    dev = "cuda:0"
    x, w = torch.zeros(4, 2, 8, device=dev), torch.ones(8, device=dev)
    places, f = torch.zeros(4, 2, dtype=torch.int32, device=dev), torch.zeros(4, dtype=torch.float64, device=dev)
    for host in _hosts():
        for args, text in (((x[..., :7], places, f, [2, 2]), "even number"), ((x, places, f, [2, 3]), "half of the channels"),
                           ((x, places, f, [-2, 2]), "pairs of up to 8"), ((x, places, f, [4]), "one entry per axis"),
                           ((x, places.long(), f, [2, 2]), "int32"), ((x, places[:3], f, [2, 2]), "int32"),
                           ((x, places, f.float(), [2, 2]), "float64"), ((x, places, f[:3], [2, 2]), "one entry per pair"),
                           ((x.half(), places, f, [2, 2]), "dtype"), ((x, None, f, [2, 2]), "need positions"),
                           ((x, places, None, [2, 2]), "need positions"), ((x[0], places, f, [2, 2]), "rows, heads, channels"),
                           ((x, places.cpu(), f, [2, 2]), "CUDA")):
            with pytest.raises(RuntimeError, match=text):
                host.rotary_positions(*args)
        for args, text in (((x, x[:3], w, w, places, f, [2, 2]), "same rows"), ((x, x.bfloat16(), w, w, places, f, [2, 2]), "same dtype"),
                           ((x, x, w[:4], w, places, f, [2, 2]), "one entry per channel"), ((x, x, w, w.bfloat16(), places, f, [2, 2]), "same dtype"),
                           ((x, x, w, w, places, f, [2, 2], -1.0), "eps")):
            with pytest.raises(RuntimeError, match=text):
                host.qk_norm_rotary(*args)
    wide = torch.zeros(2, 1, 258, device=dev)
    for host in _hosts():
        with pytest.raises(RuntimeError, match="unsupported|not supported"):
            host.rotary_positions(wide, places[:2], torch.zeros(129, dtype=torch.float64, device=dev), [100, 29])
