"""Attention with a window: what the C ABI refuses before it touches a GPU; and the mask of the tests, against the words that describe
it."""
import ctypes

from riemannengine_b200 import capi
from tests import plain_window as W


def _problem(**change):
    p = capi.Attention()
    for name in ("q", "k", "v", "offsets"):
        setattr(p, name, 16)  # never read: every call below is refused
    p.q_row = p.k_row = p.v_row = 128
    p.q_head = p.k_head = p.v_head = 32
    p.rows_q = p.rows_k = 10
    p.sequences, p.heads, p.kv_heads, p.dim, p.scale = 2, 4, 4, 32, 0.1
    for name, value in change.items():
        setattr(p, name, value)
    return p


def test_arguments():
    lib, p = capi.lib(), ctypes.c_void_p(16)
    big = 1 << 30

    def forward(problem, window=5, sinks=1, ws=p, nbytes=big):
        return lib.rmn_window_attention_forward(ctypes.byref(problem), window, sinks, p, None, None, ws, nbytes, None)

    def backward(problem, window=5, sinks=1, ws=p, nbytes=big):
        return lib.rmn_window_attention_backward(ctypes.byref(problem), window, sinks, p, None, p, p, 128, 32, p, p, p, ws, nbytes, None)

    for window, sinks in ((0, 0), (-1, 0), (5, -1), (5, 1 << 30)):
        assert forward(_problem(), window, sinks) == backward(_problem(), window, sinks) == capi.ERR_BAD_ARG
        for size in (lib.rmn_window_attention_forward_workspace_bytes, lib.rmn_window_attention_backward_workspace_bytes):
            assert size(ctypes.byref(_problem()), window, sinks) == 0
    for change in (dict(heads=0), dict(kv_heads=3), dict(dim=0), dict(dtype=2), dict(offsets=None), dict(q=None), dict(v_head=-3),
                   dict(rows_k=11), dict(scale=float("nan"))):
        assert forward(_problem(**change)) == backward(_problem(**change)) == capi.ERR_BAD_ARG, change
    assert forward(_problem(dim=257)) == capi.ERR_UNSUPPORTED
    need = lib.rmn_window_attention_backward_workspace_bytes(ctypes.byref(_problem()), 5, 1)
    assert need >= 4 * 10 * 4
    assert backward(_problem(), nbytes=need - 1) == capi.ERR_ALLOC
    assert backward(_problem(), ws=None) == backward(_problem(), ws=ctypes.c_void_p(20)) == capi.ERR_BAD_ARG


def test_mask():
    see = W.seen(4, 6, 2, 1, True)  # places 2 ... 5
    assert see.int().tolist() == [[1, 1, 1, 0, 0, 0], [1, 0, 1, 1, 0, 0], [1, 0, 0, 1, 1, 0], [1, 0, 0, 0, 1, 1]]
    see = W.seen(3, 2, 1, 0, False)  # places -1, 0, 1
    assert see.int().tolist() == [[0, 0], [1, 0], [0, 1]]
    see = W.seen(2, 5, 2, 2, False)  # places 3, 4
    assert see.int().tolist() == [[1, 1, 1, 1, 1], [1, 1, 0, 1, 1]]
