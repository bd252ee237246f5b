"""A thread's first call, before it has called the CUDA runtime, runs the same kernels as any other: the same bits."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _of_a_new_thread(f):
    got = []
    thread = threading.Thread(target=lambda: got.append(f()))
    thread.start()
    thread.join()
    assert got, "the thread failed"
    return got[0]


@pytest.mark.parametrize("window", [None, 40])
@pytest.mark.parametrize("d", [64, 128])
def test_attention(d, window):
    from riemannengine_b200 import cpp
    attend = cpp.load().packed_attention
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    q, k, v = (torch.randn(300, 4, d, generator=g, device=DEV).bfloat16() for _ in range(3))
    offsets = torch.tensor([0, 120, 300], dtype=torch.int32, device=DEV)

    def run():
        with torch.no_grad():
            return attend(q, k, v, offsets, causal=True, window=window)

    for _ in range(3):  # the outputs' memory is there when the thread asks for it
        want = run()
        torch.cuda.synchronize()
    assert torch.equal(_of_a_new_thread(run), want)
