"""What a bind lays down on the device is there before the first run, whichever
stream that is on and however long the default stream's queue is."""
import ctypes

import pytest
import torch

import momiru_b200 as mb

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("cuda_lib")]
V = mb.DeviceView.from_torch


def leave_ones():
    """Freed device allocations of the small sizes a bind makes, all bits set."""
    rt = ctypes.CDLL("libcudart.so.12")
    made = []
    for nbytes in [4, 256, 4, 256, 4096, 65536]:
        p = ctypes.c_void_p()
        assert rt.cudaMalloc(ctypes.byref(p), ctypes.c_size_t(nbytes)) == 0
        assert rt.cudaMemset(p, 255, ctypes.c_size_t(nbytes)) == 0
        made.append(p)
    torch.cuda.synchronize()
    for p in made:
        assert rt.cudaFree(p) == 0


@pytest.mark.parametrize("dtype,m,n,k,bound", [
    (torch.bfloat16, 300, 520, 1000, 2.0 ** -8), (torch.bfloat16, 16, 512, 2048, 2.0 ** -8),
    (torch.float32, 300, 264, 4096, 1e-5), (torch.float32, 12, 512, 512, 1e-5)])
def test_a_run_right_after_bind_on_another_stream(dtype, m, n, k, bound):
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    lhs, rhs = (torch.randn(*s, generator=g, device="cuda").to(dtype) for s in ((m, k), (k, n)))
    out = torch.zeros(m, n, dtype=dtype, device="cuda")
    want = lhs.double() @ rhs.double()
    stream = torch.cuda.Stream()
    leave_ones()
    torch.cuda.synchronize()
    torch.cuda._sleep(int(3e8))  # the default stream's own work
    op = mb.BoundLinear(mb.LinearNode(), V(lhs), V(rhs), V(out))
    op.replay(stream.cuda_stream)
    stream.synchronize()
    got = torch.empty_like(out)
    with torch.cuda.stream(stream):
        got.copy_(out)
        op.replay(stream.cuda_stream)
    op.quiesce_or_abort(20)
    torch.cuda.synchronize()
    for x in (got, out):
        assert float((x.double() - want).norm() / want.norm()) <= bound
    op.close()
