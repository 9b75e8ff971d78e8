"""The ctypes binding of the dense C ABI on another stream than the current one."""

import pytest
import torch

from vectra_amd.kernels import dense_capi as capi

pytestmark = pytest.mark.gpu


def test_scratch_of_a_call_on_another_stream_is_not_handed_out_early():
    """The call waits on its stream behind a long product; what the current
    stream allocates meanwhile is not the call's workspace."""
    x, w, dy = (torch.randn(*s, device='cuda') for s in ((2000, 256), (512, 256), (2000, 512)))
    want = [torch.empty_like(x), torch.empty_like(w)]
    capi.backward(dy, x, w, dx=want[0], dweight=want[1], activation='gelu')
    got = [torch.empty_like(x), torch.empty_like(w)]
    big = torch.randn(8192, 8192, device='cuda')
    out = torch.empty_like(big)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(8):
            torch.mm(big, big, out=out)
    capi.backward(dy, x, w, dx=got[0], dweight=got[1], activation='gelu', stream=side.cuda_stream)
    # As many blocks of every size as could be the one that was freed.
    markers = [torch.full((n,), 77, dtype=torch.uint8, device='cuda') for n in range(1 << 20, 12 << 20, 1 << 18)]
    torch.cuda.synchronize()
    assert all(bool((m == 77).all()) for m in markers)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_call_on_the_default_and_on_the_current_stream():
    x, w = torch.randn(300, 2048, device='cuda'), torch.randn(520, 2048, device='cuda')
    want = torch.empty(300, 520, device='cuda')
    capi.forward(x, w, out=want)
    for stream in (torch.cuda.default_stream(), torch.cuda.Stream()):
        out = torch.empty_like(want)
        torch.cuda.synchronize()
        capi.forward(x, w, out=out, stream=stream.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            capi.forward(x, w, out=out)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
