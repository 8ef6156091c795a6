"""A launch of the layer for a few tokens that fails is that call's error and no other's."""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_a_launch_that_fails_is_not_reported_again_by_the_next_call():
    """The launch fails on the host: its stream is under a capture that a synchronisation has ended (an error the
    runtime returns, nothing reaches the GPU). The next call, on a stream of its own, is healthy."""
    from mlops_b200 import layer, ops

    g = torch.Generator().manual_seed(1)
    new = lambda *shape: (torch.randn(*shape, generator=g) * 0.1).bfloat16().to(DEV)  # noqa: E731
    x, router, w13, w2 = new(3, 256), new(8, 256), new(8, 256, 256), new(8, 256, 128)
    rows = ops.quantize_rows(x)
    call = lambda: layer.forward_decode(x, x, router, w13, w2, top_k=2, routing_mode="softmax_then_topk")  # noqa: E731
    good = call()
    torch.cuda.synchronize()
    runtime = ctypes.CDLL("libcudart.so.12")
    stream = torch.cuda.Stream()
    handle, graph = ctypes.c_void_p(stream.cuda_stream), ctypes.c_void_p()
    with torch.cuda.stream(stream):
        buffers = [torch.empty(1 << 20, dtype=torch.uint8, device=DEV) for _ in range(4)]  # (the call allocates on it)
        del buffers
        call()
        torch.cuda.synchronize()
        assert runtime.cudaStreamBeginCapture(handle, 2) == 0
        assert runtime.cudaStreamSynchronize(handle) != 0  # not allowed under capture: the capture is void
        try:
            with pytest.raises(ops.NativeError, match="launch"):
                call()
        finally:
            runtime.cudaStreamEndCapture(handle, ctypes.byref(graph))
            runtime.cudaGetLastError()
    again = ops.quantize_rows(x)
    assert torch.equal(rows[0].view(torch.uint8), again[0].view(torch.uint8)) and torch.equal(rows[1], again[1])
    assert all(torch.equal(a, b) for a, b in zip(call(), good))
    ops.check_status(DEV)
