"""Attention over caches captured by other means than torch.cuda.graph: a call that needs no workspace
runs in the replays, one that needs a workspace is refused (torch would hand it on before them)."""
import ctypes

import pytest
import torch

from pyasc_amd import kernels
from test_gpu_workspace_streams import _hip

pytestmark = pytest.mark.gpu


def _case(kv_len, device):
    g = torch.Generator(device=device).manual_seed(kv_len)

    def rows(*shape):
        return torch.randn(shape, generator=g, device=device).bfloat16()

    q, d = rows(1, 4, 3, 64), rows(1, 2, 3, 64)
    k, v = rows(1, 2, kv_len, 64), rows(1, 2, kv_len, 64)
    n = torch.full((1,), kv_len, dtype=torch.int32, device=device)
    return lambda o, stream=None: kernels.tree_attention(q, k, v, n, d, d, None, o, 0.125, stream=stream), q


@pytest.mark.parametrize("current", [True, False])
def test_a_call_without_a_workspace(device, current):
    hip, relaxed = _hip(), 2
    call, q = _case(100, device)
    out, want = torch.empty_like(q), torch.empty_like(q)
    call(want)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph, executable = ctypes.c_void_p(), ctypes.c_void_p()
    with torch.cuda.stream(s if current else torch.cuda.current_stream()):
        assert hip.hipStreamBeginCapture(s.cuda_stream, relaxed) == 0
        call(out, None if current else s)
        assert hip.hipStreamEndCapture(s.cuda_stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(executable), graph, None, None, 0) == 0
    for _ in range(3):
        out.zero_()
        q.copy_(torch.randn(q.shape, device=device))
        call(want)
        torch.cuda.synchronize()
        assert hip.hipGraphLaunch(executable, s.cuda_stream) == 0
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert hip.hipGraphExecDestroy(executable) == 0 and hip.hipGraphDestroy(graph) == 0


@pytest.mark.parametrize("current", [True, False])
def test_a_call_with_a_workspace_is_refused(device, current):
    hip, relaxed = _hip(), 2
    call, q = _case(20000, device)
    out = torch.empty_like(q)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = ctypes.c_void_p()
    with torch.cuda.stream(s if current else torch.cuda.current_stream()):
        assert hip.hipStreamBeginCapture(s.cuda_stream, relaxed) == 0
        try:
            with pytest.raises(RuntimeError, match="torch.cuda.graph"):
                call(out, None if current else s)
        finally:
            assert hip.hipStreamEndCapture(s.cuda_stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphDestroy(graph) == 0
    call(out)  # and works again outside of it
    torch.cuda.synchronize()
    assert torch.isfinite(out.float()).all()
