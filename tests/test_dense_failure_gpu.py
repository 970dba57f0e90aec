"""Failure path of the dense products without a GPU fault: with one tile's loads
left out, every wait for them gives up after its limit, the status word says so,
the tile is NaN, the others are right, and the context stays usable."""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


def _params(x, w, y, pre, status):
    from selectssm_b200 import _lib
    p = _lib.SSMDenseParams()
    code = _lib.SSM_BF16 if x.dtype == torch.bfloat16 else _lib.SSM_F32
    p.rows, (p.fin, p.fout) = x.shape[0], w.shape
    p.dtype = p.bias_dtype = p.dkernel_dtype = code
    p.act = _lib.ACT_CODES["silu"]
    p.x, p.kernel, p.y, p.pre, p.status = (t.data_ptr() for t in (x, w, y, pre, status))
    n = _lib.load().ssm_dense_fwd_workspace_bytes(ctypes.byref(p))
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device=x.device)
    p.workspace, p.workspace_bytes = ws.data_ptr(), n
    return p, ws


# fp32 and bf16 by one CTA a tile, with the K loop whole and cut, and by pairs of CTAs
@pytest.mark.parametrize("dtype,sizes", [(torch.float32, (300, 96, 257)), (torch.float32, (129, 5000, 136)),
                                         (torch.float32, (2000, 72, 1300)), (torch.bfloat16, (300, 96, 257)),
                                         (torch.bfloat16, (129, 5000, 136)), (torch.bfloat16, (20001, 1536, 776))])
def test_a_wait_that_gives_up_is_reported_and_leaves_nan(cuda, dtype, sizes):
    from selectssm_b200 import _lib
    lib = _lib.load()
    torch.manual_seed(0)
    M, K, N = sizes
    x, w = torch.randn(M, K, device=cuda).to(dtype), (torch.randn(K, N, device=cuda) / K ** 0.5).to(dtype)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    stream = torch.cuda.current_stream().cuda_stream
    runs = []
    for call in (lib.ssm_dense_act_fwd, lambda p, s: lib.ssm_selftest_dense_timeout(p, 1 << 14, s), lib.ssm_dense_act_fwd):
        y, pre = torch.empty(M, N, device=cuda, dtype=dtype), torch.empty(M, N, device=cuda, dtype=dtype)
        p, ws = _params(x, w, y, pre, status)
        status.zero_()
        assert call(ctypes.byref(p), stream) == _lib.SSM_OK
        torch.cuda.synchronize()
        runs.append((y, pre, int(status.item())))
    (y0, pre0, s0), (y1, pre1, s1), (y2, pre2, s2) = runs
    assert (s0, s1, s2) == (0, _lib.SSM_ERR_TIMEOUT, 0)
    assert torch.equal(y0, y2) and torch.equal(pre0, pre2) and bool(torch.isfinite(y0).all())
    tile = 256 if dtype == torch.bfloat16 and M > 8192 else 128
    last = torch.zeros(M, N, dtype=torch.bool, device=cuda)
    last[(M - 1) // tile * tile:, (N - 1) // tile * tile:] = True
    for got, want in ((y1, y0), (pre1, pre0)):
        assert torch.equal(torch.isnan(got), last) and torch.equal(got[~last], want[~last])


def test_refusals_of_the_self_test():
    from selectssm_b200 import _lib
    lib = _lib.load()
    p = _lib.SSMDenseParams()
    p.rows, p.fin, p.fout = 100, 8, 8
    assert lib.ssm_selftest_dense_timeout(ctypes.byref(p), 100, None) == _lib.SSM_ERR_NULL
    p.status = 0x1000
    assert lib.ssm_selftest_dense_timeout(ctypes.byref(p), 1, None) == _lib.SSM_ERR_SHAPE
    assert lib.ssm_selftest_dense_timeout(ctypes.byref(p), (1 << 20) + 1, None) == _lib.SSM_ERR_SHAPE
    p.rows = 16
    assert lib.ssm_selftest_dense_timeout(ctypes.byref(p), 100, None) == _lib.SSM_ERR_SHAPE


@pytest.mark.parametrize("where", ["forward", "backward"])
def test_dense_act_raises_what_an_earlier_call_left(cuda, where):
    from selectssm_b200 import _lib, block_ops, dense_act
    x, w = torch.randn(200, 64, device=cuda, requires_grad=True), torch.randn(64, 72, device=cuda)
    want = dense_act(x, w)  # its status word is the device's
    p, ws = _params(x, w, torch.empty_like(want), torch.empty_like(want), want)
    p.status = block_ops._status_word(x.get_device())
    assert _lib.load().ssm_selftest_dense_timeout(ctypes.byref(p), 1 << 14, torch.cuda.current_stream().cuda_stream) == _lib.SSM_OK
    torch.cuda.synchronize()
    with pytest.raises(_lib.SSMLibraryError, match="earlier dense_act call"):
        dense_act(x, w) if where == "forward" else torch.autograd.grad(want.sum(), x, retain_graph=True)
    assert torch.equal(dense_act(x, w), want)
    torch.autograd.grad(want.sum(), x)


def test_first_call_under_capture(cuda):
    """In a process of its own, where no call has made the status word yet."""
    import os
    import subprocess
    import sys
    code = """if True:
        import torch
        from selectssm_b200 import dense_act
        x, w = torch.randn(200, 64, device="cuda"), torch.randn(64, 72, device="cuda")
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = dense_act(x, w)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, dense_act(x, w))
        """
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
