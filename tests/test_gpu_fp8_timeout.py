"""The FP8 products' bounded waits run out (no GPU fault is involved: the copies stop
and wait on a barrier that nothing signals, under a limit of 1 ms). The call returns,
hf_fp8_status reports HF_ERR_TIMEOUT, outputs without their sum are NaN, and the next
call on the workspace is right."""
import contextlib

import numpy as np
import pytest

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu


def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def test_hooks_take_and_refuse():
    from hummingflight_b200 import _lib, fp8
    L = _lib.lib()
    assert L.hf_fp8_debug_stall(-2 ** 31) == _lib.HF_ERR_ARG
    fp8.set_wait_timeout(0)
    fp8.debug_stall(0)


@contextlib.contextmanager
def stalled(block):
    from hummingflight_b200 import fp8
    fp8.set_wait_timeout(1_000_000)
    fp8.debug_stall(block)
    try:
        yield
    finally:
        torch.cuda.synchronize()
        fp8.debug_stall(0)
        fp8.set_wait_timeout(0)


def run(call, ws, blocks):
    from hummingflight_b200 import fp8
    good = call().clone()
    fp8.status(ws)
    for block in blocks:
        with stalled(block):
            bad = call()
            with pytest.raises(fp8.HfError) as e:
                fp8.status(ws)
            assert e.value.status == 4  # HF_ERR_TIMEOUT
            assert bad.isnan().all() if abs(block) == 1 else bad.isnan().any()
            assert ((bad == good) | bad.isnan()).all()
        again = call()
        fp8.status(ws)
        assert torch.equal(again, good)


# tiles of 32 and 64 positions, CTA pairs; one tile a CTA, several, runs of K. Blocks: the
# first, one with MMAs and copies in flight, one of a later tile
@gpu
@pytest.mark.parametrize("T,N,K,blocks", [
    (8, 600, 2048, (1, 2)), (64, 640, 384, (1, 3)), (40, 40100, 256, (1, 2, 4)),
    (64, 40100, 256, (2, 3)), (300, 512, 2048, (1, 4, -1, -4)), (300, 20000, 272, (2, 5, -2, -5))])
def test_product(T, N, K, blocks):
    need_gpu()
    from hummingflight_b200 import fp8
    g = torch.Generator(device="cuda").manual_seed(T + N)
    xq, sx = fp8.quantize(torch.randn((T, K), generator=g, device="cuda"))
    wq = torch.randn((N, K), generator=g, device="cuda").mul_(50).to(torch.float8_e4m3fn)
    sw = torch.rand((fp8.blocks(N), fp8.blocks(K)), generator=g, device="cuda")
    ws = torch.empty(fp8.gemm_workspace_size(T, N, K), dtype=torch.uint8, device="cuda")
    run(lambda: fp8.gemm(xq, sx, wq, sw, workspace=ws), ws, blocks)


# gate/up and down, of tiles of 32 and 64 positions (also in runs of K) and CTA pairs
@gpu
@pytest.mark.parametrize("T,E,k,H,I,blocks", [
    (3, 4, 2, 2048, 384, (1, 3)), (40, 8, 2, 512, 384, (1, 2, 4)), (100, 64, 8, 256, 640, (1, 2, 5)),
    (120, 4, 2, 640, 256, (1, 3)), (400, 16, 2, 512, 1024, (2, 5)),
    (900, 4, 2, 640, 512, (1, 4, -1, -4)), (3000, 8, 2, 512, 1024, (2, 9, -2, -9))])
def test_experts(T, E, k, H, I, blocks):
    need_gpu()
    from hummingflight_b200 import fp8, moe
    g = torch.Generator(device="cuda").manual_seed(T)
    q = torch.randn((E, 3 * I * H), generator=g, device="cuda").mul_(50).to(torch.float8_e4m3fn)
    s = torch.rand((E, 3 * fp8.blocks(I) * fp8.blocks(H)), generator=g, device="cuda") * 1e-3
    x = torch.randn((T, H), generator=g, device="cuda").bfloat16()
    r = moe.route_logits(torch.randn((T, E), generator=g, device="cuda"), None, k, "softmax")
    ws = torch.empty(fp8.moe_experts_workspace_size(T, k, E, H, I), dtype=torch.uint8,
                     device="cuda")
    run(lambda: fp8.moe_experts(x, q, s, r, workspace=ws), ws, blocks)


@gpu
def test_captured_limit_stays():
    """A graph keeps the limit and the hook that were in force at its capture."""
    need_gpu()
    from hummingflight_b200 import fp8
    T, N, K = 8, 512, 1024
    xq, sx = fp8.quantize(torch.randn((T, K), device="cuda"))
    wq = torch.randn((N, K), device="cuda").to(torch.float8_e4m3fn)
    sw = torch.ones((fp8.blocks(N), fp8.blocks(K)), device="cuda")
    ws = torch.empty(fp8.gemm_workspace_size(T, N, K), dtype=torch.uint8, device="cuda")
    y = fp8.gemm(xq, sx, wq, sw, workspace=ws)
    good, graphs = y.clone(), []
    for block in (0, 1):
        graphs.append(torch.cuda.CUDAGraph())
        with stalled(block), torch.cuda.graph(graphs[-1]):
            fp8.gemm(xq, sx, wq, sw, y, workspace=ws)
    for _ in range(2):
        graphs[1].replay()
        with pytest.raises(fp8.HfError):
            fp8.status(ws)
        graphs[0].replay()
        fp8.status(ws)
        assert np.array_equal(y.float().cpu().numpy(), good.float().cpu().numpy())


@gpu
def test_longest_limit():
    """The largest number of nanoseconds is a long limit, not none."""
    need_gpu()
    from hummingflight_b200 import fp8
    fp8.set_wait_timeout(2 ** 64 - 1)
    try:
        for T in (8, 300):
            xq, sx = fp8.quantize(torch.ones((T, 6144), device="cuda"))
            wq = torch.ones((2048, 6144), device="cuda").to(torch.float8_e4m3fn)
            sw = torch.ones((16, 48), device="cuda")
            ws = torch.empty(fp8.gemm_workspace_size(T, 2048, 6144), dtype=torch.uint8,
                             device="cuda")
            assert (fp8.gemm(xq, sx, wq, sw, out_dtype="f32", workspace=ws) == 6144).all()
            fp8.status(ws)
    finally:
        fp8.set_wait_timeout(0)
