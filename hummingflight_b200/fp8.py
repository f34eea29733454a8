"""FP8 (e4m3) operators over libhf_moe.so: quantised rows, the block-scaled
product and the routed SwiGLU experts over FP8 weights (include/hf_fp8.h holds
the formulas).

A value is q * s: q in torch.float8_e4m3fn (or its bits as uint8), s an fp32
scale per 128 columns of a row or per 128 x 128 block of a weight, as FP8
checkpoints store them. Errors raise :class:`HfError` or ValueError; nothing
falls back to the CPU.
"""
from __future__ import annotations


from . import _lib
from ._lib import HfError, HfMoeRouting, call
from .moe import _ACT, _dtype_code, _ptr, _stream, _torch, check_tensor, on_device, scratch

BLOCK = 128


def blocks(n: int) -> int:
    """Scales along n columns (or weight rows)."""
    return (n + BLOCK - 1) // BLOCK


def _q_types():
    torch = _torch()
    return (torch.float8_e4m3fn, torch.uint8)


def _act_types():
    torch = _torch()
    return (torch.bfloat16, torch.float32)


def quantize(x, q=None, scales=None, stream=None):
    """Rows x [T x K] (device, bf16 or fp32; the rows may lie apart) -> e4m3
    [T x K] and power-of-two fp32 scales [T x ceil(K/128)]. K a multiple of 16."""
    torch = _torch()
    T, K = x.shape
    check_tensor("x", x, _act_types(), (T, K), rows=True)
    dev = x.device
    if q is None:
        q = torch.empty((T, K), dtype=torch.float8_e4m3fn, device=dev)
    else:
        check_tensor("q", q, _q_types(), (T, K), dev)
    if scales is None:
        scales = torch.empty((T, blocks(K)), dtype=torch.float32, device=dev)
    else:
        check_tensor("scales", scales, (torch.float32,), (T, blocks(K)), dev)
    with on_device(dev, stream) as s:
        call("hf_fp8_quantize", x.data_ptr(), _dtype_code(x), _pitch(x), T, K, q.data_ptr(),
             scales.data_ptr(), s)
    return q, scales


def _pitch(x):
    # the stride of a single row is arbitrary
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def gemm_workspace_size(T: int, N: int, K: int) -> int:
    return int(_lib.lib().hf_fp8_gemm_workspace_size(T, N, K))


def gemm(xq, sx, wq, sw, out=None, out_dtype: str = "bf16", workspace=None, stream=None):
    """(xq * sx) (wq * sw)^T: xq e4m3 [T x K] with scales sx [T x ceil(K/128)]
    (from :func:`quantize`), wq e4m3 [N x K] with scales sw [ceil(N/128) x
    ceil(K/128)] -> [T x N] bf16 or fp32 (the type of `out` when given).
    `workspace`: uint8 scratch of gemm_workspace_size bytes, kept by callers that
    check :func:`status`."""
    torch = _torch()
    T, K = xq.shape
    N = wq.shape[0]
    dev = xq.device
    check_tensor("xq", xq, _q_types(), (T, K))
    check_tensor("sx", sx, (torch.float32,), (T, blocks(K)), dev)
    check_tensor("wq", wq, _q_types(), (N, K), dev)
    check_tensor("sw", sw, (torch.float32,), (blocks(N), blocks(K)), dev)
    if out is None:
        out = torch.empty((T, N), dtype=torch.float32 if out_dtype == "f32" else torch.bfloat16,
                          device=dev)
    else:
        check_tensor("out", out, _act_types(), (T, N), dev)
    with on_device(dev, stream) as s:
        need = int(_lib.lib().hf_fp8_gemm_workspace_size(T, N, K))
        workspace = scratch(workspace, need, dev)
        call("hf_fp8_gemm", xq.data_ptr(), sx.data_ptr(), wq.data_ptr(), sw.data_ptr(), T, N, K,
             out.data_ptr(), _dtype_code(out), _ptr(workspace), need, s)
    return out


def moe_experts_workspace_size(T: int, top_k: int, num_experts: int, hidden: int, inter: int,
                               out_dtype: str = "bf16") -> int:
    return int(_lib.lib().hf_fp8_moe_experts_workspace_size(T, top_k, num_experts, hidden, inter,
                                                            _ACT[out_dtype]))


def moe_experts(x, experts, scales, routing: dict, resid=None, out=None, out_dtype: str = "bf16",
                workspace=None, stream=None):
    """The routed SwiGLU experts over FP8 weights: x [T x H] (device, bf16 or
    fp32; the rows may lie apart) -> [T x H] bf16 or fp32 (the type of `out` when
    given), resid + the weighted sum of each token's experts.

    experts: e4m3 [E x 3*I*H], each row one expert's [gate | up | down] block;
    scales: fp32 [E x 3*ceil(I/128)*ceil(H/128)] in the same order; routing: the
    dict of route_logits or MoELayer.route (topk_weights, offsets and perm are
    read); resid: [T x H] of out's type, may be `out`."""
    torch = _torch()
    T, H = x.shape
    dev = x.device
    E = experts.shape[0]
    w = routing["topk_weights"]
    k = w.shape[1]
    I = experts.shape[1] // (3 * H)
    check_tensor("x", x, _act_types(), (T, H), rows=True)
    check_tensor("experts", experts, _q_types(), (E, 3 * I * H), dev)
    check_tensor("scales", scales, (torch.float32,), (E, 3 * blocks(I) * blocks(H)), dev)
    check_tensor("topk_weights", w, (torch.float32,), (T, k), dev)
    offsets, perm = routing["offsets"], routing["perm"]
    for name, t, least in (("offsets", offsets, E + 1), ("perm", perm, T * k)):
        check_tensor(name, t, (torch.int32,), t.shape, dev)
        if t.numel() < least:
            raise ValueError(f"{name}: {t.numel()} entries, {least} are needed")
    if out is None:
        out = torch.empty((T, H), dtype=torch.float32 if out_dtype == "f32" else torch.bfloat16,
                          device=dev)
    else:
        check_tensor("out", out, _act_types(), (T, H), dev)
    if resid is not None:
        check_tensor("resid", resid, (out.dtype,), (T, H), dev)
    r = HfMoeRouting(None, w.data_ptr(), None, None, offsets.data_ptr(), perm.data_ptr(), None)
    code = _dtype_code(out)
    with on_device(dev, stream) as s:
        need = int(_lib.lib().hf_fp8_moe_experts_workspace_size(T, k, E, H, I, code))
        workspace = scratch(workspace, need, dev)
        call("hf_fp8_moe_experts", experts.data_ptr(), scales.data_ptr(), E, H, I, x.data_ptr(),
             _dtype_code(x), _pitch(x), T, k, r, _ptr(resid), out.data_ptr(), code,
             _ptr(workspace), need, s)
    return out


def status(workspace, stream=None):
    """Waits for the stream; raises HfError (HF_ERR_TIMEOUT) if the last product
    on this workspace hit a bounded-wait timeout."""
    call("hf_fp8_status", _ptr(workspace), _stream(stream))


__all__ = ["BLOCK", "blocks", "quantize", "gemm", "gemm_workspace_size", "moe_experts",
           "moe_experts_workspace_size", "status", "HfError"]
