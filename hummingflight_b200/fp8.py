"""FP8 (e4m3) operators over libhf_moe.so: quantised rows, the block-scaled
product and the routed SwiGLU experts over FP8 weights (include/hf_fp8.h holds
the formulas).

A value is q * s: q in torch.float8_e4m3fn (or its bits as uint8), s an fp32
scale per 128 columns of a row or per 128 x 128 block of a weight, as FP8
checkpoints store them. Errors raise :class:`HfError` or ValueError; nothing
falls back to the CPU.
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from ._lib import HF_BF16, HF_F32, HfError, HfMoeRouting, call
from .moe import _ACT, check_tensor, new_tensor, on_device, scratch

BLOCK = 128
_Q = (torch.float8_e4m3fn, torch.uint8)
_X = (torch.bfloat16, torch.float32)
_F32 = (torch.float32,)
_I32 = (torch.int32,)


def blocks(n: int) -> int:
    """Scales along n columns (or weight rows)."""
    return (n + BLOCK - 1) // BLOCK


def _code(dtype) -> int:
    return HF_F32 if dtype == torch.float32 else HF_BF16


def quantize(x, q=None, scales=None, stream=None):
    """Rows x [T x K] (device, bf16 or fp32; the rows may lie apart) -> e4m3
    [T x K] and power-of-two fp32 scales [T x ceil(K/128)]. K a multiple of 16."""
    T, K = x.shape
    check_tensor("x", x, _X, (T, K), rows=True)
    dev = x.device
    if q is None:
        q = new_tensor((T, K), torch.float8_e4m3fn, dev, stream)
    else:
        check_tensor("q", q, _Q, (T, K), dev)
    if scales is None:
        scales = new_tensor((T, blocks(K)), torch.float32, dev, stream)
    else:
        check_tensor("scales", scales, _F32, (T, blocks(K)), dev)
    with on_device(dev, stream) as s:
        call("hf_fp8_quantize", x.data_ptr(), _code(x.dtype), _pitch(x), T, K, q.data_ptr(),
             scales.data_ptr(), s)
    return q, scales


def _pitch(x):
    # the stride of a single row is arbitrary
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


@functools.lru_cache(maxsize=256)
def gemm_workspace_size(T: int, N: int, K: int) -> int:
    return int(_lib.lib().hf_fp8_gemm_workspace_size(T, N, K))


def gemm(xq, sx, wq, sw, out=None, out_dtype: str = "bf16", workspace=None, stream=None):
    """(xq * sx) (wq * sw)^T: xq e4m3 [T x K] with scales sx [T x ceil(K/128)]
    (from :func:`quantize`), wq e4m3 [N x K] with scales sw [ceil(N/128) x
    ceil(K/128)] -> [T x N] bf16 or fp32 (the type of `out` when given).
    `workspace`: uint8 scratch of gemm_workspace_size bytes, kept by callers that
    check :func:`status`; without one a bounded wait that gave up shows as NaN only."""
    T, K = xq.shape
    N, _ = wq.shape
    dev = xq.device
    check_tensor("xq", xq, _Q, (T, K))
    check_tensor("sx", sx, _F32, (T, blocks(K)), dev)
    check_tensor("wq", wq, _Q, (N, K), dev)
    check_tensor("sw", sw, _F32, (blocks(N), blocks(K)), dev)
    if out is None:
        out = new_tensor((T, N), torch.float32 if out_dtype == "f32" else torch.bfloat16, dev,
                         stream)
    else:
        check_tensor("out", out, _X, (T, N), dev)
    with on_device(dev, stream) as s:
        need = gemm_workspace_size(T, N, K)
        workspace = scratch(workspace, need, dev, stream)
        call("hf_fp8_gemm", xq.data_ptr(), sx.data_ptr(), wq.data_ptr(), sw.data_ptr(), T, N, K,
             out.data_ptr(), _code(out.dtype),
             None if workspace is None else workspace.data_ptr(), need, s)
    return out


@functools.lru_cache(maxsize=256)
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
    read); resid: [T x H] of out's type, may be `out`. `workspace`: uint8 scratch of
    moe_experts_workspace_size bytes, kept by callers that check :func:`status`; without
    one a bounded wait that gave up shows as NaN only."""
    T, H = x.shape
    dev = x.device
    E, block = experts.shape
    w = routing["topk_weights"]
    _, k = w.shape
    if H == 0:
        raise ValueError("x: rows of no columns")
    I = block // (3 * H)
    check_tensor("x", x, _X, (T, H), rows=True)
    check_tensor("experts", experts, _Q, (E, 3 * I * H), dev)
    check_tensor("scales", scales, _F32, (E, 3 * blocks(I) * blocks(H)), dev)
    check_tensor("topk_weights", w, _F32, (T, k), dev)
    offsets, perm = routing["offsets"], routing["perm"]
    check_tensor("offsets", offsets, _I32, offsets.shape, dev)
    check_tensor("perm", perm, _I32, perm.shape, dev)
    if offsets.numel() < E + 1 or perm.numel() < T * k:
        raise ValueError(f"offsets, perm: {offsets.numel()} and {perm.numel()} entries, {E + 1} "
                         f"and {T * k} are needed")
    if out is None:
        out = new_tensor((T, H), torch.float32 if out_dtype == "f32" else torch.bfloat16, dev,
                         stream)
    else:
        check_tensor("out", out, _X, (T, H), dev)
    if resid is not None:
        check_tensor("resid", resid, (out.dtype,), (T, H), dev)
    r = HfMoeRouting(None, w.data_ptr(), None, None, offsets.data_ptr(), perm.data_ptr(), None)
    code = _code(out.dtype)
    with on_device(dev, stream) as s:
        need = moe_experts_workspace_size(T, k, E, H, I, "f32" if code == HF_F32 else "bf16")
        workspace = scratch(workspace, need, dev, stream)
        call("hf_fp8_moe_experts", experts.data_ptr(), scales.data_ptr(), E, H, I, x.data_ptr(),
             _code(x.dtype), _pitch(x), T, k, r,
             None if resid is None else resid.data_ptr(), out.data_ptr(), code,
             None if workspace is None else workspace.data_ptr(), need, s)
    return out


def status(workspace, stream=None):
    """Waits for the stream; raises HfError (HF_ERR_TIMEOUT) if the last product
    on this workspace hit a bounded-wait timeout (its outputs are right or NaN). The
    stream: that of the product, by default the current one of the workspace's device."""
    with on_device(workspace.device, stream) as s:
        call("hf_fp8_status", workspace.data_ptr(), s)


def set_wait_timeout(ns: int):
    """Limit of every bounded device wait of the products from now on (0: the default, 2 s)."""
    call("hf_fp8_set_wait_timeout", ns)


def debug_stall(block: int):
    """Test hook: the products' copies stop ahead of a CTA's block-th 128 columns of K
    (hf_fp8_debug_stall in include/hf_fp8.h); 0 turns it off."""
    call("hf_fp8_debug_stall", block)


__all__ = ["BLOCK", "blocks", "quantize", "gemm", "gemm_workspace_size", "moe_experts",
           "moe_experts_workspace_size", "status", "set_wait_timeout", "debug_stall", "HfError"]
