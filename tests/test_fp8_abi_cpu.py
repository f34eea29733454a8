"""Routing and FP8 entry points without a GPU: exported, bound, and every refusal
made on the host (the fake pointers are never dereferenced)."""
import ctypes
import os
import re

import pytest

from hummingflight_b200 import _lib

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P, WS = 0x10000, 0x100000


def declared():
    src = open(os.path.join(ROOT, "include", "hf_fp8.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    return re.findall(r"^\s*HF_API\s+[\w\s\*]*?\b(hf_\w+)\s*\(", src, flags=re.M)


def test_declared_symbols_are_exported_and_bound():
    names = declared()
    assert len(names) >= 6
    L = ctypes.CDLL(_lib.LIB_PATH)
    for n in names + ["hf_route_logits", "hf_route_workspace_size"]:
        assert hasattr(L, n) and n in _lib.SIGNATURES


def spec(**kw):
    v = dict(num_experts=64, top_k=8, score=0, n_group=1, topk_group=1, group_top=2, scale=1.0,
             norm=1)
    v.update(kw)
    return _lib.HfRouteSpec(*v.values())


def test_route_refusals():
    L = _lib.lib()
    full = dict(topk_ids=P, topk_weights=P, margins=None, counts=P, offsets=P, perm=P,
                slot_out=None)

    def call(T=200, dt=1, logits=P, ws=WS, nb=1 << 20, r=None, **kw):
        rr = _lib.HfMoeRouting(*{**full, **(r or {})}.values())
        return L.hf_route_logits(logits, dt, None, T, spec(**kw), rr, ws, nb, None)

    bad = [dict(num_experts=0), dict(num_experts=1025), dict(top_k=0), dict(top_k=33),
           dict(num_experts=4, top_k=5), dict(score=2), dict(n_group=3), dict(n_group=0),
           dict(n_group=64), dict(n_group=4, topk_group=5), dict(n_group=4, topk_group=0),
           dict(n_group=16, topk_group=1, top_k=5), dict(group_top=0), dict(group_top=3),
           dict(T=-1), dict(T=1 << 28), dict(dt=7), dict(logits=None), dict(ws=None),
           dict(ws=WS + 16), dict(nb=64), dict(r=dict(perm=None)), dict(r=dict(counts=None)),
           dict(r=dict(margins=P)), dict(r=dict(slot_out=P)), dict(r=dict(topk_ids=None))]
    for b in bad:
        assert call(**b) == _lib.HF_ERR_ARG, b
        assert L.hf_last_error(), b
    assert L.hf_route_logits(P, 1, None, 4, None, None, None, 0, None) == _lib.HF_ERR_ARG
    assert L.hf_route_logits(P, 1, None, 4, spec(), None, None, 0, None) == _lib.HF_ERR_ARG
    assert L.hf_route_workspace_size(16, spec()) == 0
    assert L.hf_route_workspace_size(17, spec()) > 0
    assert L.hf_route_workspace_size(17, spec(top_k=0)) == 0


def test_quantize_refusals():
    L = _lib.lib()
    ok = dict(x=P, dt=0, ldx=64, T=4, K=64, q=P, s=P, st=None)

    def call(**kw):
        return L.hf_fp8_quantize(*{**ok, **kw}.values())

    for b in (dict(T=-1), dict(K=0), dict(K=72), dict(dt=5), dict(x=None), dict(q=None),
              dict(s=None), dict(x=P + 8), dict(q=P + 8), dict(ldx=48), dict(ldx=68),
              dict(dt=1, ldx=66)):
        assert call(**b) == _lib.HF_ERR_ARG, b
    assert call(T=0) == _lib.HF_OK


def test_gemm_refusals():
    L = _lib.lib()
    need = L.hf_fp8_gemm_workspace_size(4, 100, 64)
    assert need > 0 and L.hf_fp8_gemm_workspace_size(0, 100, 64) == 0
    ok = dict(xq=P, sx=P, wq=P, sw=P, T=4, N=100, K=64, out=P, dt=0, ws=WS, nb=need, st=None)

    def call(**kw):
        return L.hf_fp8_gemm(*{**ok, **kw}.values())

    for b in (dict(T=-1), dict(N=0), dict(K=0), dict(K=72), dict(dt=9), dict(xq=None),
              dict(sx=None), dict(wq=None), dict(sw=None), dict(out=None), dict(ws=None),
              dict(xq=P + 8), dict(wq=P + 4), dict(ws=WS + 16), dict(nb=need - 1)):
        assert call(**b) == _lib.HF_ERR_ARG, b
    assert call(T=0) == _lib.HF_OK
    assert L.hf_fp8_status(None, None) == _lib.HF_ERR_ARG


def test_experts_refusals():
    L = _lib.lib()
    T, k, E, H, I = 4, 2, 8, 256, 128
    need = L.hf_fp8_moe_experts_workspace_size(T, k, E, H, I, 0)
    assert need > 0 and L.hf_fp8_moe_experts_workspace_size(0, k, E, H, I, 0) == 0
    assert L.hf_fp8_moe_experts_workspace_size(T, k, E, H, I, 1) > need
    r = _lib.HfMoeRouting(None, P, None, None, P, P, None)
    ok = dict(w=P, s=P, E=E, H=H, I=I, x=P, xt=0, ldx=H, T=T, k=k, r=r, resid=None, out=2 * P,
              ot=0, ws=WS, nb=need, st=None)

    def call(**kw):
        return L.hf_fp8_moe_experts(*{**ok, **kw}.values())

    for b in (dict(E=0), dict(E=1025), dict(H=0), dict(H=248), dict(I=0), dict(I=120), dict(T=-1),
              dict(k=0), dict(k=33), dict(T=1 << 30, k=4), dict(E=1024, H=1 << 20), dict(xt=4), dict(ot=4), dict(w=None),
              dict(s=None), dict(x=None), dict(out=None), dict(ws=None), dict(r=None),
              dict(r=_lib.HfMoeRouting(None, None, None, None, P, P, None)),
              dict(r=_lib.HfMoeRouting(None, P, None, None, None, P, None)),
              dict(r=_lib.HfMoeRouting(None, P, None, None, P, None, None)),
              dict(x=P + 8), dict(ldx=H - 16), dict(ldx=H + 4), dict(w=P + 8), dict(out=P + 8),
              dict(resid=P + 8), dict(resid=2 * P + 64), dict(ws=WS + 128), dict(nb=need - 1)):
        assert call(**b) == _lib.HF_ERR_ARG, b
    assert call(T=0) == _lib.HF_OK


def test_python_refusals():
    from hummingflight_b200 import fp8, moe
    f32, u8 = torch.float32, torch.uint8
    l = torch.zeros((4, 16))
    with pytest.raises(ValueError):
        moe.route_logits(l, None, 4)                       # not on a GPU
    with pytest.raises(ValueError):
        moe.route_logits(l.double(), None, 4)              # type
    with pytest.raises(ValueError):
        moe.route_logits(l.t().contiguous().t(), None, 4)  # order
    with pytest.raises(ValueError):
        moe.route_logits(l, torch.zeros(15), 4)
    with pytest.raises(ValueError):
        moe.route_logits(l, None, 4, "tanh")
    x = torch.zeros((4, 256), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        fp8.quantize(x.half())
    with pytest.raises(ValueError):
        fp8.quantize(x.t())
    with pytest.raises(ValueError):
        fp8.quantize(x)
    q, s = torch.zeros((4, 256), dtype=u8), torch.zeros((4, 2))
    w, ws = torch.zeros((130, 256), dtype=u8), torch.zeros((2, 2))
    for bad in ((q, s[:, :1], w, ws), (q, s, w[:, :128], ws), (q, s, w, ws[:1]),
                (q.float(), s, w, ws), (q, s.double(), w, ws), (q[:, ::2], s, w, ws)):
        with pytest.raises(ValueError):
            fp8.gemm(*bad)
    E, I = 3, 128
    ex, es = torch.zeros((E, 3 * I * 256), dtype=u8), torch.zeros((E, 6))
    r = dict(topk_weights=torch.zeros((4, 2)), offsets=torch.zeros(E + 2, dtype=torch.int32),
             perm=torch.zeros(8, dtype=torch.int32))
    for kw in (dict(experts=ex[:, :-1]), dict(scales=es[:, :5]), dict(resid=x.float()),
               dict(routing={**r, "perm": r["perm"][:7]}),
               dict(routing={**r, "offsets": r["offsets"][:3]}),
               dict(routing={**r, "topk_weights": torch.zeros((3, 2))}),
               dict(routing={**r, "perm": r["perm"].long()})):
        with pytest.raises(ValueError):
            fp8.moe_experts(**{**dict(x=x, experts=ex, scales=es, routing=r), **kw})
    with pytest.raises(ValueError):
        moe.scratch(torch.zeros(4, dtype=u8), 8, torch.device("cpu"))
    assert f32 is torch.float32


def test_calls_run_on_the_device_of_their_tensors(monkeypatch):
    """A call on another device's tensors makes that device current, uses its
    current stream and goes back, also when the call raises."""
    from hummingflight_b200 import moe
    cur, log = [0], []

    class Stream:
        def __init__(self, n):
            self.cuda_stream = n

    monkeypatch.setattr(moe, "_get_device", lambda: cur[0])
    monkeypatch.setattr(moe, "_set_device", lambda d: (log.append(d), cur.__setitem__(0, d)))
    monkeypatch.setattr(moe, "_raw_stream", lambda i: 100 + i)
    with moe.on_device(torch.device("cuda", 1)) as s:
        assert s == 101 and cur[0] == 1
    assert cur[0] == 0 and log == [1, 0]
    with pytest.raises(KeyError):
        with moe.on_device(torch.device("cuda", 2), Stream(7)) as s:
            assert s == 7 and cur[0] == 2
            raise KeyError
    assert cur[0] == 0
    with moe.on_device(torch.device("cuda", 0)) as s:
        assert s == 100
    assert log == [1, 0, 2, 0]


def test_sizes_next_to_2_31_are_refused():
    """Rounded up to tiles, these would pass 32 bits."""
    L = _lib.lib()
    big, ws = 0x7fffffff - 15, 1 << 62
    r = _lib.HfMoeRouting(P, P, None, P, P, P, None)
    assert L.hf_route_logits(P, 1, None, big, spec(num_experts=1, top_k=1), r, WS, ws,
                             None) == _lib.HF_ERR_ARG
    assert L.hf_route_workspace_size(big, spec(num_experts=1, top_k=1)) == 0
    assert L.hf_fp8_quantize(P, 0, big, 1, big, P, P, None) == _lib.HF_ERR_ARG
    assert L.hf_fp8_quantize(P, 0, 16, big, 16, P, P, None) == _lib.HF_ERR_ARG
    for T, N, K in ((big, 16, 16), (16, big, 16), (16, 16, big)):
        assert L.hf_fp8_gemm_workspace_size(T, N, K) == 0
        assert L.hf_fp8_gemm(P, P, P, P, T, N, K, P, 0, WS, ws, None) == _lib.HF_ERR_ARG
    for T, k, E, H, I in ((big, 1, 1, 16, 16), (big // 4, 4, 1, 16, 16), (1, 1, 1, 715827872, 16),
                          (1, 1, 1, 16, 715827872)):
        assert L.hf_fp8_moe_experts_workspace_size(T, k, E, H, I, 0) == 0
        assert L.hf_fp8_moe_experts(P, P, E, H, I, P, 0, H, T, k, r, None, P, 0, WS, ws,
                                    None) == _lib.HF_ERR_ARG


def test_status_asks_the_device_of_the_workspace(monkeypatch):
    from hummingflight_b200 import fp8, moe
    cur, seen = [0], []

    class Workspace:
        device = torch.device("cuda", 1)

        def data_ptr(self):
            return P

    monkeypatch.setattr(moe, "_get_device", lambda: cur[0])
    monkeypatch.setattr(moe, "_set_device", lambda d: cur.__setitem__(0, d))
    monkeypatch.setattr(moe, "_raw_stream", lambda i: 100 + i)
    monkeypatch.setattr(fp8, "call", lambda *a: seen.append((cur[0], *a)))
    fp8.status(Workspace())
    assert seen == [(1, "hf_fp8_status", P, 101)] and cur[0] == 0
