"""Arguments of the wrong rank, and rows of no columns, are refused as ValueError."""
import pytest

torch = pytest.importorskip("torch")


def test_ranks_and_empty_rows():
    from hummingflight_b200 import fp8
    u8, i32 = torch.uint8, torch.int32
    x = torch.zeros((4, 256), dtype=torch.bfloat16)
    q, s, w, ws = (torch.zeros(v, dtype=d) for v, d in (((4, 256), u8), ((4, 2), torch.float32),
                                                        ((128, 256), u8), ((1, 2), torch.float32)))
    for bad in ((q[0], s, w, ws), (q, s[0], w, ws), (q, s, w[0], ws), (q, s, w.view(-1)[0], ws),
                (q, s, w, ws[0])):
        with pytest.raises(ValueError):
            fp8.gemm(*bad)
    with pytest.raises(ValueError):
        fp8.quantize(x[0])
    ex, es = torch.zeros((3, 3 * 128 * 256), dtype=u8), torch.zeros((3, 6))
    r = dict(topk_weights=torch.zeros((4, 2)), offsets=torch.zeros(5, dtype=i32),
             perm=torch.zeros(8, dtype=i32))
    ok = dict(x=x, experts=ex, scales=es, routing=r)
    for kw in (dict(x=x[0]), dict(x=x[:, :0]), dict(experts=ex[0]), dict(experts=ex[:, :0]),
               dict(scales=es[0]), dict(routing={**r, "topk_weights": torch.zeros(4)})):
        with pytest.raises(ValueError):
            fp8.moe_experts(**{**ok, **kw})
