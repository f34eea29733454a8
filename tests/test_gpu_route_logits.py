"""hf_route_logits against the 64-bit plain form: ids, counts, offsets and the
permutation equal, weights within the derived rounding of the fp32 scores."""
import numpy as np
import pytest

import fp8_ref as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def doubles(t):
    return t.float().cpu().numpy().astype(np.float64)


def check(logits, bias, k, score, n_group=1, topk_group=1, group_top=2, scale=1.0, norm=True,
          got=None):
    from hummingflight_b200 import moe
    if got is None:
        got = moe.route_logits(logits, bias, k, score, n_group, topk_group, group_top, scale, norm)
    l = doubles(logits)
    ids, w, counts, offsets, perm = R.route(l, None if bias is None else doubles(bias), k, score,
                                            n_group, topk_group, group_top, scale, norm)
    g = {n: v.cpu().numpy() for n, v in got.items()}
    assert np.array_equal(g["topk_ids"], ids)
    assert np.array_equal(g["counts"], counts)
    assert np.array_equal(g["offsets"], offsets)
    assert np.array_equal(g["perm"], perm)
    # scores: the exponent's rounding (|l - m| half steps), a sum of E terms, expf
    # and the divisions; the sum of k picks and its division
    fin = l[np.isfinite(l)]
    spread = (fin.max() - fin.min()) if fin.size else 0.0
    tol = (spread + 100 + 2 * k) * R.U
    gw = g["topk_weights"].astype(np.float64)
    assert np.array_equal(np.isnan(gw), np.isnan(w))
    ok = ~np.isnan(w)
    assert (np.abs(gw - w)[ok] <= tol * np.abs(w[ok]) + 1e-37).all()


CASES = [  # T, E, k, score, bias, n_group, topk_group, group_top, norm, dtype
    (1, 256, 8, "sigmoid", True, 1, 1, 2, True, "f32"),
    (1, 1, 1, "softmax", False, 1, 1, 1, False, "f32"),
    (2, 7, 7, "softmax", True, 1, 1, 2, True, "bf16"),
    (31, 33, 5, "sigmoid", False, 1, 1, 2, False, "f32"),
    (33, 32, 32, "sigmoid", True, 1, 1, 2, True, "f32"),
    (64, 256, 8, "sigmoid", True, 8, 4, 2, True, "f32"),
    (128, 160, 6, "softmax", False, 8, 3, 1, False, "bf16"),
    (129, 64, 6, "softmax", False, 4, 2, 2, True, "f32"),
    (257, 300, 9, "softmax", True, 10, 3, 2, True, "f32"),
    (200, 1024, 32, "sigmoid", True, 32, 5, 1, False, "f32"),
    (63, 512, 10, "softmax", False, 1, 1, 2, True, "f32"),
    (50, 96, 3, "sigmoid", True, 32, 32, 2, True, "f32"),
    (77, 32, 4, "softmax", True, 32, 6, 2, False, "f32"),
    (1999, 160, 6, "softmax", False, 1, 1, 1, False, "bf16"),
]


@pytest.mark.parametrize("T,E,k,score,bias,ng,tg,gt,norm,dtype", CASES)
def test_matches_plain_form(T, E, k, score, bias, ng, tg, gt, norm, dtype):
    need_gpu()
    g = torch.Generator().manual_seed(T * 1000 + E)
    l = (torch.randn((T, E), generator=g) * 1.7).to(
        torch.float32 if dtype == "f32" else torch.bfloat16).cuda()
    b = (torch.rand(E, generator=g) * 0.2 - 0.1).cuda() if bias else None
    check(l, b, k, score, ng, tg, gt, 2.5, norm)


@pytest.mark.parametrize("T,E", [(1190, 40), (9473, 8), (70000, 8), (270000, 3)])
def test_long_batches(T, E):
    """Blocks of 16, 72, 480 and 512 tokens, the last so many that their counts are scanned."""
    need_gpu()
    g = torch.Generator().manual_seed(T)
    check(torch.randn((T, E), generator=g).cuda(), None, 2, "softmax")


def test_empty_batch():
    need_gpu()
    from hummingflight_b200 import moe
    r = moe.route_logits(torch.empty((0, 16), device="cuda"), None, 4)
    assert r["counts"].tolist() == [0] * 17 and r["offsets"].tolist() == [0] * 18


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("groups", [(1, 1, 2), (4, 2, 2), (4, 2, 1)])
def test_ties_go_to_the_lowest_id(score, groups):
    """Logits and biases on a coarse grid: most keys (and group scores) tie."""
    need_gpu()
    g = torch.Generator().manual_seed(5)
    l = torch.randint(-2, 3, (150, 64), generator=g).float().cuda()
    b = (torch.randint(0, 2, (64,), generator=g).float() * 0.25).cuda()
    check(l, None, 6, score, *groups)
    check(l, b, 6, score, *groups)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_near_ties_rank_as_in_64_bits(score):
    """Expert 2j + 1's bias lifts its key onto expert 2j's up to fp32 rounding: on
    fp32 keys about half of the pairs would come out the other way or tied."""
    need_gpu()
    g = torch.Generator().manual_seed(6)
    T, E = 96, 64
    row = torch.randn(E, generator=g)
    l = row.repeat(T, 1) + 2.0 ** -22 * torch.randint(-3, 4, (T, E), generator=g)
    d = row.double()
    p = torch.sigmoid(d) if score == "sigmoid" else torch.softmax(d, 0)
    b = torch.zeros(E)
    b[1::2] = (p[0::2] - p[1::2]).float()
    check(l.cuda(), b.cuda(), 12, score)
    check(l.cuda(), b.cuda(), 12, score, 8, 4, 2)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups", [(1, 1, 2), (4, 2, 2)])
def test_masked_and_non_finite_logits(score, biased, groups):
    need_gpu()
    g = torch.Generator().manual_seed(7)
    E = 40
    l = torch.randn((140, E), generator=g)
    inf, low = float("inf"), torch.finfo(torch.float32).min
    l[0] = -inf                    # nothing left
    l[1, 5:] = -inf                # fewer experts left than picks
    l[2, ::2] = low
    l[3, :] = low
    l[4, 7] = low
    l[5, 1:] = -inf
    b = (torch.rand(E, generator=g) * 0.2 - 0.1) if biased else None
    check(l.cuda(), b.cuda() if biased else None, 8, score, *groups, 1.0, True)
    if biased:                     # experts switched off by their bias
        b[3], b[4], b[30] = -inf, low, -inf
        check(l.cuda(), b.cuda(), 8, score, *groups, 1.0, True)


def test_scores_near_the_smallest_numbers_rank_as_in_64_bits():
    """Biases of the size of the scores, 1e-39 and below: a quotient flushed to 0
    must not count as exact."""
    need_gpu()
    l = torch.full((20, 8), -100.0)
    l[:, 3], l[:, 6] = -88.0, -95.0
    b = torch.zeros(8)
    b[3], b[6] = 1e-39, 3e-39
    check(l.cuda(), b.cuda(), 1, "sigmoid", 1, 1, 2, 1.0, False)
    check(l.cuda(), b.cuda(), 4, "sigmoid", 1, 1, 2, 1.0, False)
    check(l.cuda(), b.cuda(), 2, "sigmoid", 4, 2, 2, 1.0, False)


def test_nan_logits():
    """A NaN key ranks below every number; a softmax row with one has NaN weights."""
    need_gpu()
    from hummingflight_b200 import moe
    g = torch.Generator().manual_seed(8)
    l = torch.randn((130, 24), generator=g)
    l[1, 3] = float("nan")
    l[2, :] = float("nan")
    l[3, 4:] = float("nan")
    check(l.cuda(), None, 6, "sigmoid", 1, 1, 2, 1.0, False)
    b = torch.rand(24, generator=g).cuda()
    check(l.cuda(), b, 6, "sigmoid", 1, 1, 2, 1.0, False)
    r = moe.route_logits(l.cuda(), None, 6, "softmax")
    w = r["topk_weights"].cpu()
    assert w[1].isnan().all() and w[2].isnan().all() and not w[0].isnan().any()
    assert r["topk_ids"][2].tolist() == list(range(6))


def test_stream_capture_and_reuse():
    """Captured, replayed on new logits, on a stream of its own; the workspace and
    the outputs keep nothing of the call before."""
    need_gpu()
    from hummingflight_b200 import moe
    T, E, k = 700, 48, 4
    l = torch.randn((T, E), device="cuda")
    b = torch.rand(E, device="cuda") * 0.1
    ws = torch.full((moe.route_workspace_size(T, E, k),), 255, dtype=torch.uint8, device="cuda")
    out = moe.route_logits(l, b, k, workspace=ws)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        moe.route_logits(l, b, k, out=out, workspace=ws)
    for seed in (1, 2):
        l.copy_(torch.randn((T, E), generator=torch.Generator().manual_seed(seed)))
        for v in out.values():
            v.fill_(-7)
        ws.fill_(17)
        graph.replay()
        torch.cuda.synchronize()
        check(l, b, k, "sigmoid", got=out)
    other = moe.route_logits(l, b, k, stream=side)
    side.synchronize()
    check(l, b, k, "sigmoid", got=other)
