"""hf_route_logits where keys or group scores differ by a few units of 64-bit
arithmetic or not at all. A sigmoid of 0 is 1/2 exactly, so with biases that are
multiples of u = 2^-53 (the step of doubles below 1) every key is exact and the
expected choice does not hang on anyone's exponential."""
import numpy as np
import pytest

import fp8_ref as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
U = 2.0 ** -53


def check(logits, bias, k, n_group=1, topk_group=1, group_top=2):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from hummingflight_b200 import moe
    b = None if bias is None else torch.from_numpy(bias).float().cuda()
    got = moe.route_logits(torch.from_numpy(logits).float().cuda(), b, k, "sigmoid", n_group,
                           topk_group, group_top)
    ids, _, counts, _, perm = R.route(logits, bias, k, "sigmoid", n_group, topk_group, group_top,
                                      1.0, True)
    assert np.array_equal(got["topk_ids"].cpu().numpy(), ids)
    assert np.array_equal(got["counts"].cpu().numpy(), counts)
    assert np.array_equal(got["perm"].cpu().numpy(), perm)


@pytest.mark.parametrize("E,n_group", [(32, 2), (64, 4), (100, 4), (256, 8), (512, 16), (1024, 32)])
@pytest.mark.parametrize("swap", [False, True])
def test_groups_of_equal_sums(E, n_group, swap):
    """1/2 + 2u and 1/2 + 6u in one group, 1/2 + 8u and 1/2 in another: the scores are
    the same double, and the lower group is kept."""
    gs = E // n_group
    l, b = np.full((3, E), -100.0), np.zeros(E)
    one, two = (gs * (n_group - 1), 0) if swap else (0, gs * (n_group - 1))
    for at, units in ((one, (6, 2)), (two, (0, 8))):
        for i, v in zip((1, gs - 1), units):
            l[:, at + i], b[at + i] = 0.0, v * U
    check(l, b, 2, n_group, 1)


@pytest.mark.parametrize("E,groups", [(40, (1, 1)), (64, (1, 1)), (256, (1, 1)), (1000, (1, 1)),
                                      (64, (4, 2)), (256, (8, 3)), (512, (16, 5))])
def test_keys_a_few_units_apart(E, groups):
    """Up to all of the experts within fp32 rounding of each other; per token other ones
    are out of the choice."""
    rng = np.random.default_rng(E)
    b = rng.permutation(E).astype(float) * U
    l = np.where(rng.random((37, E)) < 0.3, -100.0, 0.0)
    l[:3] = 0.0
    check(l, b, min(8, E // 8), *groups)
    check(l, b, min(8, E // 8), *groups, 1)
    check(l, np.zeros(E), min(8, E // 8), *groups)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,n_group,group_top", [(64, 8, 1), (300, 10, 1), (512, 32, 1), (32, 32, 2),
                                                 (8, 8, 2)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_groups_without_a_bias_rank_by_logit(score, E, n_group, group_top, dtype):
    """One key a group: their order is that of the largest logits, also where every
    score is the same number (1, or a softmax of 0), far apart and one step apart."""
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from hummingflight_b200 import moe
    rng = np.random.default_rng(E)
    keep, k = n_group // 2, min(8, E // n_group * (n_group // 2))
    t = torch.float32 if dtype == "f32" else torch.bfloat16
    for base, step in ((100.0, 2.0 ** -17), (40.0, 0.5), (100.0, 1.0), (-1000.0, 2.0 ** -14),
                       (-1000.0, 8.0)):
        l = base + step * rng.integers(0, E, (29, E))
        if score == "softmax" and base < 0:
            l[:, 0] = 0.0
        l = torch.from_numpy(l).to(t)
        d = l.double().numpy()
        top = d.reshape(29, n_group, -1).max(2)
        ids = np.empty((29, k), np.int64)
        for i in range(29):
            kept = sorted(range(n_group), key=lambda g: (-top[i, g], g))[:keep]
            ids[i] = sorted((e for e in range(E) if e // (E // n_group) in kept),
                            key=lambda e: (-d[i, e], e))[:k]
        got = moe.route_logits(l.cuda(), None, k, score, n_group, keep, group_top)
        assert np.array_equal(got["topk_ids"].cpu().numpy(), ids)
