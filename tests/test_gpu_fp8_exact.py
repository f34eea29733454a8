"""The routed FP8 experts on inputs whose products and sums are exact in fp32: what
is left is silu's rounding, which the inputs keep away from every border of the
quantised intermediate, and the roundings that the operator states. (On random inputs
an intermediate near a border may go either way, and the bound has to allow for it.)"""
import numpy as np
import pytest

import fp8_ref as R

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu


def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def inputs(seed, T, E, k, H, I, shift=0):
    """Tokens, expert weights (values, scales as floats), routing and the outputs y of
    every pick. g is 2..5 and u is 1, 2 or 4 in magnitude, from three columns in
    different blocks of K; the other columns cancel in pairs. shift: of the exponent
    of the down weights' scales."""
    rng = np.random.default_rng(seed)
    ca, cb, cu = 0, H // 2, H - 1
    pairs = rng.permutation([c for c in range(H) if c not in (ca, cb, cu)])
    p, q = pairs[:len(pairs) // 2], pairs[len(pairs) // 2:len(pairs) // 2 * 2]
    x = np.zeros((T, H))
    x[:, p] = x[:, q] = rng.integers(-2, 3, (T, len(p)))
    x[:, ca], x[:, cb] = 1, rng.integers(0, 2, T)
    x[:, cu] = rng.choice([-2, -1, 1, 2], T)
    blocks = []
    for _ in range(E):
        gate, upw = np.zeros((I, H)), np.zeros((I, H))
        gate[:, ca], gate[:, cb] = rng.integers(2, 4, I), rng.integers(0, 3, I)
        upw[:, cu] = rng.integers(1, 3, I)
        for w in (gate, upw):
            w[:, p] = rng.integers(-3, 4, (I, len(p)))
            w[:, q] = -w[:, p]
        down = rng.integers(-3, 4, (H, I)).astype(float)
        parts = []
        for w, e in ((gate, 0), (upw, 0), (down, shift)):
            # scales 2^-3 and 2^-2, the stored values larger by as much
            s = np.exp2(rng.integers(-3, -1, (R.blocks(w.shape[0]), R.blocks(w.shape[1]))))
            full = np.repeat(np.repeat(s, 128, 0), 128, 1)[:w.shape[0], :w.shape[1]]
            parts.append((w / full, s * 2.0 ** e, w * 2.0 ** e))
        blocks.append(parts)
    ids = np.stack([rng.permutation(E)[:k] for _ in range(T)])
    w = np.array([0.75, 0.5, 0.25, 1.25])[rng.integers(0, 4, (T, k))]
    y = np.zeros((T, k, H))
    for e in range(E):
        t, i = np.nonzero(ids == e)
        if not len(t):
            continue
        g, u = x[t] @ blocks[e][0][2].T, x[t] @ blocks[e][1][2].T
        m, em = R.silu_mul(g, 0.0, u, 0.0)
        mv, far = R.quantize_interval(m, em)
        assert far.max() == 0  # no intermediate near a border
        y[t, i] = mv @ blocks[e][2][2].T
        # multiples of 2^-4, so that 24 bits hold every sum of them, of any order
        assert (mv % 2.0 ** -4 == 0).all()
        assert (np.abs(mv) @ np.abs(blocks[e][2][2].T)).max() < 2.0 ** (24 - 4 + shift)
    # and the weighted sum: multiples of 2^-6
    assert (np.abs(y) * w[:, :, None]).sum(1).max() < 2.0 ** (24 - 6 + shift)
    flat = ids.reshape(-1)
    counts = np.bincount(flat, minlength=E)
    routing = dict(topk_weights=w, offsets=np.concatenate([[0], np.cumsum(counts)]),
                   perm=np.argsort(flat, kind="stable"))
    return x, blocks, routing, y


def to_gpu(x, blocks, routing):
    q = torch.stack([torch.cat([R.bits(v).view(-1) for v, _, _ in b]) for b in blocks]).cuda()
    s = np.stack([np.concatenate([v.reshape(-1) for _, v, _ in b]) for b in blocks])
    r = dict(topk_weights=torch.from_numpy(routing["topk_weights"]).float().cuda(),
             offsets=torch.from_numpy(routing["offsets"]).int().cuda(),
             perm=torch.from_numpy(routing["perm"]).int().cuda())
    return (torch.from_numpy(x).bfloat16().cuda(), q,
            torch.from_numpy(s).float().cuda(), r)


SIZES = [  # T, E, k, H, I: one token, runs of K, tiles of 32 and 64 positions, CTA pairs
    (1, 2, 1, 144, 128), (1, 2, 2, 272, 2048), (20, 3, 2, 2048, 384), (40, 4, 2, 400, 272),
    (300, 16, 2, 528, 256), (120, 4, 2, 656, 256), (700, 8, 2, 400, 128), (300, 2, 2, 640, 400),
    (600, 4, 4, 272, 256)]


def test_inputs_are_exact():
    for i, size in enumerate(SIZES):
        inputs(i, *size)


@gpu
@pytest.mark.parametrize("i", range(len(SIZES)))
def test_fp32_outputs_are_exact(i):
    need_gpu()
    from hummingflight_b200 import fp8
    T, E, k, H, I = SIZES[i]
    x, blocks, routing, y = inputs(i, T, E, k, H, I)
    ref = (y * routing["topk_weights"][:, :, None]).sum(1)
    resid = np.random.default_rng(i).integers(-9, 10, (T, H)).astype(float)
    xg, q, s, r = to_gpu(x, blocks, routing)
    out = fp8.moe_experts(xg, q, s, r, torch.from_numpy(resid).float().cuda(), out_dtype="f32")
    assert np.array_equal(out.double().cpu().numpy(), ref + resid)


@gpu
@pytest.mark.parametrize("shift", [0, 80, -100])
@pytest.mark.parametrize("i", range(len(SIZES)))
def test_bf16_outputs_are_rounded_once(i, shift):
    """The residual takes nearly all of the sum away, so that what the expert outputs
    lost before the sum shows: less than a step of 16 significant bits each, or half a
    step of FP16 where there are many positions, then half a step of bf16 of what is left
    (2 (k + 2) half steps of fp32 for the sum)."""
    need_gpu()
    from hummingflight_b200 import fp8
    T, E, k, H, I = SIZES[i]
    x, blocks, routing, y = inputs(i, T, E, k, H, I, shift)
    wy = y * routing["topk_weights"][:, :, None]
    resid = torch.from_numpy(-wy.sum(1)).bfloat16()
    ref = wy.sum(1) + resid.double().numpy()
    xg, q, s, r = to_gpu(x, blocks, routing)
    out = fp8.moe_experts(xg, q, s, r, resid.cuda()).double().cpu().numpy()
    lost = np.abs(wy).sum(1)
    tol = (2.0 ** (-15 if T * k <= 96 * E else -11) + 2 * (k + 2) * R.U) * lost
    assert (np.abs(out - ref) <= tol + 2.0 ** -8 * (np.abs(ref) + tol)).all()


@gpu
@pytest.mark.parametrize("i", [3, 5, 7])
def test_non_finite_output_columns_stay_apart(i):
    """A NaN in one row of an expert's down weights: that column of its tokens, none
    beside it."""
    need_gpu()
    from hummingflight_b200 import fp8
    T, E, k, H, I = SIZES[i]
    x, blocks, routing, _ = inputs(i, T, E, k, H, I)
    xg, q, s, r = to_gpu(x, blocks, routing)
    good = fp8.moe_experts(xg, q, s, r).clone()
    row = 37
    q[0, 2 * I * H + row * I + 5] = 0x7f
    bad = fp8.moe_experts(xg, q, s, r)
    perm, off = routing["perm"], routing["offsets"]
    hit = np.zeros(T, bool)
    hit[perm[off[0]:off[1]] // k] = True
    hit = torch.from_numpy(hit).cuda()
    assert bad[hit, row].isnan().all()
    bad[hit, row] = good[hit, row]
    assert torch.equal(bad, good)
