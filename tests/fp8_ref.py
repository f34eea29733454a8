"""64-bit plain forms of the routing and FP8 operators (numpy / torch doubles on
the CPU) and the error bounds their tests use."""
import math

import numpy as np
import torch

BLOCK = 128
U = 2.0 ** -24  # half a step of fp32


def blocks(n):
    return -(-n // BLOCK)


# ------------------------------------------------------------------ routing
def route(logits, bias, k, score, n_group, topk_group, group_top, scale, norm):
    """ids, weights, counts [E+1], offsets [E+2], perm; logits double [T x E]."""
    T, E = logits.shape
    with np.errstate(all="ignore"):
        if score == "sigmoid":
            p = 1 / (1 + np.exp(-logits))
        else:
            m = np.fmax.reduce(logits, axis=1, keepdims=True)
            e = np.where(logits == -np.inf, 0.0, np.exp(logits - m))
            s = e.sum(1, keepdims=True)
            p = np.where(s == 0, 0.0, e / np.where(s == 0, 1, s))
        key = p if bias is None else p + bias
        rank_key = logits if bias is None else key
        gs = E // n_group
        ids = np.empty((T, k), np.int64)
        w = np.empty((T, k))
        low = lambda v: (1, 0.0) if math.isnan(v) else (0, -v)  # noqa: E731  best first, NaN last
        for t in range(T):
            allowed = range(E)
            if topk_group < n_group:
                gsc = []
                for g in range(n_group):
                    best = sorted(key[t, g * gs:(g + 1) * gs], key=low)[:group_top]
                    gsc.append(sum(best))
                kept = sorted(range(n_group), key=lambda g: (low(gsc[g]), g))[:topk_group]
                allowed = [e for e in range(E) if e // gs in kept]
            ids[t] = sorted(allowed, key=lambda e: (low(rank_key[t, e]), e))[:k]
            w[t] = p[t, ids[t]]
            if norm and not w[t].sum() <= 0:
                w[t] = w[t] / w[t].sum()
        flat = ids.reshape(-1)
        perm = np.argsort(flat, kind="stable")
        counts = np.bincount(flat, minlength=E + 1)
        return ids, w * scale, counts, np.concatenate([[0], np.cumsum(counts)]), perm


# ------------------------------------------------------------------ e4m3
def e4m3(v):
    """Nearest e4m3 value of doubles |v| <= 448 (ties to even); NaN stays."""
    e = np.frexp(v)[1].clip(min=-5)
    step = np.ldexp(1.0, e - 4)
    return np.rint(v / step) * step


def scale_of(top):
    """Smallest power of two s with top <= 448 s; 1 for 0, NaN for Inf and NaN."""
    m, e = np.frexp(np.where(np.isfinite(top), top, 1.0))
    j = np.where(m > 0.875, e - 8, e - 9).clip(min=-126)
    s = np.where(top == 0, 1.0, np.ldexp(1.0, j))
    return np.where(np.isfinite(top), s, np.nan)


def quantize(x):
    """q (as values) [T x K] and scales [T x blocks] of doubles x."""
    T, K = x.shape
    nb = blocks(K)
    v = np.zeros((T, nb * BLOCK))
    v[:, :K] = x
    v = v.reshape(T, nb, BLOCK)
    top = np.abs(v).max(2) if T else np.zeros((0, nb))
    s = scale_of(top)
    with np.errstate(invalid="ignore"):
        q = e4m3(v / s[:, :, None]).reshape(T, nb * BLOCK)[:, :K]
    return q, s


def bits(v):
    """e4m3 bits (uint8 tensor) of e4m3 values."""
    return torch.from_numpy(np.ascontiguousarray(v)).to(torch.float8_e4m3fn).view(torch.uint8)


def values(q, s, rows, cols, weight=False):
    """Doubles that e4m3 values and their scales stand for."""
    if weight:
        s = np.repeat(s, BLOCK, 0)[:rows]
    return q.reshape(rows, cols) * np.repeat(s, BLOCK, 1)[:, :cols]


def weight(rng, n, k, sigma=0.02):
    """Seeded e4m3 weight values [n x k] and fp32 block scales (as doubles)."""
    q = e4m3((rng.standard_normal((n, k)) * 106).clip(-448, 448))
    s = (sigma / 106 * rng.uniform(0.8, 1.2, (blocks(n), blocks(k)))).astype(np.float32)
    return q, s.astype(np.float64)


def product(x, w):
    """x w^T and the bound on its fp32 evaluation: per output, products are
    exact, a block's 128 products are added in any order (tensor cores may cut
    instead of round: 2 half steps per addition), a block's sum takes the
    rounding of the two scales' product and one fused multiply-add."""
    kb = blocks(x.shape[1])
    return x @ w.T, (2 * (BLOCK + 2) + 2 * kb) * U * (np.abs(x) @ np.abs(w).T)


def rounding(y, bf16):
    """Half a step of the output type at y."""
    return np.abs(y) * (2.0 ** -8 if bf16 else U)


def silu_mul(g, eg, u, eu):
    """silu(g) * u and its bound from the bounds on g and u: |silu'| <= 1.1,
    |silu(g)| <= |g|; the fast exponential (2 + 1.2 |g| steps of 2^-23) and
    quotient."""
    m = g / (1 + np.exp(-g)) * u
    return m, 1.1 * eg * (np.abs(u) + eu) + np.abs(g) * eu + (8 + 2.4 * np.abs(g)) * U * np.abs(m)


def quantize_interval(m, em):
    """quantize(m) as values, and how far the quantised values of anything within
    em of m can be from them: the values at both ends, under the scales that both
    ends' maxima give (rounding is monotone)."""
    T, K = m.shape
    q0, s0 = quantize(m)
    mid = values(q0, s0, T, K)
    far = np.zeros_like(mid)
    nb = blocks(K)
    pad = np.zeros((T, nb * BLOCK))
    pe = np.zeros((T, nb * BLOCK))
    pad[:, :K], pe[:, :K] = m, em
    a = np.abs(pad).reshape(T, nb, BLOCK)
    e = pe.reshape(T, nb, BLOCK)
    for top in ((a + e).max(2), np.maximum(a - e, 0).max(2)):
        s = np.repeat(scale_of(top), BLOCK, 1)[:, :K]
        for end in (m - em, m + em):
            far = np.maximum(far, np.abs(e4m3((end / s).clip(-448, 448)) * s - mid))
    return mid, far


def experts(x, gate_up_down, ids, w, I, resid=None, bf16=True, slot_bf16=True):
    """The experts' output and its bound. x: doubles [T x H] as stored;
    gate_up_down: per expert three weights as doubles; ids, w [T x k]."""
    T, H = x.shape
    k = ids.shape[1]
    xv = values(*quantize(x), T, H)
    out = np.zeros((T, H))
    err = np.zeros((T, H))
    mag = np.zeros((T, H))
    for e in np.unique(ids):
        t, i = np.nonzero(ids == e)
        wg, wu, wd = gate_up_down[e]
        g, eg = product(xv[t], wg)
        u, eu = product(xv[t], wu)
        m, em = silu_mul(g, eg, u, eu)
        mv, far = quantize_interval(m, em)
        y, ey = product(mv, wd)
        ey = ey * 1.01 + far @ np.abs(wd).T  # 1.01: the bound of the moved values
        ey = ey + rounding(y, slot_bf16)
        wt = w[t, i][:, None]
        np.add.at(out, t, y * wt)
        np.add.at(err, t, ey * np.abs(wt))
        np.add.at(mag, t, np.abs(y * wt))
    if resid is not None:
        out = out + resid
        mag = mag + np.abs(resid)
    err = err + 2 * (k + 2) * U * mag
    return out, err + rounding(out, bf16) * 1.01
