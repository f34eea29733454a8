"""Cases of the routing and FP8 operators: inputs, plain forms, the framework's
calls and 64-bit values.

Four operators:

  route    hf_route_logits: router logits [T x E] -> experts, weights and the
           permutation into expert segments
  quant    hf_fp8_quantize: rows -> e4m3 with a power-of-two scale per 128 columns
  gemm     hf_fp8_gemm: rows x weight in e4m3, a scale per 128 (rows) and per
           128 x 128 block (weight)
  experts  hf_fp8_moe_experts: the routed SwiGLU experts over e4m3 weights

Sizes are those of the framework's layer (hidden 6144, 256 experts, top-8,
intermediate 2048, dense intermediate 12288) and its batches (1, 64, 4096 and
16384 tokens), and ragged ones around them.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 128
E4M3 = torch.float8_e4m3fn
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decoded token: latency
        {"name": "route_t1", "op": "route", "T": 1, "E": 256, "k": 8, "score": "sigmoid",
         "bias": True, "n_group": 1, "topk_group": 1, "group_top": 2, "norm": True,
         "scale": 2.5, "dtype": "f32"},
        # a decode batch, experts limited to 4 of 8 groups
        {"name": "route_groups_t64", "op": "route", "T": 64, "E": 256, "k": 8, "score": "sigmoid",
         "bias": True, "n_group": 8, "topk_group": 4, "group_top": 2, "norm": True,
         "scale": 2.5, "dtype": "f32"},
        # a prefill batch with a biased sigmoid router
        {"name": "route_t16384", "op": "route", "T": 16384, "E": 256, "k": 8, "score": "sigmoid",
         "bias": True, "n_group": 1, "topk_group": 1, "group_top": 2, "norm": True,
         "scale": 2.5, "dtype": "f32"},
        # an odd prompt, softmax scores, no bias, bf16 logits (exact ties occur)
        {"name": "route_softmax_t1999", "op": "route", "T": 1999, "E": 160, "k": 6,
         "score": "softmax", "bias": False, "n_group": 1, "topk_group": 1, "group_top": 1,
         "norm": False, "scale": 1.0, "dtype": "bf16"},
        # activations of a decode batch and of a prefill batch
        {"name": "quant_t64", "op": "quant", "T": 64, "K": 6144, "dtype": "bf16"},
        {"name": "quant_t16384", "op": "quant", "T": 16384, "K": 6144, "dtype": "bf16"},
        # a dense layer's up projection for one token
        {"name": "gemm_t1", "op": "gemm", "T": 1, "N": 12288, "K": 6144, "out": "f32"},
        # its down projection for a decode batch
        {"name": "gemm_t64", "op": "gemm", "T": 64, "N": 6144, "K": 12288, "out": "bf16"},
        # its up projection for a prefill batch
        {"name": "gemm_t4096", "op": "gemm", "T": 4096, "N": 12288, "K": 6144, "out": "bf16"},
        # the experts of one layer: a token, a decode batch, a prefill batch
        {"name": "experts_t1", "op": "experts", "T": 1, "E": 256, "k": 8, "H": 6144, "I": 2048,
         "resid": False},
        {"name": "experts_t64", "op": "experts", "T": 64, "E": 256, "k": 8, "H": 6144, "I": 2048,
         "resid": True},
        {"name": "experts_t16384", "op": "experts", "T": 16384, "E": 256, "k": 8, "H": 6144,
         "I": 2048, "resid": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _step(rng, lo, hi, step):
    return step * _log_int(rng, max(1, lo // step), hi // step)


def draw(rng):
    op = rng.choice(["route", "quant", "gemm", "gemm", "experts", "experts"])
    if op == "route":
        n_group = rng.choice([1, 1, 2, 4, 8])
        E = n_group * rng.randint(4, 512 // n_group)
        topk_group = rng.randint(max(1, n_group // 2), n_group)
        return {"op": op, "T": _log_int(rng, 1, 16384), "E": E,
                "k": rng.randint(1, min(16, topk_group * (E // n_group))),
                "score": rng.choice(["sigmoid", "softmax"]), "bias": rng.random() < 0.6,
                "n_group": n_group, "topk_group": topk_group, "group_top": rng.choice([1, 2]),
                "norm": rng.random() < 0.6, "scale": rng.choice([1.0, 2.5]),
                "dtype": rng.choice(["f32", "f32", "bf16"])}
    if op == "quant":
        return {"op": op, "T": _log_int(rng, 1, 16384), "K": _step(rng, 16, 6144, 16),
                "dtype": rng.choice(["bf16", "bf16", "f32"])}
    if op == "gemm":
        return {"op": op, "T": _log_int(rng, 1, 4096), "N": _log_int(rng, 16, 12288),
                "K": _step(rng, 64, 6144, 16), "out": rng.choice(["bf16", "bf16", "f32"])}
    E = rng.choice([4, 8, 16, 33, 64, 128, 256])
    return {"op": op, "T": _log_int(rng, 1, 8192), "E": E, "k": rng.randint(1, min(8, E)),
            "H": _step(rng, 256, 6144, 16), "I": _step(rng, 128, 2048, 16),
            "resid": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs
def _weights(gen, rows, cols):
    """e4m3 weight ~N(0, 0.02) and its fp32 scales, one per 128 x 128 block
    (a block's largest weight sits near the type's largest value)."""
    q = torch.randn((rows, cols), generator=gen, device="cuda").mul_(106.0).clamp_(-448, 448).to(E4M3)
    s = torch.rand((_blocks(rows), _blocks(cols)), generator=gen, device="cuda")
    return q, (0.02 / 106.0) * (0.8 + 0.4 * s)


def _rows(gen, T, K, dtype):
    """Activations: unit normal, each row of its own size, a few large columns."""
    x = torch.randn((T, K), generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn((T, 1), generator=gen, device="cuda"))
    x *= torch.where(torch.rand((1, K), generator=gen, device="cuda") < 0.01, 12.0, 1.0)
    return x.to(TYPES[dtype])


def _popular_logits(gen, T, E):
    """Router logits with popular and rare experts."""
    return (torch.randn((T, E), generator=gen, device="cuda") * 1.5
            + 0.7 * torch.randn((1, E), generator=gen, device="cuda"))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = dict(case)
    T = case["T"]
    dev = "cuda"
    i32 = torch.int32
    if case["op"] == "route":
        E, k = case["E"], case["k"]
        s["logits"] = _popular_logits(gen, T, E).to(TYPES[case["dtype"]])
        s["b"] = (torch.rand(E, generator=gen, device=dev) * 0.2 - 0.1) if case["bias"] else None
        s["outputs"] = {"topk_ids": torch.empty((T, k), dtype=i32, device=dev),
                        "topk_weights": torch.empty((T, k), device=dev),
                        "counts": torch.empty(E + 1, dtype=i32, device=dev),
                        "offsets": torch.empty(E + 2, dtype=i32, device=dev),
                        "perm": torch.empty(T * k, dtype=i32, device=dev)}
    elif case["op"] == "quant":
        K = case["K"]
        s["x"] = _rows(gen, T, K, case["dtype"])
        s["q"] = torch.empty((T, K), dtype=E4M3, device=dev)
        s["scales"] = torch.empty((T, _blocks(K)), device=dev)
    elif case["op"] == "gemm":
        N, K = case["N"], case["K"]
        s["xq"], s["sx"] = _plain_quant(_rows(gen, T, K, "bf16"))
        s["wq"], s["sw"] = _weights(gen, N, K)
        s["y"] = torch.empty((T, N), dtype=TYPES[case["out"]], device=dev)
    else:
        E, k, H, I = case["E"], case["k"], case["H"], case["I"]
        s["x"] = _rows(gen, T, H, "bf16")
        s["w"] = torch.empty((E, 3 * I * H), dtype=E4M3, device=dev)
        s["ws"] = torch.empty((E, 3 * _blocks(I) * _blocks(H)), device=dev)
        for e in range(E):
            nb = _blocks(I) * _blocks(H)
            for j, (r, c) in enumerate(((I, H), (I, H), (H, I))):
                q, sc = _weights(gen, r, c)
                s["w"][e, j * I * H:(j + 1) * I * H] = q.view(-1)
                s["ws"][e, j * nb:(j + 1) * nb] = sc.view(-1)
        p = torch.sigmoid(_popular_logits(gen, T, E))
        w, ids = torch.topk(p, k, dim=1)
        flat = ids.view(-1)
        counts = torch.bincount(flat, minlength=E + 1)
        s["routing"] = {"topk_ids": ids.to(i32), "topk_weights": w / w.sum(1, keepdim=True) * 2.5,
                        "counts": counts.to(i32),
                        "offsets": torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(i32),
                        "perm": torch.sort(flat, stable=True).indices.to(i32)}
        s["sizes"] = counts[:E].tolist()
        s["r"] = _rows(gen, T, H, "bf16") if case["resid"] else None
        s["y"] = torch.empty((T, H), dtype=torch.bfloat16, device=dev)
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _own(state)
    return {"route": _plain_route, "quant": _plain_quant_state, "gemm": _plain_gemm,
            "experts": _plain_experts}[state["op"]](state)


def _own(s):
    from hummingflight_b200 import fp8, moe
    if s["op"] == "route":
        return moe.route_logits(s["logits"], s["b"], s["k"], s["score"], s["n_group"],
                                s["topk_group"], s["group_top"], s["scale"], s["norm"],
                                out=s["outputs"])
    if s["op"] == "quant":
        fp8.quantize(s["x"], s["q"], s["scales"])
        return {"q": s["q"], "scales": s["scales"]}
    if s["op"] == "gemm":
        return fp8.gemm(s["xq"], s["sx"], s["wq"], s["sw"], s["y"])
    return fp8.moe_experts(s["x"], s["w"], s["ws"], s["routing"], s["r"], s["y"])


def _plain_route(s):
    T, E, k, G = s["T"], s["E"], s["k"], s["n_group"]
    # in 64 bits: which expert ranks before which is decided next to a border
    l = s["logits"].double()
    p = torch.sigmoid(l) if s["score"] == "sigmoid" else torch.softmax(l, 1)
    key = p if s["b"] is None else p + s["b"].double()
    if s["topk_group"] < G:
        best = torch.sort(key.view(T, G, E // G), dim=2, descending=True).values
        group = best[:, :, :s["group_top"]].sum(2)
        kept = torch.sort(group, dim=1, descending=True, stable=True).indices[:, :s["topk_group"]]
        allowed = torch.zeros((T, G), dtype=torch.bool, device=l.device).scatter_(1, kept, True)
        key = key.masked_fill(~allowed.repeat_interleave(E // G, 1), -math.inf)
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]
    w = p.gather(1, ids)
    if s["norm"]:
        w = w / w.sum(1, keepdim=True)
    flat = ids.reshape(-1)
    perm = torch.sort(flat, stable=True).indices
    counts = (flat[:, None] == torch.arange(E + 1, device=l.device)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    i32 = torch.int32
    return {"topk_ids": ids.to(i32), "topk_weights": (w * s["scale"]).float(),
            "counts": counts.to(i32), "offsets": offsets.to(i32), "perm": perm.to(i32)}


def _plain_quant(x):
    T, K = x.shape
    nb = _blocks(K)
    v = torch.nn.functional.pad(x.float(), (0, nb * BLOCK - K)).view(T, nb, BLOCK)
    m, e = torch.frexp(v.abs().amax(2))
    j = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)
    scale = torch.where(m == 0, torch.ones_like(m), torch.ldexp(torch.ones_like(m), j))
    q = (v / scale[:, :, None]).view(T, nb * BLOCK)[:, :K].to(E4M3)
    return q.contiguous(), scale


def _plain_quant_state(s):
    q, scale = _plain_quant(s["x"])
    return {"q": q, "scales": scale}


def _values(q, s, rows, cols, block_rows):
    """fp32 [rows x cols] that e4m3 values and block scales stand for."""
    s = s.repeat_interleave(block_rows, 0)[:rows] if block_rows > 1 else s
    return q.view(rows, cols).float() * s.repeat_interleave(BLOCK, 1)[:, :cols]


def _plain_gemm(s):
    T, N, K = s["T"], s["N"], s["K"]
    x = _values(s["xq"], s["sx"], T, K, 1)
    w = _values(s["wq"], s["sw"], N, K, BLOCK)
    return (x @ w.t()).to(TYPES[s["out"]])


def _plain_experts(s):
    T, k, H, I = s["T"], s["k"], s["H"], s["I"]
    n, nb = I * H, _blocks(I) * _blocks(H)
    r = s["routing"]
    perm = r["perm"].long()
    xq, sx = _plain_quant(s["x"])
    x = _values(xq, sx, T, H, 1)[perm // k]
    y = torch.empty((T * k, H), device=x.device)
    at = 0
    for e, c in enumerate(s["sizes"]):  # all experts at once would need 39 GB in fp32
        if c:
            w, ws = s["w"][e], s["ws"][e]
            rows = x[at:at + c]
            g = rows @ _values(w[:n], ws[:nb].view(_blocks(I), -1), I, H, BLOCK).t()
            u = rows @ _values(w[n:2 * n], ws[nb:2 * nb].view(_blocks(I), -1), I, H, BLOCK).t()
            mq, ms = _plain_quant(g / (1 + torch.exp(-g)) * u)
            d = _values(w[2 * n:], ws[2 * nb:].view(_blocks(H), -1), H, I, BLOCK)
            y[perm[at:at + c]] = _values(mq, ms, c, I, 1) @ d.t()
            at += c
    out = (y.view(T, k, H) * r["topk_weights"][:, :, None]).sum(1)
    if s["r"] is not None:
        out = s["r"].float() + out
    return out.to(torch.bfloat16)


# ------------------------------------------------------------------ cost
def work(case):
    T = case["T"]
    size = {"f32": 4, "bf16": 2}
    if case["op"] == "route":
        E, k = case["E"], case["k"]
        return {"bytes": T * E * size[case["dtype"]] + (4 * E if case["bias"] else 0)
                + T * k * 12 + 8 * E, "flops": 5 * T * E}
    if case["op"] == "quant":
        K = case["K"]
        return {"bytes": T * K * (size[case["dtype"]] + 1) + 4 * T * _blocks(K), "flops": 2 * T * K}
    if case["op"] == "gemm":
        N, K = case["N"], case["K"]
        return {"bytes": T * K + N * K + 4 * (T * _blocks(K) + _blocks(N) * _blocks(K))
                + T * N * size[case["out"]], "flops": 2 * T * N * K}
    E, k, H, I = case["E"], case["k"], case["H"], case["I"]
    active = E * (1 - (1 - k / E) ** T)
    return {"bytes": active * (3 * H * I + 12 * _blocks(H) * _blocks(I)) + T * H * 2 * 2
            + (T * H * 2 if case["resid"] else 0) + T * k * 8, "flops": 6 * T * k * H * I}


# ------------------------------------------------------------------ 64-bit values
def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "quant": _exact_quant, "gemm": _exact_gemm,
            "experts": _exact_experts}[case["op"]](s)


def _exact_route(s):
    T, E, k, G = s["T"], s["E"], s["k"], s["n_group"]
    l = s["logits"].double().cpu().numpy()
    if s["score"] == "sigmoid":
        p = 1 / (1 + np.exp(-l))
    else:
        p = np.exp(l - l.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
    key = p + (0.0 if s["b"] is None else s["b"].double().cpu().numpy())
    if s["topk_group"] < G:
        per = key.reshape(T, G, -1)
        score = -np.partition(-per, s["group_top"] - 1, axis=2)[:, :, :s["group_top"]].sum(2)
        rank = np.argsort(np.argsort(-score, 1, kind="stable"), 1, kind="stable")
        key = np.where((rank < s["topk_group"])[:, :, None], per, -np.inf).reshape(T, E)
    ids = np.argsort(-key, 1, kind="stable")[:, :k]
    w = np.take_along_axis(p, ids, 1)
    if s["norm"]:
        w = w / w.sum(1, keepdims=True)
    slots = np.lexsort((np.arange(T * k), ids.reshape(-1)))
    counts = np.bincount(ids.reshape(-1), minlength=E + 1)
    return {"topk_ids": ids.astype(np.int32), "topk_weights": w * s["scale"],
            "counts": counts.astype(np.int32),
            "offsets": np.concatenate([[0], np.cumsum(counts)]).astype(np.int32),
            "perm": slots.astype(np.int32)}


def _round_e4m3(v):
    """The e4m3 value nearest to each v (|v| <= 448, ties to even), as doubles."""
    e = torch.frexp(v)[1].clamp(min=-5)          # |v| < 2^e; normal values from 2^-6 up
    step = torch.ldexp(torch.ones_like(v), e - 4)  # four significant bits
    return torch.round(v / step) * step


def _exact_rows(x):
    """Quantised doubles and scales, by columns of 128."""
    x = x.double()
    qs, ss = [], []
    for c in range(0, x.shape[1], BLOCK):
        v = x[:, c:c + BLOCK]
        top = v.abs().max(1).values
        j = torch.ceil(torch.log2(top.clamp(min=2.0 ** -149) / 448))
        j = torch.where(top > 448 * torch.exp2(j), j + 1, j)
        j = torch.where(top <= 448 * torch.exp2(j - 1), j - 1, j).clamp(min=-126)
        sc = torch.where(top == 0, torch.ones_like(top), torch.exp2(j))
        qs.append(_round_e4m3(v / sc[:, None]))
        ss.append(sc)
    return torch.cat(qs, 1), torch.stack(ss, 1)


def _exact_quant(s):
    q, sc = _exact_rows(s["x"])
    return {"q": q, "scales": sc}


def _exact_product(xq, sx, w, ws):
    """sum over blocks of 128 columns: (xq block)(w block)^T scaled by both."""
    n, kk = w.shape
    y = torch.zeros((xq.shape[0], n), dtype=torch.float64, device=xq.device)
    row = torch.arange(n, device=w.device) // BLOCK
    for b in range(_blocks(kk)):
        c = slice(b * BLOCK, (b + 1) * BLOCK)
        part = xq[:, c] @ w[:, c].double().t()
        y += part * sx[:, b, None].double() * ws[row, b].double()[None]
    return y


def _exact_gemm(s):
    return _exact_product(s["xq"].double(), s["sx"], s["wq"], s["sw"])


def _exact_experts(s):
    T, k, H, I = s["T"], s["k"], s["H"], s["I"]
    xq, sx = _exact_rows(s["x"])
    ids, w = s["routing"]["topk_ids"].long(), s["routing"]["topk_weights"].double()
    out = torch.zeros((T, H), dtype=torch.float64, device="cuda")
    for e in range(s["E"]):
        t, i = torch.nonzero(ids == e, as_tuple=True)
        if t.numel() == 0:
            continue
        parts = s["w"][e].view(3, -1)
        sc = s["ws"][e].view(3, -1)
        g, u = (_exact_product(xq[t], sx[t], parts[j].view(I, H), sc[j].view(_blocks(I), -1))
                for j in (0, 1))
        mq, ms = _exact_rows(g * torch.sigmoid(g) * u)
        y = _exact_product(mq, ms, parts[2].view(H, I), sc[2].view(_blocks(H), -1))
        out.index_add_(0, t, y * w[t, i, None])
    return out if s["r"] is None else out + s["r"].double()
