"""FP8 operators against 64-bit plain forms (tests/fp8_ref.py holds the bounds)."""
import numpy as np
import pytest

import fp8_ref as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def rows(rng, T, K, dtype):
    x = rng.standard_normal((T, K)) * np.exp(rng.standard_normal((T, 1)))
    x = torch.from_numpy(x).to(torch.bfloat16 if dtype == "bf16" else torch.float32)
    return x, x.double().numpy()


def dev(v):
    return torch.from_numpy(np.ascontiguousarray(v)).float().cuda()


# ------------------------------------------------------------------ quantise
@pytest.mark.parametrize("T,K", [(1, 16), (1, 6144), (3, 112), (17, 128), (5, 1040), (64, 384),
                                 (1000, 144)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantize(T, K, dtype):
    need_gpu()
    from hummingflight_b200 import fp8
    x, xd = rows(np.random.default_rng(T + K), T, K, dtype)
    q, s = fp8.quantize(x.cuda())
    qr, sr = R.quantize(xd)
    assert np.array_equal(s.cpu().numpy(), sr)
    assert np.array_equal(q.view(torch.uint8).cpu().numpy(), R.bits(qr).numpy())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantize_edges(dtype):
    """Zeros, the smallest and largest numbers, values at the border of a scale and
    on rounding ties, Inf and NaN (their block becomes NaN, the others not)."""
    need_gpu()
    from hummingflight_b200 import fp8
    t = torch.bfloat16 if dtype == "bf16" else torch.float32
    x = torch.zeros((12, 256), dtype=t)
    x[1, :5] = torch.tensor([448.0, 449.0 if dtype == "f32" else 450.0, 1.0, -3.0, 0.0])
    x[2, :4] = torch.tensor([448.0, 17.0, 19.0, -21.0])      # ties between e4m3 neighbours
    x[3, :3] = torch.tensor([2.0 ** -133, -2.0 ** -130, 0.0])  # subnormal rows
    x[4, :3] = torch.tensor([torch.finfo(t).max, -1.0, 3.0])
    x[5, :2] = torch.tensor([float("inf"), 1.0])
    x[6, 130] = float("nan")
    x[7, 3] = -float("inf")
    x[8, :3] = torch.tensor([448.0, 2.0 ** -9, 2.0 ** -10])   # the smallest e4m3, and half of it
    x[9, :] = -0.0
    x[10, :3] = torch.tensor([448.0, 1.5 * 2.0 ** -9, -1.5 * 2.0 ** -9])
    x[11, :2] = torch.tensor([1.75, 1.7578125])
    q, s = fp8.quantize(x.cuda())
    qr, sr = R.quantize(x.double().numpy())
    assert np.array_equal(s.cpu().numpy(), sr, equal_nan=True)
    assert np.array_equal(q.float().cpu().numpy(), qr, equal_nan=True)


def test_quantize_rows_apart_and_out():
    """A view of wider rows, given outputs, rows behind the last left as they were."""
    need_gpu()
    from hummingflight_b200 import fp8
    x, xd = rows(np.random.default_rng(3), 9, 512, "bf16")
    view = x.cuda()[:, 128:128 + 176]
    q = torch.full((12, 176), 9, dtype=torch.uint8, device="cuda")
    s = torch.full((12, 2), 9.0, device="cuda")
    fp8.quantize(view, q[:9], s[:9])
    qr, sr = R.quantize(xd[:, 128:128 + 176])
    assert np.array_equal(q[:9].cpu().numpy(), R.bits(qr).numpy())
    assert np.array_equal(s[:9].cpu().numpy(), sr)
    assert (q[9:] == 9).all() and (s[9:] == 9).all()


# ------------------------------------------------------------------ product
GEMM = [(1, 1, 16), (1, 128, 128), (1, 1000, 2064), (2, 257, 144), (7, 384, 1024), (16, 130, 256),
        (17, 64, 4112), (31, 1, 512), (33, 513, 640), (64, 640, 384), (100, 129, 1040),
        (128, 256, 128), (129, 300, 272), (333, 1000, 528), (515, 260, 160),
        (97, 384, 2048), (49, 200, 1024),
        # more tiles than CTAs or CTA pairs: several a CTA
        (40, 40100, 256), (300, 10000, 272)]


@pytest.mark.parametrize("T,N,K", GEMM)
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_gemm(T, N, K, out):
    need_gpu()
    from hummingflight_b200 import fp8
    rng = np.random.default_rng(T * 7 + N + K)
    xq, sx = R.quantize(rows(rng, T, K, "bf16")[1])
    sx = sx * rng.uniform(0.5, 1.0, sx.shape).astype(np.float32)  # any scales, not powers of two
    sx = sx.astype(np.float32).astype(np.float64)
    wq, sw = R.weight(rng, N, K)
    y = fp8.gemm(R.bits(xq).cuda(), dev(sx), R.bits(wq).cuda(), dev(sw), out_dtype=out)
    ref, tol = R.product(R.values(xq, sx, T, K), R.values(wq, sw, N, K, True))
    err = np.abs(y.double().cpu().numpy() - ref)
    assert (err <= tol + R.rounding(ref, out == "bf16") * 1.01).all()


@pytest.mark.parametrize("T", [1, 40, 200])
def test_gemm_non_finite_rows_stay_apart(T):
    """NaN in one row (values or scale) and Inf in another's scale reach no other row,
    nor any row behind the last."""
    need_gpu()
    from hummingflight_b200 import fp8
    rng = np.random.default_rng(T)
    N, K = 192, 400
    xq, sx = R.quantize(rows(rng, T, K, "bf16")[1])
    wq, sw = R.weight(rng, N, K)
    xb, sd = R.bits(xq).cuda(), dev(sx)
    buf = torch.full((T + 3, N), 7.0, device="cuda")
    clean = fp8.gemm(xb, sd, R.bits(wq).cuda(), dev(sw), buf[:T])
    assert (buf[T:] == 7).all()
    clean = clean.clone()
    bad = T // 2
    xb[bad, 5] = 0x7f
    y = fp8.gemm(xb, sd, R.bits(wq).cuda(), dev(sw), out_dtype="f32")
    assert y[bad].isnan().all()
    keep = [t for t in range(T) if t != bad]
    assert torch.equal(y[keep], clean[keep])
    sd[T - 1, 1] = float("inf")
    y = fp8.gemm(R.bits(xq).cuda(), sd, R.bits(wq).cuda(), dev(sw), out_dtype="f32")
    assert not y[T - 1].isfinite().any()
    assert torch.equal(y[:T - 1], clean[:T - 1])


def test_gemm_is_deterministic_and_captured():
    """Two graphs that share a workspace, replayed in turn on new inputs."""
    need_gpu()
    from hummingflight_b200 import fp8
    rng = np.random.default_rng(9)
    graphs = []
    ws = None
    for T, N, K in ((1, 512, 1024), (48, 256, 2048), (300, 512, 512)):
        xq, sx = R.quantize(rows(rng, T, K, "bf16")[1])
        wq, sw = R.weight(rng, N, K)
        need = fp8.gemm_workspace_size(T, N, K)
        if ws is None or ws.numel() < need:
            ws = torch.empty(need + 4096, dtype=torch.uint8, device="cuda")
        t = [R.bits(xq).cuda(), dev(sx), R.bits(wq).cuda(), dev(sw)]
        y = fp8.gemm(*t, out_dtype="f32", workspace=ws)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            fp8.gemm(*t, out=y, workspace=ws)
        graphs.append((g, t, y, ws))
    for _ in range(2):
        for g, t, y, w in graphs:
            t[1].mul_(1.25)
            y.fill_(3.0)
            g.replay()
            torch.cuda.synchronize()
            fp8.status(w)
            assert torch.equal(y, fp8.gemm(*t, out_dtype="f32"))


# ------------------------------------------------------------------ experts
def make_experts(rng, E, H, I):
    n, nb = I * H, R.blocks(I) * R.blocks(H)
    q = np.empty((E, 3 * n))
    s = np.empty((E, 3 * nb))
    full = []
    for e in range(E):
        full.append([])
        for j, (r, c) in enumerate(((I, H), (I, H), (H, I))):
            a, b = R.weight(rng, r, c, 0.05)
            q[e, j * n:(j + 1) * n], s[e, j * nb:(j + 1) * nb] = a.reshape(-1), b.reshape(-1)
            full[e].append(R.values(a, b, r, c, True))
    return R.bits(q).cuda(), dev(s), full


def make_routing(rng, T, E, k, skew=1.0, only=None):
    l = rng.standard_normal((T, E)) + skew * rng.standard_normal(E)
    if only is not None:
        l[:, [e for e in range(E) if e not in only]] -= 100
    from hummingflight_b200 import moe
    r = moe.route_logits(torch.from_numpy(l).float().cuda(), None, k, "softmax")
    return r, r["topk_ids"].cpu().numpy(), r["topk_weights"].double().cpu().numpy()


EXPERTS = [  # T, E, k, H, I
    (1, 4, 2, 256, 128), (1, 1, 1, 16, 16), (1, 8, 8, 400, 144), (2, 16, 4, 256, 256),
    (5, 8, 3, 528, 272), (16, 33, 6, 384, 128), (40, 8, 2, 512, 384), (64, 16, 4, 144, 400),
    (130, 4, 2, 640, 256), (257, 3, 3, 256, 160), (300, 2, 1, 272, 512),
    # runs of K of the gate/up product (whole blocks of I) and of the down product
    (1, 4, 2, 4096, 256), (3, 6, 2, 2048, 384), (2, 4, 2, 2048, 272), (1, 2, 2, 256, 2048),
    # many picks; many tiles; tokens enough for the token-major gather
    (4, 40, 32, 128, 128), (100, 40, 2, 256, 512), (1000, 16, 2, 256, 1024),
    (2100, 4, 2, 272, 128)]


@pytest.mark.parametrize("T,E,k,H,I", EXPERTS)
@pytest.mark.parametrize("out,xt", [("bf16", "bf16"), ("f32", "f32")])
def test_experts(T, E, k, H, I, out, xt):
    need_gpu()
    from hummingflight_b200 import fp8
    rng = np.random.default_rng(T + 31 * E + H)
    q, s, full = make_experts(rng, E, H, I)
    routing, ids, w = make_routing(rng, T, E, k)
    x, xd = rows(rng, T, H, xt)
    resid, rd = rows(rng, T, H, out)
    y = fp8.moe_experts(x.cuda(), q, s, routing, resid.cuda(), out_dtype=out)
    ref, tol = R.experts(xd, full, ids, w, I, rd, out == "bf16", out == "bf16")
    assert (np.abs(y.double().cpu().numpy() - ref) <= tol).all()


@pytest.mark.parametrize("T", [3, 90, 400])
def test_experts_empty_segments_and_one_hot_expert(T):
    """Most experts without a token, the last one with all of them; no residual;
    a workspace full of other calls' bytes; rows that lie apart."""
    need_gpu()
    from hummingflight_b200 import fp8
    rng = np.random.default_rng(T)
    E, k, H, I = 20, 2, 256, 192
    q, s, full = make_experts(rng, E, H, I)
    routing, ids, w = make_routing(rng, T, E, k, only=(4, E - 1))
    x, xd = rows(rng, T, 2 * H, "bf16")
    ws = torch.full((fp8.moe_experts_workspace_size(T, k, E, H, I),), 255, dtype=torch.uint8,
                    device="cuda")
    y = fp8.moe_experts(x.cuda()[:, H:], q, s, routing, workspace=ws)
    fp8.status(ws)
    ref, tol = R.experts(xd[:, H:], full, ids, w, I)
    assert (np.abs(y.double().cpu().numpy() - ref) <= tol).all()


def test_experts_non_finite_token_stays_apart():
    need_gpu()
    from hummingflight_b200 import fp8
    rng = np.random.default_rng(2)
    T, E, k, H, I = 50, 4, 2, 256, 256
    q, s, _ = make_experts(rng, E, H, I)
    routing, _, _ = make_routing(rng, T, E, k)
    x = rows(rng, T, H, "bf16")[0].cuda()
    y = fp8.moe_experts(x, q, s, routing).clone()
    x[7, 3], x[20, 200] = float("inf"), float("nan")
    z = fp8.moe_experts(x, q, s, routing)
    assert z[7].isnan().all() and z[20].isnan().all()
    keep = [t for t in range(T) if t not in (7, 20)]
    assert torch.equal(y[keep], z[keep])


def test_layer_of_operators():
    """A layer as an engine runs it: routing, the routed experts onto the residual,
    the shared expert (E = 1) in place on top; captured and replayed."""
    need_gpu()
    from hummingflight_b200 import fp8, moe
    rng = np.random.default_rng(12)
    T, E, k, H, I, Is = 70, 16, 4, 384, 256, 128
    q, s, full = make_experts(rng, E, H, I)
    qs, ss, fs = make_experts(rng, 1, H, Is)
    x, xd = rows(rng, T, H, "bf16")
    xg = x.cuda()
    hidden, hd = rows(rng, T, H, "f32")
    hg = hidden.cuda()
    logits = torch.from_numpy(rng.standard_normal((T, E))).float().cuda()
    bias = torch.from_numpy(rng.uniform(-0.1, 0.1, E)).float().cuda()
    one = dict(topk_weights=torch.ones((T, 1), device="cuda"),
               offsets=torch.tensor([0, T], dtype=torch.int32, device="cuda"),
               perm=torch.arange(T, dtype=torch.int32, device="cuda"))
    out = torch.empty((T, H), device="cuda")

    def layer():
        r = moe.route_logits(logits, bias, k, "sigmoid", 4, 2, 2, 2.5, True)
        fp8.moe_experts(xg, q, s, r, hg, out)
        fp8.moe_experts(xg, qs, ss, one, out, out)
        return r

    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = layer()
    for seed in (3, 4):
        logits.copy_(torch.randn((T, E), generator=torch.Generator().manual_seed(seed)))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        ids, w, _, _, _ = R.route(logits.double().cpu().numpy(), bias.double().cpu().numpy(), k,
                                  "sigmoid", 4, 2, 2, 2.5, True)
        assert np.array_equal(r["topk_ids"].cpu().numpy(), ids)
        w = r["topk_weights"].double().cpu().numpy()
        a, ea = R.experts(xd, full, ids, w, I, hd, False, False)
        b, eb = R.experts(xd, fs, np.zeros((T, 1), int), np.ones((T, 1)), Is, a, False, False)
        assert (np.abs(out.double().cpu().numpy() - b) <= ea + eb).all()


@pytest.mark.parametrize("T,H,I", [(1, 2048, 384), (24, 512, 256), (600, 512, 256)])
def test_inputs_written_just_before_the_call(T, H, I):
    """Weights, scales, tokens and routing that the launches right ahead of the call
    wrote are the ones it reads (the products ask for weights early): eager and
    replayed, equal to the same call with the stream idle in between."""
    need_gpu()
    from hummingflight_b200 import fp8, moe
    E, k = 8, 2
    rng = np.random.default_rng(T)
    sets = []
    for _ in range(2):
        q, s, _ = make_experts(rng, E, H, I)
        sets.append((q, s, rows(rng, T, H, "bf16")[0].cuda(), torch.randn((T, E), device="cuda")))
    q, s, x, l = (v.clone() for v in sets[0])
    out = torch.empty((T, H), dtype=torch.bfloat16, device="cuda")

    def write(v):
        l.copy_(v[3])
        x.copy_(v[2])
        s.copy_(v[1])
        q.copy_(v[0])

    def call():
        return fp8.moe_experts(x, q, s, moe.route_logits(l, None, k), out=out)

    want = []
    for v in sets:
        write(v)
        torch.cuda.synchronize()
        call()
        torch.cuda.synchronize()
        want.append(out.clone())
    assert not torch.equal(*want)
    for i in [0, 1] * 4:  # back to back: the writes overwrite what the call before read
        write(sets[i])
        assert torch.equal(call(), want[i])
    graphs = []
    for v in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            write(v)
            call()
    for i in [0, 1] * 4:
        graphs[i].replay()
        assert torch.equal(out, want[i])


def test_routing_of_the_bf16_layer_is_taken():
    """The dict of MoELayer.route (its permutation has the shared expert's slots
    behind the routed ones)."""
    need_gpu()
    from hummingflight_b200 import fp8, moe
    from hummingflight_b200.configs import LayerShape
    rng = np.random.default_rng(5)
    shape = LayerShape(256, 8, 2, 128, 128, 2.5, True)
    L = moe.MoELayer(shape, 1, 64)
    L.synth_layer(0, 3)
    T = 37
    x, xd = rows(rng, T, 256, "bf16")
    r = L.route(0, x.cuda())
    q, s, full = make_experts(rng, 8, 256, 128)
    y = fp8.moe_experts(x.cuda(), q, s, r)
    ref, tol = R.experts(xd, full, r["topk_ids"].cpu().numpy(),
                         r["topk_weights"].double().cpu().numpy(), 128)
    assert (np.abs(y.double().cpu().numpy() - ref) <= tol).all()
    L.close()


def test_experts_whose_offsets_pass_32_bits():
    """The last expert's block starts beyond 2^32 bytes; the other experts' bytes are
    left as they came (never read)."""
    need_gpu()
    from hummingflight_b200 import fp8
    rng = np.random.default_rng(8)
    E, H, I, T = 400, 2048, 1792, 3
    n, nb = I * H, R.blocks(I) * R.blocks(H)
    q = torch.empty((E, 3 * n), dtype=torch.uint8, device="cuda")
    s = torch.empty((E, 3 * nb), device="cuda")
    assert (E - 1) * 3 * n > 2 ** 32
    one, os, full = make_experts(rng, 1, H, I)
    q[E - 1], s[E - 1] = one[0], os[0]
    off = torch.zeros(E + 2, dtype=torch.int32, device="cuda")
    off[E:] = T
    routing = dict(topk_weights=torch.full((T, 1), 0.75, device="cuda"), offsets=off,
                   perm=torch.arange(T, dtype=torch.int32, device="cuda"))
    for rows_ in (T, 100):
        routing.update(topk_weights=torch.full((rows_, 1), 0.75, device="cuda"),
                       perm=torch.arange(rows_, dtype=torch.int32, device="cuda"))
        off[E:] = rows_
        x, xd = rows(rng, rows_, H, "bf16")
        y = fp8.moe_experts(x.cuda(), q, s, routing)
        ref, tol = R.experts(xd, full, np.zeros((rows_, 1), int), np.full((rows_, 1), 0.75), I)
        assert (np.abs(y.double().cpu().numpy() - ref) <= tol).all()


def test_experts_bad_permutation_stays_in_bounds():
    """Entries and offsets out of range: the call returns, and rows that are named
    properly keep their values."""
    need_gpu()
    from hummingflight_b200 import fp8
    rng = np.random.default_rng(3)
    for T in (6, 1200):
        E, k, H, I = 4, 1, 256, 128
        q, s, _ = make_experts(rng, E, H, I)
        x = rows(rng, T, H, "bf16")[0].cuda()
        r = dict(topk_weights=torch.ones((T, k), device="cuda"),
                 offsets=torch.tensor([0, T, T, T, T, T], dtype=torch.int32, device="cuda"),
                 perm=torch.arange(T, dtype=torch.int32, device="cuda"))
        good = fp8.moe_experts(x, q, s, r).clone()
        r["perm"][2], r["perm"][3] = -5, 2 ** 30
        ws = torch.full((fp8.moe_experts_workspace_size(T, k, E, H, I),), 255, dtype=torch.uint8,
                        device="cuda")
        y = fp8.moe_experts(x, q, s, r, workspace=ws)
        keep = [t for t in range(T) if t not in (2, 3)]
        assert torch.equal(y[keep], good[keep])
        r["offsets"].copy_(torch.tensor([-7, T + 100, 2 ** 30, 5, -1, T], dtype=torch.int32))
        fp8.moe_experts(x, q, s, r, workspace=ws)
        fp8.status(ws)


def test_memory_of_a_call_on_another_stream(monkeypatch):
    """What a call allocates belongs to the stream that it runs on: the next tensor
    of the current stream is not given the workspace of a call still running there."""
    need_gpu()
    from hummingflight_b200 import fp8, moe
    T, N, K = 8, 512, 4096
    need = fp8.gemm_workspace_size(T, N, K)
    assert need > 1 << 16  # runs of K
    xq, sx = fp8.quantize(torch.randn((T, K), device="cuda"))
    wq = torch.randn((N, K), device="cuda").to(torch.float8_e4m3fn)
    sw = torch.ones((fp8.blocks(N), fp8.blocks(K)), device="cuda")
    made = []

    def scratch(*args):
        ws = moe.scratch(*args)
        made.append(ws.data_ptr())
        return ws

    monkeypatch.setattr(fp8, "scratch", scratch)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    y = fp8.gemm(xq, sx, wq, sw, stream=side)
    here = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in range(4)]
    assert made and not set(made) & {t.data_ptr() for t in here}
    side.synchronize()
    assert torch.equal(y, fp8.gemm(xq, sx, wq, sw))


def test_two_streams_at_once():
    """Independent calls that overlap on two streams, each with its own workspace."""
    need_gpu()
    from hummingflight_b200 import fp8
    rng = np.random.default_rng(11)
    T, E, k, H, I = 200, 8, 2, 512, 256
    q, s, _ = make_experts(rng, E, H, I)
    a, _, _ = make_routing(rng, T, E, k)
    b, _, _ = make_routing(rng, T, E, k)
    x = rows(rng, T, H, "bf16")[0].cuda()
    want = [fp8.moe_experts(x, q, s, r).clone() for r in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        got = [fp8.moe_experts(x, q, s, r, stream=st) for r, st in zip((a, b), streams)]
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
