"""The routed FP8 experts over permutations and offsets that leave slots out, on a
workspace that an earlier call has filled with positions of its own."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


# T, E, k, H, I: positions gathered one by one, runs of K, by tokens; CTA pairs
@pytest.mark.parametrize("T,E,k,H,I", [(3, 4, 2, 2048, 384), (50, 6, 3, 256, 128),
                                       (700, 5, 2, 256, 128), (40, 70, 32, 128, 128)])
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_left_out_slots_add_nothing(T, E, k, H, I, out):
    """Equal to the call that names every slot with the left out ones' weights at 0."""
    need_gpu()
    from hummingflight_b200 import fp8, moe
    g = torch.Generator(device="cuda").manual_seed(T)
    q = torch.randn((E, 3 * I * H), generator=g, device="cuda").mul_(50).to(torch.float8_e4m3fn)
    s = torch.rand((E, 3 * fp8.blocks(I) * fp8.blocks(H)), generator=g, device="cuda") * 1e-3
    x = torch.randn((T, H), generator=g, device="cuda").bfloat16()
    ws = torch.empty(fp8.moe_experts_workspace_size(T, k, E, H, I, out), dtype=torch.uint8,
                     device="cuda")

    def call(r):
        return fp8.moe_experts(x, q, s, r, out_dtype=out, workspace=ws).clone()

    def routing(seed):
        l = torch.randn((T, E), generator=g.manual_seed(seed), device="cuda")
        return moe.route_logits(l, None, k, "softmax")

    n = T * k
    rng = np.random.default_rng(T)
    for kind in ("unnamed", "offsets"):
        r = routing(1)
        perm = r["perm"].clone()
        if kind == "unnamed":
            gone = torch.from_numpy(rng.permutation(n)[:max(1, n // 3)]).cuda()  # positions
            r["perm"][gone] = torch.tensor([-1, n, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32,
                                           device="cuda").repeat(len(gone))[:len(gone)]
        else:
            first, end = n // 5, n - max(1, n // 4)
            gone = torch.cat([torch.arange(first), torch.arange(end, n)]).cuda()
            r["offsets"].clamp_(first, end)
        w = r["topk_weights"].clone()
        w.view(-1)[perm[gone].long()] = 0
        # the same positions hold the rest: the sums are equal bit by bit
        call(routing(2))
        got = call(r)
        call(routing(3))
        assert torch.equal(call(r), got)
        want = call({**routing(1), "topk_weights": w})
        assert torch.equal(got, want)
