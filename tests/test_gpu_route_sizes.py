"""hf_route_logits at sizes whose shared memory lies next to what a launch gets without
asking for it (48 KB with the kernels' static part), each as its kernel's first call."""
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# tokens, experts, groups: 49088 and 49152 bytes of dynamic shared memory; the second
# needs as much for the permutation
SIZES = [(11000, 208, 8), (65536, 768, 1), (24576, 512, 4)]

CHECK = """
import torch
from hummingflight_b200 import moe
for T, E, G in %r:
    l = torch.randn((T, E), generator=torch.Generator(device="cuda").manual_seed(T), device="cuda")
    keep = max(1, G // 2)
    r = moe.route_logits(l, None, 8, "softmax", G, keep, 1)
    key = l.double()
    if G > 1:  # softmax, one key a group: groups rank by their largest logit
        best = torch.sort(key.view(T, G, -1).amax(2), dim=1, descending=True, stable=True).indices[:, :keep]
        ok = torch.zeros((T, G), dtype=torch.bool, device="cuda").scatter_(1, best, True)
        key = key.masked_fill(~ok.repeat_interleave(E // G, 1), -float("inf"))
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :8]
    assert torch.equal(r["topk_ids"].long(), ids)
    w = torch.softmax(l.double(), 1).gather(1, ids)
    w /= w.sum(1, keepdim=True)
    # the tolerance of the fp32 scores: |l - m| + E + picks half steps
    assert ((r["topk_weights"] - w).abs() <= (20 + 100 + 16) * 2.0 ** -24 * w).all()
    flat = ids.reshape(-1)
    assert torch.equal(r["perm"].long(), torch.sort(flat, stable=True).indices)
    assert torch.equal(r["counts"].long(), torch.bincount(flat, minlength=E + 1))
""" % (SIZES,)


@pytest.mark.gpu
def test_shared_memory_next_to_the_plain_limit():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    r = subprocess.run([sys.executable, "-c", CHECK], cwd=ROOT, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
