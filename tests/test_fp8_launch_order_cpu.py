"""The FP8 kernels' programmatic launches, from the source: a product may read weights and
offsets ahead of its own wait because every launch before it in the call lets it start
only behind its wait, when all earlier work is done."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "hummingflight_b200", "csrc")


def kernels(name):
    src = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
    for m in re.finditer(r"__global__[^;{]*?\b(k_\w+)\(", src):
        at = src.index("{", m.end())
        depth, end = 0, at
        while True:
            depth += {"{": 1, "}": -1}.get(src[end], 0)
            if depth == 0:
                break
            end += 1
        yield m.group(1), src[at:end]


def test_a_launch_lets_the_next_start_behind_its_own_wait():
    seen = 0
    for name in ("hf_fp8.cu", "hf_fp8_gemm.cu"):
        for kernel, body in kernels(name):
            trigger = body.find("griddep_launch_dependents()")
            if trigger >= 0:
                seen += 1
                assert 0 <= body.find("griddep_wait()") < trigger, kernel
    assert seen >= 5


def test_kernels_that_start_early_do_not_read_through_the_read_only_path():
    """ld.global.nc is for memory that nobody writes while the kernel lives; a kernel
    that starts ahead of its predecessor's end lives while its inputs are written."""
    for name in ("hf_fp8.cu", "hf_fp8_gemm.cu", "hf_logits.cu"):
        src = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
        assert not re.findall(r"\b(ld_nc_\w+|ld_stream_\w+|__ldg)\(|ld\.global\.nc", src), name
