"""What the assembler makes of kernels that only run with one outcome (needs nvcc, no GPU)."""
import re


def test_prompt_attention_has_the_registers_that_its_warps_share_out(pkg):
    """The launch refuses any other number; here a compiler that gives one is noticed without a
    GPU.  All ten kernels: two types, head sizes of 32 and 64 with two unit lengths, 128 with one."""
    from gpt_oss_b200 import build

    source = build.CSRC / "prompt_attention.cu"
    kernels = build.kernel_resources(source)
    assert len(kernels) == 10 and all("prompt_attention_kernel" in name for name in kernels)
    threads = int(re.search(r"kAttnThreads = (\d+);", source.read_text()).group(1))
    want = 65536 // threads // 8 * 8
    assert {name: r for name, r in kernels.items() if r != (want, 0, 0)} == {}
