"""What head_logprobs' kernels need of their build, without a GPU."""
import re
import subprocess

import pytest

from nano_vllm_b200 import build


def test_the_kernels_of_long_sums_have_the_registers_that_their_warps_share(tmp_path):
    """Their warp groups trade registers of what the block was launched with: fewer, and the library refuses the call."""
    source = build.CSRC / "head_logprobs.cu"
    needed = int(re.search(r"\bREGS = (\d+),", source.read_text()).group(1))
    flags = [f for f in build.NVCC_FLAGS if f not in ("-shared", "-cudart", "static")]
    try:
        nvcc = build._nvcc()
    except RuntimeError:
        pytest.skip("no nvcc")
    done = subprocess.run([nvcc, *flags, "-Xptxas", "-v", "-c", str(source), "-o", str(tmp_path / "head.o")], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    used = {}
    for kernel, report in re.findall(r"Compiling entry function '(\S+)'(.*?Used \d+ registers)", done.stderr, re.S):
        used[kernel] = int(re.search(r"Used (\d+) registers", report).group(1))
    forms = {k: n for k, n in used.items() if "head_logprobs_kernel" in k}
    assert len(forms) == 4
    long_sums = {k: n for k, n in forms.items() if "Lb1EEE" in k}  # the second template argument
    assert len(long_sums) == 2 and set(long_sums.values()) == {needed}, forms
