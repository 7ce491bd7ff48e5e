"""CPU: the attention kernels hand registers from one role to another (setmaxnreg).  What the roles ask for has to fit what the block was launched
with, or the last to ask waits for good."""

from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

from tq_local_b200.build import CSRC, NVCC_FLAGS

NVCC = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"


@pytest.mark.skipif(not os.path.exists(NVCC), reason="needs nvcc")
@pytest.mark.parametrize("source,kernel,variants,roles", [
    # (threads, their registers after setmaxnreg)
    ("tq_prompt.cu", "tq_prompt_kernel", 2, [(256, "inc", 208), (128, "dec", 88)]),
    ("tq_tree.cu", "tq_tree_kernel", 6, [(256, "inc", 104), (512, "dec", 56), (128, "dec", 56)]),
])
@pytest.mark.parametrize("checked", [False, True])
def test_the_roles_registers_fit_the_launch(tmp_path, source, kernel, variants, roles, checked):
    text = open(os.path.join(CSRC, source)).read()
    asked = sorted((way, int(n)) for way, n in re.findall(r"setmaxnreg\.(inc|dec)\.sync\.aligned\.u32 (\d+)", text))
    assert asked == sorted((way, n) for _, way, n in roles)
    flags = [f for f in NVCC_FLAGS if f != "--shared"] + ["-Xptxas", "-v"] + (["-DTQ_DEBUG_BOUNDS"] if checked else [])
    said = subprocess.run([NVCC, *flags, "-c", os.path.join(CSRC, source), "-o", str(tmp_path / "out.o")], check=True, capture_output=True, text=True)
    used = [int(n) for name, n in re.findall(r"Compiling entry function '(\S+)'.*?Used (\d+) registers", said.stdout + said.stderr, re.S) if kernel in name]
    assert len(used) == variants
    threads = sum(n for n, _, _ in roles)
    for n in used:
        launched = (n + 7) // 8 * 8
        assert threads * launched <= 65536
        assert sum(t * r for t, _, r in roles) <= threads * launched, (n, roles)
        assert all(r <= launched if way == "dec" else r >= launched for _, way, r in roles)
