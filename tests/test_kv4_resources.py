"""Registers of the attention kernels (CPU: the sources are compiled, not run): a spill in a loop
over the cache's tokens goes to memory and back in every block."""
import os
import re

import pytest

from test_kernel_resources import CSRC, HIPCC, demangle, kernel_resources


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not installed")
@pytest.mark.parametrize("src,kernel,bars", [
    # bytes of scratch allowed by 64 elements of head_dim: one block of f32 rows of 192 keeps a
    # few words out of its loop, and the 256-row kernel is at its 256 registers
    ("kern_attn.hip", "k_kv4_attn", {1: 0, 2: 0, 3: 32, 4: 32}),
    ("kern_prompt.hip", "k_kv4_prompt", {1: 0, 2: 96, 3: 64, 4: 720})])
def test_attention_kernels_within_register_budget(tmp_path, src, kernel, bars):
    res = kernel_resources(os.path.join(CSRC, src), tmp_path)
    names = demangle(list(res))
    seen = 0
    for mangled, (scratch, _) in res.items():
        # (names with bf16 are left mangled by older demanglers)
        m = re.search(kernel + r"<\d, (\d)", names[mangled]) or \
            re.search(kernel + r"ILi\dELi(\d)E", names[mangled])
        if m:
            seen += 1
            bar = bars[int(m.group(1))]
            assert scratch <= bar, f"{names[mangled]}: {scratch} bytes of scratch (bar {bar})"
    assert seen >= 16
