"""Rules that kernels keep so that no wait is endless, read off their sources: what breaks one shows on a GPU as a hang, if at
all, so it is not tried there."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "objectsam_b200", "csrc")


def kernels():
    """(file:name, body) of every __global__ function of the package, comments taken out."""
    out = []
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))):
        text = re.sub(r"//[^\n]*", "", open(path, encoding="utf-8").read())
        for m in re.finditer(r"__global__\s+void\b[^{;]*?\b(k_\w+)\s*\(", text):
            at = depth = text.index("{", m.end())
            depth = 0
            for end in range(at, len(text)):
                depth += (text[end] == "{") - (text[end] == "}")
                if not depth:
                    break
            out.append((f"{os.path.basename(path)}:{m.group(1)}", text[at:end + 1]))
    return out


def test_kernels_are_found():
    names = [n for n, _ in kernels()]
    assert "attn_fwd.cuh:k_attn_fwd" in names and "attn_bwd.cuh:k_attn_bwd" in names and len(names) > 40


def test_dependents_start_after_tensor_memory_is_taken():
    """A kernel that lets the next one start before its own CTAs have their TMEM columns may find them taken by CTAs that
    wait for it to end."""
    both = [(n, b) for n, b in kernels() if "tmem_alloc" in b and "grid_dep_launch" in b]
    assert {"attn_fwd.cuh:k_attn_fwd", "attn_bwd.cuh:k_attn_bwd", "conv_fprop.cuh:k_conv_fprop"} <= {n for n, _ in both}
    for name, body in both:
        between = body[body.rindex("tmem_alloc"):body.index("grid_dep_launch")]
        assert body.rindex("tmem_alloc") < body.index("grid_dep_launch") and "__syncthreads" in between, name
