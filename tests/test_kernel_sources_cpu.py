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
        # the warp that has allocated signals, or the CTA has met since
        assert body.rindex("tmem_alloc") < body.index("grid_dep_launch"), name
        assert "__syncthreads" in between or not re.search(r"[{}]", between), name


def block(text, start):
    """The brace block that follows `start`."""
    at = text.index("{", text.index(start))
    depth = 0
    for end in range(at, len(text)):
        depth += (text[end] == "{") - (text[end] == "}")
        if not depth:
            return text[at:end + 1]


@pytest.mark.parametrize("kernel,loop", [("attn_fwd.cuh:k_attn_fwd", "for (int t = tiles.first(); t < tiles.end; it++)"),
                                         ("attn_bwd.cuh:k_attn_bwd", "for (; x.more(tiles, streams); x.step(tiles), it++)")])
def test_warps_whose_wait_ran_out_stay_in_step(kernel, loop):
    """The softmax warps share named barriers, which have no bound: none leaves the loop over the tiles early, waits again
    after a failed wait, or arrives for others after one."""
    body = dict(kernels())[kernel]
    tiles = block(body, loop)
    assert "named_bar_sync" in tiles and not re.search(r"\b(break|return|goto)\b", tiles)
    for wait in re.finditer(r"[^;{}]*\bat_wait\w*\(", tiles):
        assert re.search(r"ok = ok && |\bif \([^=]*\bok\b[^=]*\) (lead &= )?ok = ", wait.group(0)), wait.group(0)
    for arrive in re.finditer(r"[^;{}]*\bat_arrive\(", tiles):
        assert re.search(r"if \((lead|lane == 0 && ok)\)", arrive.group(0)), arrive.group(0)
    if "if (lead)" in tiles:  # `lead` is what is agreed on in the tile in which a wait ran out
        assert re.search(r"ok = !at_pair_any\(pair_bar, !ok\);.*?ok = at_wait_warp\(&pv_done[^;]*;\s*lead &= ok;", tiles, re.S)


def test_results_are_written_by_agreement():
    """The forward's barriers behind its loop over the tiles: a failed wait is agreed on before any that only some pass."""
    body = dict(kernels())["attn_fwd.cuh:k_attn_fwd"]
    tail = body[body.index("at_wait_warp(&o_done, 0, A.err);\n    tc_fence_after"):]
    head = tail[:tail.index("if (ok)")]
    assert "at_pair_any(pair_bar, !ok)" in head and "at_any(1, !ok, kAfSoft)" in head


def test_buffers_of_the_columns_go_by_their_barriers():
    """The forward fills its two buffers of per-key data in some tiles only, with a barrier in those: a buffer chosen by the
    tile's number could be filled again while a warp still reads what it held two tiles ago."""
    tiles = block(dict(kernels())["attn_fwd.cuh:k_attn_fwd"], "for (int t = tiles.first(); t < tiles.end; it++)")
    fill = block(tiles, "if (by_doc || BIAS == 2)")
    assert "fills++;" in fill and "named_bar_sync(1, kAfSoft);" in fill and tiles.count("fills++") == 1
    assert "const int slot = fills & 1;" in tiles[:tiles.index(fill)]
    uses = re.findall(r"col_(?:doc|y|x)\[([^]]*)\]", tiles)
    assert len(uses) == 6 and set(uses) == {"slot"}
