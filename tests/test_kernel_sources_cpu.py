"""Rules of synchronisation that the kernels' sources have to keep and that no run shows reliably (no GPU)."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bytes_b200", "csrc")
KERNELS = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
SOURCES = sorted(KERNELS + glob.glob(os.path.join(CSRC, "*.cuh")))


def code(path):
    """The source without comments."""
    src = re.sub(r"/\*.*?\*/", "", open(path).read(), flags=re.S)
    return re.sub(r"//[^\n]*", "", src)


def enclosing_block(src, at):
    """(the text before the brace that opens the innermost block around `at`, the block)."""
    depth, start = 0, at
    while True:
        start -= 1
        depth += {"}": 1, "{": -1}.get(src[start], 0)
        if depth < 0:
            break
    depth, end = 0, at
    while depth >= 0:
        depth += {"{": 1, "}": -1}.get(src[end], 0)
        end += 1
    return src[:start].rstrip(), src[start:end]


@pytest.mark.parametrize("path", KERNELS, ids=os.path.basename)
def test_barriers_are_initialised_by_the_thread_that_fences_them(path):
    """fence.mbarrier_init orders the executing thread's own inits ahead of the copies that complete on
    them: one thread makes all of a set of barriers, and the same one fences."""
    src = code(path)
    for m in re.finditer(r"\bmbar_init\(", src):
        head, block = enclosing_block(src, m.start())
        assert re.search(r"if \([^{};]*(threadIdx\.x|lane) == 0\)$", head), head[-80:]
        inits = [i.start() for i in re.finditer(r"\bmbar_init\(", block)]
        assert "mbar_fence_init()" in block[inits[-1]:]


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_aligned_cluster_barriers_have_their_warps_together(path):
    """barrier.cluster.*.aligned wants all lanes of a warp at it together: the statement before it sees to that."""
    src = code(path)
    for m in re.finditer(r"barrier\.cluster\.arrive[a-z.]*\.aligned", src):
        before = src[:m.start()].rsplit("asm", 1)[0].rstrip()
        assert before.endswith(("__syncwarp();", "__syncthreads();")), before[-80:]


def test_lengths_that_are_read_ahead_of_a_wait_come_from_l2():
    """The joins, and the tile kernel after a choice, read the lengths before they wait for the kernel ahead of them: past
    L1, which may hold them from an earlier step. Nothing in that file reads them in another way."""
    assert "early ? __ldcg(at) : *at" in code(os.path.join(CSRC, "paged.cuh"))
    attn = code(os.path.join(CSRC, "paged_attn.cu"))
    assert not re.search(r"\blens\s*[\[+]", attn)
    tiles, joins = attn.index("int row_slots"), attn.index("struct Parts")
    for m in re.finditer(r"paged_len\(([^()]*)\)", attn):
        early = m.group(1).split(",")[2:]
        assert early == ([] if m.start() < tiles else [" p.after_select"] if m.start() < joins else [" true"])
