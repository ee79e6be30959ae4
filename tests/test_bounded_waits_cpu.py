"""What the kernels do when a wait has run out, read from their source: the state cannot be brought about on a GPU without a stall."""
import os
import re

import pytest

from archscale_b200 import build

CU = sorted(f for f in os.listdir(build.CSRC) if f.endswith(".cu"))


def _source(name):
    text = open(os.path.join(build.CSRC, name), encoding="utf-8").read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


def _block(text, start):
    """The text from ``start`` to the bracket that closes the first one after it."""
    at = text.index("{", start)
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[at + 1:i]
    raise AssertionError("brackets do not match")


def test_block():
    assert _block("for (;;) { a { b } c } d { e }", 0) == " a { b } c "


@pytest.mark.parametrize("name", [f for f in CU if "fp8" in f])
def test_every_warp_reaches_every_named_barrier(name):
    """A loop with a barrier that only some warps of a block take part in (``bar.sync`` with a number) is left by all of them after the same turn: by its
    condition, which they share, not by one warp whose own wait has failed; and nothing before the barrier skips a turn."""
    text = _source(name)
    for m in re.finditer(r"\bfor \(int", text):
        loop = _block(text, m.start())
        if not re.search(r"bar\.sync [1-9]", loop):
            continue
        assert not re.search(r"\b(break|goto|return)\b", loop), loop
        last = max(x.start() for x in re.finditer(r"bar\.sync [1-9]", loop))
        assert "continue" not in loop[:last]


@pytest.mark.parametrize("name", ["gemm_fp8_block.cu", "gemm2_fp8_block.cu"])
def test_a_kernel_that_gives_up_waits_for_what_it_has_issued(name):
    """After the block's last barrier the warps of the loads and of the products look at the flag of a wait that ran out, and drain their rings before the
    cluster parts and tensor memory is freed; copies of single threads are waited for by the threads themselves."""
    text = _source(name)
    kernel = _block(text, text.index("gemm2_fp8_block_kernel(" if "2" in name else "gemm_fp8_block_kernel("))
    barrier, drain, free = (kernel.rindex(w) for w in ("__syncthreads()", "drain_ring(", "tmem_dealloc"))
    assert barrier < drain < kernel.rindex("cluster_sync_all()") and drain < free
    assert re.search(r"warp < 2 && \*abort_flag\) drain_ring\(", kernel)
    assert kernel.count("++issued;") == 2
    if "f2_cp_async" in kernel:
        assert barrier > kernel.rindex("cp.async.wait_all") > kernel.index("done:")
