"""Rules of the kernels' source that no run can show: what they prevent needs a wait to
give up at one moment in one warp, and then hangs the GPU (no GPU needed)."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mix_precision_kernel_b200", "csrc")


def _source(name):
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    return re.sub(r"//[^\n]*", "", text)  # comments name the functions too


def _block(text, start):
    """The brace-enclosed block that opens at or after `start`."""
    at = text.index("{", start)
    depth = 0
    for i in range(at, len(text)):
        depth += (text[i] == "{") - (text[i] == "}")
        if depth == 0:
            return text[at:i + 1]
    raise AssertionError("unbalanced braces")


def test_warps_leave_a_wait_together():
    """Lanes of a warp see a wait expire each for itself, so a whole warp that waits takes a
    vote before it branches.  Only the elected lane of a producer or issuer waits alone."""
    text = _source("products.cu")
    kernel = _block(text, text.index("product_kernel(const __grid_constant__"))
    alone = []
    for elected in re.finditer(r"if \((?:rank == 0 && )?elect_one\(\)\) ", kernel):
        alone.append(_block(kernel, elected.end()))
    assert len(alone) == 2 and all("mbar_wait(" in a for a in alone)
    together = kernel
    for a in alone:
        together = together.replace(a, "")
    assert "mbar_wait(" not in together
    # the tail rows, the epilogue of whole tiles and the join of split ones
    assert together.count("mbar_wait_warp(") == 3
    helper = _block(_source("mpk_ptx.cuh"), _source("mpk_ptx.cuh").index("bool mbar_wait_warp("))
    assert re.search(r"__all_sync\(0xFFFFFFFFu, mbar_wait\(", helper)


def test_warps_meet_before_warp_wide_instructions():
    """Lanes past N leave a chunk's stores early, and rows of x end in different lanes: the
    aligned instructions that follow come after a __syncwarp."""
    text = _source("products.cu")
    kernel = _block(text, text.index("product_kernel(const __grid_constant__"))
    chunks = [_block(kernel, m.end()) for m in re.finditer(r"for \(int c = 32 \* turn; [^{]*", kernel)]
    assert len(chunks) == 2
    for c in chunks:
        assert 0 < c.index("__syncwarp()") < c.index("tmem_ld_32x32b_x32(")
    for scope in (_block(kernel, kernel.index("if (p.splits > 1 && unit")),
                  _block(text, text.index("void make_codes("))):
        syncs = list(re.finditer(r"(?:cluster_sync_all|named_bar_sync)\(", scope))
        assert syncs
        for s in syncs:
            before = re.split(r"[;{}]", scope[:s.start()])
            assert "__syncwarp()" in before[-2], scope[s.start() - 120:s.end()]


def test_an_expired_wait_stops_the_whole_join():
    """CTAs that share a tile's reduction hand their sums to one another.  One whose wait gave up
    hands over nothing: it raises the flag of every CTA of the cluster before the barrier
    behind which the sums are added, and each looks at its flag there."""
    text = _source("products.cu")
    kernel = _block(text, text.index("product_kernel(const __grid_constant__"))
    join = _block(kernel, kernel.index("if (p.splits > 1 && unit"))
    wait = join.index("mbar_wait_warp(")
    raised = re.search(r"if \(!ok && lane < ctas\)\s*st_shared_cluster_u32\(mapa_shared\("
                       r"smem_u32\(const_cast<int\*>\(abort_flag\)\), \(uint32_t\)lane\), 1u\);", join)
    assert raised and wait < raised.start()
    parts = join.index("st_shared_cluster_v4(")
    barrier = join.index("cluster_sync_all();", parts)
    added = join.index("if (busy && *abort_flag == 0)")
    assert raised.end() < parts < barrier < added


def test_warps_of_the_gemm_kernels_leave_a_wait_together():
    """The same rule in the MXFP8 GEMM: epilogues and the on-chip kernel's transform wait as warps."""
    text = _source("gemm.cu")
    alone = 0
    for name in ("void run_epilogue(", "void run_epilogue_onchip("):
        body = _block(text, text.index("\n{", text.index(name)))  # behind a default argument's braces
        for single in re.finditer(r"if \(lane == 0\) (?=\{)", body):
            block = _block(body, single.end())
            alone += block.count("mbar_wait(")
            body = body.replace(block, "")
        assert "mbar_wait(" not in body and "mbar_wait_warp(" in body
        # adding partials waits lane by lane, and its callers vote
        for call in re.finditer(r"const bool ok = sk_add_pieces\([^;]*;\s*", body):
            assert body[call.end():].startswith("if (!__all_sync(0xFFFFFFFFu, ok))")
    assert alone == 1
    transform = _block(text, text.index("} else if (warp < kFirstEpilogueWarp) ") + 1)
    assert "tmem_st_32x32b_x16(" in transform
    assert "mbar_wait(" not in transform and transform.count("mbar_wait_warp(") == 2
