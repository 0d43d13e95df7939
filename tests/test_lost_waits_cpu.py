"""CPU tests, on the source, of what kernels leave behind a wait that ran out.

A partial tile lies where the operands' ring was, and copies to the ring may still be
under way when the epilogue's wait has run out: NaN that is stored at once may be
overwritten by them and read as numbers.  So it is stored behind the block's barrier, at
which the producer has waited for its copies, or the loss is told by a flag."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fusiongpu_b200", "csrc")


def _kernel(file, name):
    """The kernel's text, comments left out."""
    s = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, file)).read())
    start = re.search(r"\s" + name + r"\(const", s).start()
    depth, i = 0, s.index("{", start)
    for j in range(i, len(s)):
        depth += {"{": 1, "}": -1}.get(s[j], 0)
        if depth == 0:
            return s[i:j]
    raise AssertionError(name)


def _products(file, name, word="lost"):
    k = _kernel(file, name)
    told = k.index(word + " = !ok")
    barrier = k.index(f"__syncthreads_or({word})", told)
    cluster = k.index("tc::cluster_sync()", barrier)
    filled = k.index("part[i] = NAN", barrier)
    assert told < barrier < filled < cluster
    assert "NAN" not in k[:barrier], "NaN stored while copies may be under way"
    wait = k.index("if (!ok)", k.index("tma_load_3d"))
    assert re.search(r"mbar_wait\(&full", k[wait:told]), "the producer waits for its copies"


def test_orthogonalised_update():
    _products("orth.cu", "orth_product_kernel")


def test_split_tiles_of_the_linear_and_gated_layers():
    _products("linear_tc.cu", "gemm_split_kernel", "gone")
    k = _kernel("linear_tc.cu", "gemm_split_kernel")  # integer sums have no NaN: a flag, which all of the cluster read
    assert "if (MODE == TC_INT8 && !ok) s_lost = 1;" in k and "if (lost) z = make_float4(NAN, NAN, NAN, NAN);" in k


def test_one_launch_update_ends_with_nothing_under_way():
    k = _kernel("orth.cu", "orth_small_kernel")
    for bar in ("&done", "&copied"):
        assert f"landed({bar}" in k
    assert k.count("mbar_wait_warp(") == 1  # landed's own
    assert re.search(r"auto landed = .*?mbar_wait_warp\(bar, parity, fail\)\) return true;\s*tc::mbar_wait\(bar, parity\);", k, re.S)
