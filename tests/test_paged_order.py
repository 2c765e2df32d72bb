"""Orders between the warps of the kernels of attention over a block table that no run shows reliably, read from their sources."""
import os
import re

from helpers import ROOT


def _source(name):
    with open(os.path.join(ROOT, "sparse_mla_sm120_b200", "csrc", name)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    return text


def _softmax(text):
    """The softmax role's code, up to the next role."""
    return text[text.index("if (warp < P"):text.index("} else if (warp < P" if "} else if (warp < P" in text else "} else if (warp < S_WARP")]


def test_products_wait_for_every_warp_that_rescales():
    """paged_pair.cu: the products of a half of a block's rows add to all lanes of the accumulator.  A warp of the other half that still
    rescales would lose them: between the rescaling's last store and the hand-over of weights, all four warps of a row meet."""
    body = _softmax(_source("paged_pair.cu"))
    rescaled = body[body.index("tmem_wait_st();"):body.index("mbar_arrive_remote(p_ready)")]
    order = [rescaled.index(w) for w in ("tmem_wait_st();", "tc_fence_before();", "named_bar_or(1 + grp, 128, dead)", "tc_fence_after();")]
    assert order == sorted(order)
    # no way past it: a warp whose wait gave up takes part
    rescale = body[body.index("named_bar_or(1 + grp, 128, mx > m"):body.index("const float mm")]
    assert "continue" not in rescale
