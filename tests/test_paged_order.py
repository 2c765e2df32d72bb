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


def test_waits_ask_for_a_phase_next_to_one_that_is_over():
    """paged_pair.cu: a parity is that of a phase and of the one two phases earlier.  A warp may wait for a barrier only where it knows the
    phase before to be over: those that softmax warps wait for in every block are, and the others' (half 1 of V, for the warps of half 0)
    only behind a barrier that the warps of half 1 have passed too."""
    body = _softmax(_source("paged_pair.cu"))
    meets = [m.start() for m in re.finditer(r"named_bar_or\(1 \+ grp, 128", body)]
    waits = re.findall(r"mbar_wait_lean\(bar\((PB_\w+)([^)]*)\)", body)
    assert waits and {w for w, _ in waits} <= {"PB_SREADY", "PB_VFREE", "PB_VFULL"}
    for m in re.finditer(r"mbar_wait_lean\(bar\(PB_VFREE \+ 1\)", body):
        # the last thing before it that several warps do together, or wait for, is a meeting of the four
        before = body[:m.start()]
        assert max(i for i in meets if i < m.start()) > before.rindex("mbar_wait_lean")
    # nothing is read from the accumulator in the epilogue before all four warps have waited
    epilogue = body[body.rindex("mbar_wait_lean(bar(PB_VFREE + 1)"):]
    assert epilogue.index("named_bar_or(1 + grp, 128, dead)") < epilogue.index("tc_fence_after();") < epilogue.index("tmem_ld32(")


def test_who_stores_which_rows_are_there_hands_it_over():
    """The lane that stores a block's validity arrives on the barrier that makes it readable: either one elected lane does both, or lane 0
    does, behind the warp's other stores."""
    for name, at in (("paged.cu", "GV_OFF"), ("paged_pair.cu", "PPY_OFF")):
        text = _source(name)
        stores = [m.start() for m in re.finditer(r"\(sm \+ " + at + r"[^;]*\) = ", text)]
        assert stores
        for i in stores:
            elected, lane0 = text.rfind("if (elect_one()) {", 0, i), text.rfind("if (lane == 0)", 0, i)
            arrive = re.compile(r"mbar_arrive\w*\(").search(text, i).start()
            if elected > lane0:
                assert "}" not in text[elected:arrive], name
            else:
                assert "elect_one" not in text[i:arrive] and "if (lane == 0) mbar_arrive(" in text[i:arrive + 12], name
