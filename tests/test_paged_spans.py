"""What the merge of attention over a block table makes of a request's span: partitions of a wait that gave up leave none, and what the
scratch held before must not lead it outside of the records."""
import os
import re
import subprocess

from helpers import ROOT

CSRC = os.path.join(ROOT, "sparse_mla_sm120_b200", "csrc")


def test_spans_stay_within_the_records(tmp_path):
    exe = str(tmp_path / "spans")
    subprocess.run(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-I" + CSRC, "-o", exe, os.path.join(ROOT, "tests", "spans.cu")], check=True)
    assert subprocess.run([exe]).returncode == 0


def test_the_merge_reads_spans_in_this_way_alone():
    with open(os.path.join(CSRC, "paged.cu")) as f:
        kernel = f.read().split("paged_combine_kernel(const PagedParams p) {")[1]
    assert len(re.findall(r"span\.y", kernel)) == 1 and "span_parts(c0, (int)span.y, p.num_parts)" in kernel
    # nothing of the records is asked for before it is known to be one
    assert kernel.index("if (n <= 1) return;") < kernel.index("load(warp);")
