"""A block may touch another block's shared memory only once that block is known to run, which
a cluster barrier shows.  A kernel that does it too early is right as long as its own work in
front takes longer than the other block's start, so no run can show the fault: the order is
read from the sources.
"""
import os
import re

import pytest

from conftest import PKG_ROOT

REMOTE = re.compile(r"shared::cluster\.|\bmapa\(|arrive_remote\(|tma_load_2d_pair_at\(|umma_commit_pair\w*\(|"
                    r"\bexchange<|\brow_bin\(|\bjoin_lists\(|\btell\(")
BARRIER = re.compile(r"ring::cluster_(sync|wait)\(\)")


def kernel_body(source, name):
    text = open(os.path.join(PKG_ROOT, "csrc", source)).read()
    text = re.sub(r"//[^\n]*", "", text)
    at = re.search(r"__launch_bounds__\([^{;]*\b" + name + r"\([^{]*\{", text).end()
    depth, end = 1, at
    while depth:
        depth += {"{": 1, "}": -1}.get(text[end], 0)
        end += 1
    return text[at:end]


@pytest.mark.parametrize("source,name", [("k1_sample.cuh", "k1_sample_kernel"),
                                         ("k1_fp8_linear.cuh", "k1_fp8_skinny_kernel"),
                                         ("k1_fp8_linear.cuh", "k1_fp8_wide_kernel")])
def test_a_cluster_barrier_comes_before_the_first_remote_access(source, name):
    body = kernel_body(source, name)
    remote, barrier = REMOTE.search(body), BARRIER.search(body)
    assert remote and barrier, name
    assert barrier.start() < remote.start(), f"{name}: {remote.group()} before any cluster barrier"
    if barrier.group(1) == "wait":  # its other half, before that
        assert 0 <= body.find("ring::cluster_arrive()") < barrier.start()
