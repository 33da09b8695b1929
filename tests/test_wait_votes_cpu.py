"""A bounded wait that runs out in some lanes of a warp while the phase completes for the others
must not part them before the warp's next elect or TMEM load.  So in the 8-bit product one elected
lane walks the producer's and the issuer's loops, and every other wait is voted on.  It cannot be
brought about in a run; the sources are read instead."""
import re

import pytest

from test_cluster_start_cpu import kernel_body


def block_end(text, brace):
    depth, at = 1, brace + 1
    while depth:
        depth += {"{": 1, "}": -1}.get(text[at], 0)
        at += 1
    return at


@pytest.mark.parametrize("name", ["k1_fp8_skinny_kernel", "k1_fp8_wide_kernel"])
def test_waits_are_one_lanes_or_voted_on(name):
    body = kernel_body("k1_fp8_linear.cuh", name)
    elected = [(m.end(), block_end(body, m.end() - 1))
               for m in re.finditer(r"if \((?:leader && )?ring::elect_one\(\)\) \{", body)]
    assert len(elected) == 2 == len(re.findall(r"elect_one", body))  # the producer's loop and the issuer's
    for m in re.finditer(r"(?<![\w])(?:ring::)?wait\(", body):
        assert any(a <= m.start() < b for a, b in elected), body[m.start() - 60:m.start() + 60]
    for m in re.finditer(r"warp_wait\(", body):
        assert not any(a <= m.start() < b for a, b in elected)
    for a, b in elected:  # nothing that a whole warp must reach
        assert "sync" not in body[a:b] and "bar." not in body[a:b]


def test_both_ctas_of_a_pair_stay_for_their_copies():
    """A producer that stops early keeps its shared memory until its copies have landed: the pair's
    leader, whose barriers count them, and the other CTA, which has none to wait on."""
    body = kernel_body("k1_fp8_linear.cuh", "k1_fp8_wide_kernel")
    at = body.index("if (!ok && leader)")
    stay = re.match(r"if \(!ok && leader\)\s*for \([^{}]*ring::wait\([^;]*;\s*else if \(!ok\)\s*for \([^{}]*__nanosleep",
                    body[at:])
    assert stay
