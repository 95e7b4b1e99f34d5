"""Distributed shared memory may be touched only once every CTA of the cluster
runs.  What that takes is visible in a kernel's source alone: a write that comes
too early need not show in any output."""
import os
import re

import aceflow_b200

CSRC = os.path.join(os.path.dirname(aceflow_b200.__file__), "csrc")


def _body(source, kernel):
    at = source.index(kernel + "(SampleParams p) {")
    return re.sub(r"//[^\n]*", "", source[at:source.index("\n}\n", at)])


def test_the_draw_waits_for_its_cluster_before_the_first_exchange():
    with open(os.path.join(CSRC, "sample_tokens.cu")) as f:
        body = _body(f.read(), "sample_tokens_kernel")
    # what reaches another CTA's memory: exchange, and what calls it
    first = min(m.start() for m in re.finditer(r"\b(?:row\.(?:largest|exchange|total|bring|run_bins|from_first)|token_at"
                                               r"|descend|far64|far32|put_far64|in_cta)\(", body))
    said, waited = body.find("cluster_started();"), body.find("cluster_all_started();")
    assert 0 <= said < waited < first
    assert "return" not in body[:waited].split("auto keep")[0], "every thread arrives and waits"
