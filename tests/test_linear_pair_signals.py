"""The CTA pairs of the projection kernel signal each other's barriers from the tensor core, asynchronously: what is
signalled to a CTA has to be waited for by that CTA, or the signal may land in shared memory that is no longer
its own.  Read from the source, since a signal that comes late shows in no result."""

import re
from pathlib import Path

SOURCE = (Path(__file__).resolve().parent.parent / "okc_b200" / "csrc" / "linear.cu").read_text()


def test_signals_to_both_ctas_are_waited_for_by_both():
    body = SOURCE[SOURCE.index("linear_tall_kernel("):]
    commits = re.findall(r"pair_commit\(&?(\w+)(?:\[\w+\])?(?:, (\w+))?\)", body)
    assert {name for name, _ in commits} == {"empty", "accf", "drain"}
    # roles of the leading CTA alone: what lies between its issuing branch and the next role
    leader = body[body.index("warp == 1 && lane == 0 && rank == 0"):body.index("setmaxnreg.inc")]
    others = body.replace(leader, "")
    for name, who in commits:
        waits = re.findall(r"mbar_wait\(&?" + name + r"\b", others)
        assert who == "kLeader" or waits, f"{name} is signalled in a CTA that does not wait for it"
