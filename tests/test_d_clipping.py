"""The D updaters refuse a largest norm that is none before they do anything, as the Python ones do."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_norm_that_is_none_is_refused_when_the_updater_is_made():
    text = open(os.path.join(ROOT, "hip", "source", "dopt", "hip", "online.d")).read()
    body = re.search(r"^    this\(Rule rule[^)]*float maxNorm\)\n    \{\n(.*?)^    \}", text, flags=re.M | re.S).group(1)
    # the first statement, whose condition a NaN does not meet either
    assert re.match(r"\s*enforce\(maxNorm >= 0, ", body)
    # every updater's norm goes through it
    assert len(re.findall(r"new FusedUpdater\(", text)) == len(re.findall(r"new FusedUpdater\(Rule\.\w+, outputs, wrt, projs, maxNorm\)", text)) == 4
