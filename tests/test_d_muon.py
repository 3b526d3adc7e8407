"""The D form of the orthogonalised update passes on what the Python form does."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_number_of_iterations_is_the_callers():
    text = open(os.path.join(ROOT, "hip", "source", "dopt", "hip", "online.d")).read()
    head = re.search(r"^Updater muon\((.*?)\)\n\{", text, flags=re.M | re.S).group(1)
    assert re.search(r"\bint iterations = 5$", head)
    assert "u.mIterations = iterations;" in text and re.search(r"^    int mIterations;$", text, flags=re.M)
    assert re.search(r"dopt_hip_muon_step\([^;]*, mIterations\)", text, flags=re.S)
