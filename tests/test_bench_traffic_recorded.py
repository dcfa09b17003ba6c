"""CPU check that the recorded traffic is that of the kernels as they are: a
change to a measured kernel, or to a header that it includes, goes with a new
measurement (bench.PROFILE_COMMANDS), else bench.py reports none for it."""
import json
import os
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
bench = pytest.importorskip("bench")

with open(bench.TRAFFIC_JSON) as f:
    SOURCES = json.load(f)["sources"]
MEASURED = sorted({case.source for case in bench.CASES.values()} & set(SOURCES))


@pytest.mark.parametrize("source", MEASURED)
def test_recorded_traffic_is_the_current_kernels(source):
    assert SOURCES[source] == bench.source_sha(source)


def test_the_headline_has_measured_traffic():
    assert bench.measured_traffic(bench.CASES["layer_norm_fwd"])
