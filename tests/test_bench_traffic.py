"""CPU checks of what a recorded traffic measurement is tied to."""
import os
import shutil
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
bench = pytest.importorskip("bench")


@pytest.fixture
def csrc(tmp_path, monkeypatch):
    """A copy of the kernel sources that bench.py looks at instead."""
    at = tmp_path / "torch_npu_ops_amd" / "csrc"
    shutil.copytree(os.path.join(bench.REPO, "torch_npu_ops_amd", "csrc"), at)
    monkeypatch.setattr(bench, "REPO", str(tmp_path))
    monkeypatch.setattr(bench, "CSRC", str(at), raising=False)
    return at


def _append(path):
    path.write_text((path.read_text() if path.exists() else "") + "// more\n")


def test_another_kernels_header_leaves_a_measurement_valid(csrc):
    before = {f: bench.source_sha(f) for f in ("norm.hip", "rope.hip", "gdn_chunk.hip")}
    _append(csrc / "residual_norm.h")
    _append(csrc / "a_new_kernel.h")
    assert {f: bench.source_sha(f) for f in before} == before


@pytest.mark.parametrize("source, header", [("norm.hip", "norm.hip"), ("norm.hip", "xk_common.h"),
                                            ("gdn_chunk.hip", "gdn_common.h"),
                                            ("gdn_chunk.hip", "xk_common.h"),
                                            ("residual_norm_f16.hip", "residual_norm.h")])
def test_a_kernels_own_files_do_not(csrc, source, header):
    before = bench.source_sha(source)
    _append(csrc / header)
    assert bench.source_sha(source) != before
