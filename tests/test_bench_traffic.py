"""The counter figure of the headline kernel's traffic, without a GPU: it belongs
to the sources that the kernel and its streams are built from, and to no others."""
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def bench():
    sys.path.insert(0, ROOT)
    import bench
    return bench


def test_the_figure_belongs_to_these_sources(bench):
    """The line of the default tiling carries it: a change of the kernel's
    sources asks for a new measurement."""
    traffic, note = bench.pmc_traffic(*bench.DEFAULT_TILING, "refill", bench.gemv_source_hash())
    assert traffic, note


def test_other_files_of_the_library_leave_it_alone(bench, monkeypatch, tmp_path):
    more = tmp_path / "more.hip"
    more.write_text("// another operator")
    before = bench.gemv_source_hash(), bench.library_source_hash()
    monkeypatch.setattr(bench.rans, "SOURCES", bench.rans.SOURCES + [str(more)])
    assert bench.gemv_source_hash() == before[0] and bench.library_source_hash() != before[1]
    monkeypatch.setattr(bench.B, "GEMV_SOURCES", bench.B.GEMV_SOURCES + [str(more)])
    assert bench.gemv_source_hash() != before[0]


def test_the_files_are_the_kernels(bench):
    """Every file of the library that the GEMV's translation unit includes, and
    the encoder of its streams."""
    import re
    names = {os.path.basename(p) for p in bench.B.GEMV_SOURCES}
    seen = {"w64_host.cpp"}
    todo = [os.path.join(bench.rans.CSRC, "rans_gemv.hip")]
    while todo:
        path = todo.pop()
        seen.add(os.path.basename(path))
        for name in re.findall(r'#include "([^"]+)"', open(path).read()):
            there = os.path.normpath(os.path.join(os.path.dirname(path), name))
            if os.path.basename(there) not in seen:
                todo.append(there)
    assert names == seen
