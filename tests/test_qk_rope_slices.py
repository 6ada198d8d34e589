"""CPU test: the slices of heads and the workgroups of the norm and rotation's plan."""
import os
import shutil

import pytest

from tests.test_host_sanitizers import HOST, ROOT, _build_and_run


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_rope_slices_under_asan_and_ubsan(tmp_path):
    _build_and_run(tmp_path, "test_rope_slices", [os.path.join(HOST, "rope_plan.cpp"),
                                                  os.path.join(ROOT, "tests", "host", "test_rope_slices.cpp")])
