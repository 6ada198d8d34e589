"""CPU test: one address for what forking and compacting write and for something else, refused by the C ABI."""
import os
import shutil

import pytest

from tests.test_host_sanitizers import HOST, ROOT, _build_and_run


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_pages_aliases_under_asan_and_ubsan(tmp_path):
    _build_and_run(tmp_path, "test_pages_aliases", [os.path.join(HOST, n) for n in (
        "fgqa_plan.cpp", "kv_plan.cpp", "pages_plan.cpp")] + [os.path.join(ROOT, "tests", "host", "test_pages_aliases.cpp")])
