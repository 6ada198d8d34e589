"""CPU test: the eviction's sequence and new-page limits in the C ABI's validation."""
import os
import shutil

import pytest

from tests.test_host_sanitizers import HOST, ROOT, _build_and_run


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_limits_under_asan_and_ubsan(tmp_path):
    _build_and_run(tmp_path, "test_kv_evict_tokens",
                   [os.path.join(HOST, "fgqa_plan.cpp"), os.path.join(HOST, "kv_plan.cpp"),
                    os.path.join(ROOT, "tests", "host", "test_kv_evict_tokens.cpp")])
