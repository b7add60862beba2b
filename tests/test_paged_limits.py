"""The largest sizes of paged attention's launch arithmetic: no signed overflow in
what the host bounds (also run against the host-sanitized library) nor in what
the kernels share with it."""

from __future__ import annotations

import subprocess
import sys

import pytest

from legolink_amd import _native, build
from tests import test_host_sanitizer as sanitizer
from tests.test_paged_attention import _block


@pytest.mark.parametrize("requests", [2 ** 30 - 1, 2 ** 29 + 1])
@pytest.mark.parametrize("queries", [1, 2 ** 20])
def test_more_requests_than_a_launch_holds(requests, queries):
    args = _block(num_requests=requests, num_queries=queries, query_starts=64,
                  query_starts_dtype=_native.DTYPE_INT64)
    with pytest.raises(_native.NativeCallError, match="too many queries") as error:
        _native.paged_attention_workspace_bytes(args)
    assert error.value.reason == "invalid_argument"


# A signed overflow is no constant expression: this does not compile where there is one.
_PARTS = """
#include "paged_units.h"
constexpr int kMost = 0x7fffffff;
static_assert(parts_of(0, 64) == 1 && parts_of(1, 64) == 1 && parts_of(64, 64) == 1 && parts_of(65, 64) == 2);
static_assert(parts_of(65, kOneChunk * 64) == 1 && parts_of(128, kOneChunk * 64) == 1);
static_assert(parts_of((1 << 30) - 1, kOneChunk * 64) == 1 && parts_of((1 << 30) - 1, 64) == 1 << 24);
static_assert(parts_of(kMost, kMost) == 1 && parts_of(kMost, 1) == kMost && parts_of(kMost, kMost - 1) == 2);
int main() { return 0; }
"""


def test_counting_chunks_does_not_overflow(tmp_path):
    source = tmp_path / "parts.cpp"
    source.write_text(_PARTS)
    result = subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-c", "-o", str(tmp_path / "parts.o"), str(source),
                             f"-I{build.SOURCE.parent}"], capture_output=True, text=True)
    assert result.returncode == 0, result.stderr[-3000:]


@pytest.mark.timeout(900)
def test_the_step_entries_are_clean_under_asan_and_ubsan():
    env = sanitizer._sanitizer_env()
    result = subprocess.run(
        [sys.executable, "-m", "pytest", "-q", "-x", "-m", "not gpu", "-p", "no:cacheprovider", "-k",
         "c_entry or workspace or requests_than or nothing", "tests/test_head_rotary.py", "tests/test_paged_attention.py",
         "tests/test_paged_limits.py"],
        cwd=sanitizer.REPO_ROOT, env=env, capture_output=True, text=True, timeout=840)
    output = result.stdout + result.stderr
    assert "AddressSanitizer" not in output and "runtime error:" not in output, output[-6000:]
    assert result.returncode == 0, output[-6000:]
    assert " passed" in result.stdout, output[-3000:]
