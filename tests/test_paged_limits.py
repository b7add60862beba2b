"""The largest sizes of paged attention's launch arithmetic: no signed overflow in
what the host bounds (also run against the host-sanitized library) nor in what
the kernels share with it."""

from __future__ import annotations

import subprocess
import sys

import pytest

from legolink_amd import _native, build
from legolink_amd.paged_attention import PagedAttentionError, paged_attention
from tests import test_host_sanitizer as sanitizer
from tests.test_paged_attention import _arguments, _block
from tests.test_step_calls import _attend


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


@pytest.mark.parametrize("scale", [5e-324, 1e-46, 1e-40, 9e-38])
def test_scales_that_fp32_does_not_hold_are_refused(scale):
    """The kernels' scale and the maximum's slack over it are normal fp32 numbers."""

    with pytest.raises(_native.NativeCallError, match="softmax_scale") as error:
        _native.paged_attention_workspace_bytes(_block(softmax_scale=scale))
    assert error.value.reason == "invalid_argument"
    with pytest.raises(PagedAttentionError, match="scale"):
        paged_attention(**_arguments(), scale=scale)
    assert _attend({**_arguments(), "scale": scale}) is None


@pytest.mark.parametrize("scale", [1e-37, 1e-30, 9e29])
def test_scales_that_it_holds_are_taken(scale):
    assert _native.paged_attention_workspace_bytes(_block(softmax_scale=scale)) > 0
    with pytest.raises(PagedAttentionError, match="device tensors are required"):
        paged_attention(**_arguments(), scale=scale)
    assert _attend({**_arguments(), "scale": scale}) is True
