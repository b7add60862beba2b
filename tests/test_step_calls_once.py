"""A native step call that has reached the library's entry is never handed back to
the Python path, which would make it again (an in-place rotation twice): whatever
fails from there on is raised.  On the CPU, with entries that fail on purpose."""

from __future__ import annotations

import ctypes
import subprocess
import sysconfig

import pytest
import torch

from legolink_amd import _native
from tests import test_head_rotary as rotary_cases
from tests import test_paged_attention as attention_cases

_step_calls = _native.step_calls()

_ENTRIES = r"""
#include <Python.h>
#include <new>
static int calls = 0;
extern "C" {
int entry_calls() { return calls; }
int succeeds(const void *, void *) { ++calls; return 0; }
int refuses(const void *, void *) { ++calls; return -7; }
int throws(const void *, void *) { ++calls; throw std::bad_alloc(); }
int leaves_an_error(const void *, void *) { ++calls; PyErr_NoMemory(); return 0; }
long long no_workspace(const void *) { return 0; }
}
"""


@pytest.fixture(scope="module")
def entries(tmp_path_factory):
    directory = tmp_path_factory.mktemp("entries")
    source, library = directory / "entries.cpp", directory / "entries.so"
    source.write_text(_ENTRIES)
    subprocess.run(["g++", "-shared", "-fPIC", "-o", str(library), str(source),
                    f"-I{sysconfig.get_paths()['include']}"], check=True)
    return ctypes.CDLL(str(library))


def _address(entries, name):
    return ctypes.cast(getattr(entries, name), ctypes.c_void_p).value


HOST = -1  # the device index of tensors in host memory


def _calls(entries, name):
    """The three calls with this entry, on host tensors."""

    address = _address(entries, name)
    rows, _ = rotary_cases._heads()
    append, attention = rotary_cases._append(), attention_cases._arguments()
    rotary = ("query", "key", "positions", "cos_sin_cache", "rotary_dim")
    yield lambda: _step_calls.rotate_heads(address, 0, HOST, *(rows[n] for n in rotary), True, None, None, 1e-6, None,
                                           rows["query"], rows["key"])
    yield lambda: _step_calls.append(address, 0, HOST, *(append[n] for n in rotary), True, None, None, 1e-6, None, None,
                                     append["value"], append["key_buffer"], append["value_buffer"],
                                     append["destination_slots"])
    yield lambda: _step_calls.paged_attention(address, 0, HOST, _address(entries, "no_workspace"), *(
        attention[n] for n in ("query", "key_buffer", "value_buffer", "page_table", "kv_lengths", "page_size")),
        None, None)


@pytest.mark.parametrize("entry,error", [("throws", RuntimeError), ("leaves_an_error", MemoryError)])
def test_a_failure_behind_the_entry_is_raised(entries, entry, error):
    for call in _calls(entries, entry):
        before = entries.entry_calls()
        with pytest.raises(error):
            call()
        assert entries.entry_calls() == before + 1


def test_results_and_statuses(entries):
    for call, kind in zip(_calls(entries, "succeeds"), (tuple, torch.Tensor, torch.Tensor)):
        assert type(call()) is kind
    for call in _calls(entries, "refuses"):
        assert call() == -7


def test_tensors_of_another_device_are_declined(entries):
    address = _address(entries, "succeeds")
    rows, _ = rotary_cases._heads()
    before = entries.entry_calls()
    assert _step_calls.rotate_heads(address, 0, 0, rows["query"], rows["key"], rows["positions"],
                                    rows["cos_sin_cache"], 32, True, None, None, 1e-6, None, None, None) is None
    assert entries.entry_calls() == before
