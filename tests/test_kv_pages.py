"""Runs tests/cpp/test_pages.cpp, the CPU test of the key/value cache's page bookkeeping, as built and under
AddressSanitizer and UndefinedBehaviorSanitizer, and checks what the C entry points refuse without a GPU."""
import ctypes
import os
import subprocess

import pytest

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "bin")


@pytest.mark.parametrize("name", ["test_pages", "asan_test_pages"])
def test_page_bookkeeping(name):
    exe = os.path.join(BIN, name)
    if not os.path.exists(exe):
        pytest.fail(f"{exe} is missing: build with `make -C tests/cpp` (or __graft_entry__.build())")
    p = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "all checks passed" in p.stdout, p.stdout + p.stderr


def test_null_arguments_are_refused(cvs):
    lib = cvs.load()
    bad = cvs.CVS_ERR_INVALID_ARGUMENT
    h = ctypes.c_void_p()
    one = (ctypes.c_int64 * 1)(1)
    view = cvs.Heads()
    assert lib.cvs_context_create_on_stream(0, None, None) == bad
    assert lib.cvs_prompt_plan_create(None, one, None, 1, 1, 1, 1, ctypes.byref(h)) == bad
    assert lib.cvs_prompt_attention_async(None, None, view, view, view, view, None, 0.0) == bad
    assert lib.cvs_kv_cache_create(None, 1, 1, 32, 1, 64, 0, ctypes.byref(h)) == bad
    assert lib.cvs_kv_cache_pages(None, None, None) == bad
    assert lib.cvs_kv_sequence_create(None, 1, one) == bad
    assert lib.cvs_kv_sequence_fork(None, 1, -1, 1, one) == bad
    assert lib.cvs_kv_sequence_extend(None, one, one, 1) == bad
    assert lib.cvs_kv_sequence_truncate(None, 1, 0) == bad
    assert lib.cvs_kv_sequence_free(None, one, 1) == bad
    assert lib.cvs_kv_sequence_pages(None, one, 1, None, None, 0, None) == bad
    assert lib.cvs_kv_cache_compact(None, None) == bad
    assert lib.cvs_kv_plan_create(None, one, one, 1, 0, ctypes.byref(h)) == bad
    assert lib.cvs_kv_write_async(None, None, 0, 1, view, 0, view, 0) == bad
    assert lib.cvs_kv_read_async(None, None, 0, 1, view, 0, view, 0) == bad
    assert lib.cvs_kv_attention_async(None, None, 0, view, view, None, 0.0) == bad
    assert "null" in lib.cvs_last_error().decode()
    for destroy in (lib.cvs_prompt_plan_destroy, lib.cvs_kv_cache_destroy, lib.cvs_kv_plan_destroy):
        assert destroy(None) == cvs.CVS_OK
