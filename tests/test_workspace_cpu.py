"""Refusals of the entry points for workspaces of captures, error words and the counter wait, before any
device is touched."""
import ctypes

import pytest

from nanovllm_b200 import _lib

P = 4096                                          # an aligned address: never read


def test_capture_id_needs_a_destination():
    assert _lib.lib.fp8attn_capture_id(None, None) == _lib.EINVAL
    assert _lib.lib.fp8attn_last_error()


@pytest.mark.parametrize("mode", [-1, 3, 1 << 20])
def test_capture_modes_are_the_runtime_s(mode):
    m = ctypes.c_int(mode)
    assert _lib.lib.fp8attn_exchange_capture_mode(ctypes.byref(m)) == _lib.EINVAL
    assert m.value == mode
    assert _lib.lib.fp8attn_exchange_capture_mode(None) == _lib.EINVAL


def test_error_word_needs_a_destination():
    assert _lib.lib.fp8attn_fp8_moe_read_error(None, 1, None) == _lib.EINVAL


@pytest.mark.parametrize("bad", [(None, 1, 1000, P), (P, 1, 1000, None), (P, 1, -1, P)])
def test_counter_wait_rejects(bad):
    assert _lib.lib.fp8attn_diag_counter_wait(*bad, 0, None) == _lib.EINVAL
