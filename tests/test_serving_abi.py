"""Refusals of the calls for many sequences on a host without a GPU."""

import ctypes as C

import numpy as np
import pytest

from trit_amd import hip


def test_serving_calls_refuse_before_a_device_is_needed():
    """The paged cache's and cross attention's NULL handles and shapes."""
    lib = hip.lib()
    out, none = C.c_void_p(), None
    ids = (C.c_int32 * 1)(0)
    for call in (
        lambda: lib.trit_hip_paged_open(none, 1, ids),
        lambda: lib.trit_hip_paged_fork(none, ids, 1, ids, none),
        lambda: lib.trit_hip_paged_reorder(none, ids, ids, 1, none),
        lambda: lib.trit_hip_paged_copy(none, ids, 1, none, ids, none),
        lambda: lib.trit_hip_paged_close(none, ids, 1),
        lambda: lib.trit_hip_paged_compact(none, none),
        lambda: lib.trit_hip_paged_resize(none, 1, none),
        lambda: lib.trit_hip_paged_length(none, 0, 0),
        lambda: lib.trit_hip_paged_info(none, none, none, none),
        lambda: lib.trit_hip_paged_append(none, 0, ids, ids, 1, none, none),
        lambda: lib.trit_hip_paged_append_device(none, 0, ids, ids, 1, none, 64, none, 64, none),
        lambda: lib.trit_hip_paged_read(none, 0, ids, ids, ids, 1, none, none),
        lambda: lib.trit_hip_paged_read_device(none, 0, ids, ids, ids, 1, none, 64, none, 64, none),
        lambda: lib.trit_hip_paged_attention(none, 0, ids, ids, 1, none, 1, 0.0, none),
        lambda: lib.trit_hip_paged_attention_device(none, 0, ids, ids, 1, none, 64, 1, 0.0, none, none),
        lambda: lib.trit_hip_cross_set(none, 0, ids, ids, 1, none, none),
        lambda: lib.trit_hip_cross_set_device(none, 0, ids, ids, 1, none, 64, none, 64, none),
        lambda: lib.trit_hip_cross_keys(none, 0, 0),
        lambda: lib.trit_hip_cross_attention(none, 0, ids, ids, 1, none, 1, 0.0, none),
        lambda: lib.trit_hip_cross_attention_device(none, 0, ids, ids, 1, none, 64, 1, 0.0, none, none),
        lambda: lib.trit_hip_paged_new(1, 1, 64, 1, 1, None),
        lambda: lib.trit_hip_cross_new(1, 1, 64, 1, 1, None),
    ):
        assert call() == -1
        assert b"NULL" in lib.trit_hip_last_error()
    for shape in ((0, 1, 64, 1, 1), (1, 0, 64, 1, 1), (1, 1, 0, 1, 1), (1, 1, 129, 1, 1), (1, 1, 64, 0, 1),
                  (1, 1, 64, 1, 0), (1, 1, 64, 1 << 27, 1), (1, 1, 64, 1, 1 << 27), (-1, 1, 64, 1, 1)):
        if shape[3:] != (1 << 27, 1):
            assert lib.trit_hip_cross_new(*shape, C.byref(out)) == -1
            assert b"cross attention" in lib.trit_hip_last_error()
        assert lib.trit_hip_paged_new(*shape, C.byref(out)) == -1
        assert b"paged cache" in lib.trit_hip_last_error()
    lib.trit_hip_paged_free(None)
    lib.trit_hip_cross_free(None)


def test_states_past_64_bits_are_refused():
    """Sizes whose bytes, counted in 64 bits, come out as few or none."""
    lib, out = hip.lib(), C.c_void_p()
    for shape in ((1, 1 << 15, 64, 1 << 20, 1 << 26), (1, 1 << 15, 64, 1 << 20, (1 << 26) - 63),
                  (1 << 16, 65535, 128, 1 << 20, 1 << 26), (1 << 13, 1 << 13, 128, 1 << 13, 1 << 16)):
        assert lib.trit_hip_cross_new(*shape, C.byref(out)) == -1
        assert b"memory" in lib.trit_hip_last_error(), (shape, lib.trit_hip_last_error())


def test_ids_and_counts_are_32_bit_integers():
    """A value that 32 bits would change names no other sequence."""
    for values in ([1 << 31], [-(1 << 31) - 1], np.array([1 << 32]), np.array([3], np.uint64) << 40, [0.5], [1.0],
                   [True], ["1"], [None]):
        with pytest.raises(hip.TritError, match="integers"):
            hip._ids(values)
    for values in ([], np.zeros(0), [3, 1], (3, 1), np.array([3, 1]), np.array([[3], [1]], np.uint8),
                   np.array([3, 9, 1], np.int32)[::2]):
        got = hip._ids(values)
        assert got.dtype == np.int32 and got.flags.c_contiguous and got.tolist() in ([], [3, 1])


def test_no_copy_into_a_freed_cache():
    """A freed cache is not taken for the cache's own (NULL)."""
    a, b = (hip.PagedCache.__new__(hip.PagedCache) for _ in range(2))
    a.h = b.h = None
    with pytest.raises(hip.TritError, match="freed"):
        a.copy([0], into=b)
