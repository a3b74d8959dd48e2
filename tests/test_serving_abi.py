"""Refusals of the calls for many sequences on a host without a GPU."""

import ctypes as C

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
