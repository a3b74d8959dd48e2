"""Cross attention to encoder states of different lengths, against float64
(tests/paged_float64.py; here every value is held as f16)."""

import numpy as np
import pytest

from tests import paged_float64 as P
from tests.device_memory import Device
from tests.test_paged_gpu import flat, near, queries, rows_of, same
from trit_amd import hip

pytestmark = pytest.mark.gpu


def states(hd, kvh, keys, max_keys=None, layers=1, seed=50):
    c = hip.CrossStates(layers, kvh, hd, len(keys), max_keys or max(max(keys), 1))
    data = [rows_of(seed + 3 * i, n, kvh, hd) for i, n in enumerate(keys)]
    for layer in range(layers):
        c.set(layer, np.arange(len(keys)), keys, np.concatenate([k for k, _ in data]),
              np.concatenate([v for _, v in data]))
    return c, data


def check(c, data, slots, rows, heads, scale=0.0, layer=0, q=None, what=""):
    hd = c.head_dim
    if q is None:
        q = queries(60, int(sum(rows)), heads, hd)
    got = c.attention(layer, slots, rows, q, heads, scale).reshape(-1, heads, hd)
    at = 0
    for s, n in zip(slots, rows):
        k, v = (P.f16(x) for x in data[s])
        want, off = P.attention(q[at:at + n], k, v, [len(k)] * n,
                                scale or float(np.float32(1.0) / np.sqrt(np.float32(hd))))
        near(got[at:at + n], want, off, f"{what} slot {s} of {len(k)} keys, {n} rows")
        at += n
    return got


# (head_dim, heads, kv_heads, keys of each slot, the slots asked, rows of each)
SHAPES = [
    (64, 20, 20, [1500], [0], [5]),  # Whisper large-v3, 5 beams
    (64, 6, 6, [1, 63, 64, 65, 128, 0, 700], [0, 1, 2, 3, 4, 5, 6], [1] * 7),
    (128, 16, 8, [130, 33], [1, 0, 1], [2, 1, 3]),
    (64, 2, 2, [70, 200], [1, 0], [40, 17]),
    (80, 6, 3, [129], [0], [9]),
    (40, 4, 4, [10, 20], [0, 1], [1, 0]),
    (1, 1, 1, [3], [0], [1]),
    (128, 24, 1, [900], [0], [2]),
]


@pytest.mark.parametrize("hd,heads,kvh,keys,slots,rows", SHAPES)
def test_cross_attention(gpu, hd, heads, kvh, keys, slots, rows):
    print(f"case cross hd={hd} heads={heads}/{kvh} keys={keys} slots={slots} rows={rows}", flush=True)
    c, data = states(hd, kvh, keys)
    got = check(c, data, slots, rows, heads, what="cross")
    at = 0
    for s, n in zip(slots, rows):
        if not keys[s]:
            assert (got[at:at + n] == 0).all()
        at += n
    assert [c.keys(s) for s in range(len(keys))] == keys


def test_slots_take_new_states(gpu):
    """Shorter states over longer ones, of other layers and other slots none."""
    print("case new states", flush=True)
    c, data = states(64, 2, [100, 300, 64], max_keys=320, layers=2)
    k, v = rows_of(90, 75, 2, 64)
    k[0, 0, 0] = v[1, 1, 1] = np.nan  # held where it is, and gone with the next
    c.set(1, [1], [75], k, v)
    got = c.attention(1, [1], [1], queries(1, 1, 2, 64), 2).reshape(2, 64)
    assert np.isnan(got[0]).all() and np.isnan(got[1, 1]) and np.isfinite(np.delete(got[1], 1)).all()
    k, v = rows_of(91, 70, 2, 64)
    c.set(1, [1], [70], k, v)
    check(c, data, [0, 1, 2], [1, 1, 1], 2, layer=0, what="layer 0")
    check(c, [data[0], (k, v), data[2]], [0, 1, 2], [1, 1, 1], 2, layer=1, what="layer 1")
    c.set(1, [2, 0], [0, 0], k[:0], v[:0])
    assert c.keys(2, 1) == 0
    assert (c.attention(1, [2], [1], queries(1, 1, 2, 64), 2) == 0).all()


def test_cross_scales_and_magnitudes(gpu):
    print("case cross magnitudes", flush=True)
    c, data = states(64, 2, [200])
    for scale in (30.0, 1e-7, 0.5):
        check(c, data, [0], [3], 4, scale=scale, what=f"scale {scale}")
    k, v = rows_of(70, 130, 1, 64)
    k[:64] *= 1e-7
    v[64:] *= 6e-8
    v[100] = 65504.0
    one = hip.CrossStates(1, 1, 64, 1, 130)
    one.set(0, [0], [130], k, v)
    q = queries(71, 4, 1, 64)
    q[0], q[1] = 0.0, q[1] * 1e-25
    check(one, [(k, v)], [0], [4], 1, q=q, what="magnitudes")


def test_cross_device_rows(gpu):
    """Keys and values side by side in one projection's rows, queries in theirs, beams of several audios."""
    print("case cross device rows", flush=True)
    hd, kvh, heads, keys, rows = 64, 4, 4, [90, 150], [5, 5]
    c = hip.CrossStates(2, kvh, hd, 2, 150)
    data = [rows_of(80 + i, n, kvh, hd) for i, n in enumerate(keys)]
    width, total = kvh * hd, sum(keys)
    kv = np.concatenate([np.concatenate([flat(x) for x in (k, v)], axis=1) for k, v in data])
    q = queries(82, 10, heads, hd)
    hq = np.full((10, heads * hd + 3), np.nan, np.float32)
    hq[:, 3:] = q.reshape(10, -1)
    D = Device()
    try:
        dkv, dq, out = D.upload(kv), D.upload(hq), D.upload(np.full((11, heads * hd), 7.0, np.float32))
        assert kv.shape == (total, 2 * width)
        c.set_device(1, [0, 1], keys, dkv.value, 2 * width, dkv.value + 4 * width, 2 * width)
        c.attention_device(1, [0, 1], rows, dq.value + 12, heads * hd + 3, heads, out)
        got = D.download(out, (11, heads * hd))
    finally:
        D.free()
    assert (got[10] == 7.0).all()
    assert same(got[:10], c.attention(1, [0, 1], rows, q, heads))
    check(c, data, [0, 1], rows, heads, layer=1, q=q, what="device rows")


def test_cross_many_slots(gpu):
    print("case cross 200 slots", flush=True)
    keys = [(29 * i) % 90 for i in range(200)]
    c, data = states(64, 1, keys)
    slots = np.random.default_rng(1).permutation(200)[:170]
    check(c, data, slots, [1 + int(s) % 2 for s in slots], 2, what="many slots")


def test_cross_refusals(gpu):
    print("case cross refusals", flush=True)
    c, _ = states(64, 2, [10, 20], max_keys=30, layers=2)
    x = np.zeros((200, 2, 64), np.float32)
    for what, call in [
        ("slot 2", lambda: c.set(0, [2], [1], x[:1], x[:1])),
        ("slot -1", lambda: c.attention(0, [-1], [1], x[:1], 2)),
        ("layer 2", lambda: c.set(2, [0], [1], x[:1], x[:1])),
        ("twice", lambda: c.set(0, [1, 1], [1, 1], x[:2], x[:2])),
        ("31 keys", lambda: c.set(0, [1], [31], x[:31], x[:31])),
        ("negative", lambda: c.set(0, [0, 1], [2, -1], x[:1], x[:1])),
        ("evenly", lambda: c.attention(0, [0], [1], np.zeros((1, 3 * 64), np.float32), 3)),
        ("scale", lambda: c.attention(0, [0], [1], x[:1], 2, scale=float("inf"))),
        ("stride", lambda: c.set_device(0, [0], [1], 64, 127, 64, 128)),
        ("NULL", lambda: c.set_device(0, [0], [1], None, 128, 64, 128)),
        ("counts", lambda: c.set(0, [0, 1], [1], x[:1], x[:1])),
        ("values", lambda: c.attention(0, [0], [2], x[:1], 2)),
    ]:
        with pytest.raises(hip.TritError, match=what):
            call()
    fresh = hip.CrossStates(1, 2, 64, 2, 30)
    with pytest.raises(hip.TritError, match="never set"):
        fresh.attention(0, [1], [1], x[:1], 2)
    assert [c.keys(0), c.keys(1)] == [10, 20]
    assert c.attention(0, [0], [0], x[:0], 2).shape == (0, 128)


def sampled(got, data, slots, rows, heads, q, what):
    """Some rows of each slot against float64: the ends, tile borders, and others."""
    hd = q.shape[2]
    scale = float(np.float32(1.0) / np.sqrt(np.float32(hd)))
    r = np.random.default_rng(3)
    at = 0
    for s, n in zip(slots, rows):
        pick = sorted({0, n - 1, min(15, n - 1), min(16, n - 1), min(63, n - 1), *r.integers(0, n, 12).tolist()})
        k, v = (P.f16(x) for x in data[s])
        idx = at + np.array(pick)
        want, off = P.attention(q[idx], k, v, [len(k)] * len(pick), scale)
        near(got[idx], want, off, f"{what} slot {s} of {len(k)} keys, {n} rows")
        at += n


# Calls of many columns a slot, and some of few beside them.
MANY = [
    (64, 64, 8, [70, 129, 0], [1, 0, 2], [400, 3, 70]),
    (128, 32, 4, [65], [0], [900]),
    (80, 24, 3, [130, 1], [0, 1], [900, 129]),
    (40, 20, 20, [64, 200], [1, 0, 1], [700, 600, 65]),
]


@pytest.mark.parametrize("hd,heads,kvh,keys,slots,rows", MANY)
def test_cross_many_rows(gpu, hd, heads, kvh, keys, slots, rows):
    print(f"case cross many rows hd={hd} heads={heads}/{kvh} keys={keys} rows={rows}", flush=True)
    c, data = states(hd, kvh, keys)
    q = queries(61, sum(rows), heads, hd)
    got = c.attention(0, slots, rows, q, heads).reshape(-1, heads, hd)
    assert np.isfinite(got).all()
    sampled(got, data, slots, rows, heads, q, "many rows")


def test_cross_many_rows_of_every_size(gpu):
    """The many-row kernel with scores that rise from block to block, a sink, tiny and huge values, and queries that
    are 0, NaN or infinite."""
    print("case cross many rows, sizes", flush=True)
    hd, heads, kvh, n = 64, 64, 8, 400
    k, v = rows_of(75, 300, kvh, hd)
    k *= np.linspace(0.05, 6.0, 300).astype(np.float32)[:, None, None]  # each block's largest score far above the last's
    k[10, 0] *= 1e4
    v[:64] *= 6e-8
    v[200:210] = 65504.0
    c = hip.CrossStates(1, kvh, hd, 1, 300)
    c.set(0, [0], [300], k, v)
    q = queries(76, n, heads, hd)
    q[5], q[6] = 0.0, q[6] * 1e-25
    q[7, 3, 1], q[8, 9, 0] = np.nan, -np.inf
    got = c.attention(0, [0], [n], q, heads).reshape(n, heads, hd)
    bad = np.zeros((n, heads), bool)
    bad[7, 3] = bad[8, 9] = True
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
    pick = np.array([0, 5, 6, 9, 100, 255, 399])
    want, off = P.attention(q[pick], P.f16(k), P.f16(v), [300] * len(pick), 0.125)
    near(got[pick], want, off, "sizes")
    v[130, 2, 9] = np.nan
    c.set(0, [0], [300], k, v)
    again = c.attention(0, [0], [n], q, heads).reshape(n, heads, hd)
    nan = np.isnan(again) & ~np.isnan(got)
    assert nan[:, 16:24, 9][~bad[:, 16:24]].all() and nan.sum() == (~bad[:, 16:24]).sum()
