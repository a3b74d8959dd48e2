"""The paged 8-bit cache and its attention against float64 (tests/paged_float64.py)."""

import numpy as np
import pytest

from tests import paged_float64 as P
from tests.device_memory import Device
from trit_amd import hip

pytestmark = pytest.mark.gpu


def rows_of(seed, n, kvh, hd):
    """Keys with channels of different size, values around 1."""
    r = np.random.default_rng(seed)
    k = r.standard_normal((n, kvh, hd)) * np.exp(0.5 * r.standard_normal((1, kvh, hd)))
    return k.astype(np.float32), r.standard_normal((n, kvh, hd)).astype(np.float32)


def queries(seed, n, heads, hd):
    return (1.5 * np.random.default_rng(seed).standard_normal((n, heads, hd))).astype(np.float32)


def filled(hd, kvh, lens, seed=1, pages=None, sequences=None, layers=1, step=None):
    """A cache and its sequences' rows; `step`: rows a call."""
    c = hip.PagedCache(layers, kvh, hd, pages or sum(n // 64 for n in lens) + 2, sequences or len(lens))
    ids = c.open(len(lens))
    data = [rows_of(seed + 7 * i, n, kvh, hd) for i, n in enumerate(lens)]
    for layer in range(layers):
        if step is None:
            c.append(layer, ids, lens, np.concatenate([k for k, _ in data]), np.concatenate([v for _, v in data]))
            continue
        for at in range(0, max(lens), step):
            part = [(k[at:at + step], v[at:at + step]) for k, v in data]
            c.append(layer, ids, [len(k) for k, _ in part], np.concatenate([k for k, _ in part]),
                     np.concatenate([v for _, v in part]))
    return c, ids, data


def flat(rows):
    return rows.reshape(len(rows), rows.shape[1] * rows.shape[2])


def same(a, b):
    return np.array_equal(np.asarray(a, np.float32).view(np.uint32), np.asarray(b, np.float32).view(np.uint32))


def near(got, want, off, what):
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN elsewhere"
    err = np.where(np.isnan(want), 0.0, np.abs(got.astype(np.float64) - want))
    worst = np.max(err / np.maximum(off, 1e-300)) if err.size else 0.0
    print(f"{what}: at most {worst:.3f} of the bound", flush=True)
    assert (err <= off).all(), f"{what}: {worst:.3g} times the bound"


def check_attention(c, ids, data, rows, heads, scale=0.0, layer=0, seed=900, q=None, what=""):
    kvh, hd = c.kv_heads, c.head_dim
    if q is None:
        q = queries(seed, int(sum(rows)), heads, hd)
    got = c.attention(layer, ids, rows, q, heads, scale).reshape(-1, heads, hd)
    at = 0
    for i, n in enumerate(rows):
        k, v = (P.held(x) for x in data[i])
        want, off = P.attention(q[at:at + n], k, v, [len(k) - n + r + 1 for r in range(n)],
                                scale or float(np.float32(1.0) / np.sqrt(np.float32(hd))))
        near(got[at:at + n], want, off, f"{what} sequence {i} of {len(k)} tokens, {n} rows")
        at += n
    return got


@pytest.mark.parametrize("hd", [64, 128, 80, 40, 1, 127])
def test_values_held(gpu, hd):
    """Reads give the codes' values bit for bit, at any row of any block."""
    print(f"case read head_dim {hd}", flush=True)
    lens = [1, 63, 64, 65, 128, 200, 0, 321]
    c, ids, data = filled(hd, 3, lens)
    k, v = c.read(0, ids, [0] * len(lens), lens)
    want = [np.concatenate([flat(P.held(d[w])) for d in data]) for w in (0, 1)]
    assert same(k, want[0]) and same(v, want[1])
    first, rows = [0, 60, 63, 64, 5, 63, 0, 250], [1, 3, 1, 1, 100, 2, 0, 71]
    k, v = c.read(0, ids, first, rows)
    cut = [np.concatenate([flat(P.held(d[w]))[f:f + n] for d, f, n in zip(data, first, rows)])
           for w in (0, 1)]
    assert same(k, cut[0]) and same(v, cut[1])
    assert [c.length(i) for i in ids] == lens


@pytest.mark.parametrize("step", [1, 7, 64, 100])
def test_append_in_pieces(gpu, step):
    """The same values however the rows come."""
    print(f"case append by {step}", flush=True)
    lens = [150, 64, 1, 129]
    whole, ids, _ = filled(64, 2, lens)
    parts, jds, _ = filled(64, 2, lens, step=step)
    a, b = whole.read(0, ids, [0] * 4, lens), parts.read(0, jds, [0] * 4, lens)
    assert same(a[0], b[0]) and same(a[1], b[1])
    q = queries(3, 4, 4, 64)
    assert same(whole.attention(0, ids, [1] * 4, q, 4), parts.attention(0, jds, [1] * 4, q, 4))


def test_codes_at_ties(gpu):
    """Quotients that end in a half go to the even code."""
    print("case ties", flush=True)
    k = np.zeros((64, 1, 64), np.float32)
    k[0, 0, 0] = 127.0
    k[:, 0, 1:] = (np.arange(64 * 63).reshape(64, 63) % 253 - 126) * 0.5
    v = -k
    c = hip.PagedCache(1, 1, 64, 1, 1)
    ids = c.open(1)
    c.append(0, ids, [64], k, v)
    got = c.read(0, ids, [0], [64])
    assert same(got[0], P.held(k).reshape(64, -1)) and same(got[1], P.held(v).reshape(64, -1))
    # Codes that nearly tie: every f16 value below a largest one with an odd step.
    a = np.float16(100.3)
    below = np.arange(np.float16(0).view(np.uint16), a.view(np.uint16), dtype=np.uint16).view(np.float16)
    for at in range(0, below.size, 64 * 64 - 1):
        b = np.zeros(64 * 64, np.float32)
        part = below[at:at + 64 * 64 - 1].astype(np.float32)
        b[1:1 + part.size] = part
        b[0] = np.float32(a)
        one = hip.PagedCache(1, 1, 64, 1, 1)
        i = one.open(1)
        one.append(0, i, [64], b.reshape(64, 1, 64), -b.reshape(64, 1, 64))
        got = one.read(0, i, [0], [64])
        assert same(got[0], P.held(b.reshape(64, 1, 64)).reshape(64, -1))
        assert same(got[1], P.held(-b.reshape(64, 1, 64)).reshape(64, -1))


# (head_dim, heads, kv_heads, tokens of each sequence, query rows of each)
SHAPES = [
    (128, 16, 8, [700], [1]),  # Qwen3-0.6B's heads
    (128, 16, 8, [1, 2, 63, 64, 65, 127, 128, 129], [1] * 8),
    (64, 20, 20, [448, 5, 64, 300, 17], [1] * 5),  # Whisper large-v3's decoder, 5 beams
    (128, 32, 8, [90, 1300], [1, 1]),
    (64, 14, 2, [1000, 3], [1, 2]),
    (128, 8, 1, [257], [3]),
    (64, 48, 2, [130, 70], [1, 5]),  # more heads of a key head than a tile of columns
    (80, 6, 6, [100, 64], [4, 4]),
    (40, 9, 3, [77, 200], [1, 9]),
    (1, 2, 1, [65], [2]),
    (127, 3, 3, [66], [1]),
    (96, 10, 5, [64, 128, 192], [64, 128, 70]),  # prompts, whole and in part
    (128, 4, 2, [150, 321], [150, 33]),
    (64, 2, 2, [5000], [1]),
    (128, 2, 1, [4100], [2]),
]


@pytest.mark.parametrize("hd,heads,kvh,lens,rows", SHAPES)
def test_attention(gpu, hd, heads, kvh, lens, rows):
    print(f"case attention hd={hd} heads={heads}/{kvh} lens={lens} rows={rows}", flush=True)
    c, ids, data = filled(hd, kvh, lens, seed=hd + len(lens))
    check_attention(c, ids, data, rows, heads, what="attention")


# Rows enough that a workgroup takes two tiles of columns: odd numbers of tiles, sequences that ask nothing or little.
@pytest.mark.parametrize("hd,heads,kvh,lens,rows", [
    (20, 16, 8, [1300, 5, 1000, 900, 70], [1000, 0, 1000, 300, 1]),
    (128, 24, 8, [701, 690], [701, 690]),
])
def test_attention_of_many_rows(gpu, hd, heads, kvh, lens, rows):
    print(f"case attention of many rows {hd} {heads}/{kvh} lens {lens} rows {rows}", flush=True)
    c, ids, data = filled(hd, kvh, lens)
    check_attention(c, ids, data, rows, heads, what="attention of many rows")


def test_scale_and_layers(gpu):
    print("case scale, layers", flush=True)
    c, ids, data = filled(64, 2, [70, 129], layers=3)
    for layer in range(3):
        check_attention(c, ids, data, [1, 2], 4, scale=0.3, layer=layer, what=f"layer {layer}")
    # A scale that makes one key win by far, and one that makes all alike.
    check_attention(c, ids, data, [1, 2], 4, scale=40.0, what="sharp")
    check_attention(c, ids, data, [1, 2], 4, scale=1e-6, what="flat")


def test_one_large_score_among_many_small(gpu):
    """A sink: the small probabilities of the other keys still add up."""
    print("case sink", flush=True)
    k, v = rows_of(5, 6000, 1, 64)
    q = np.zeros((1, 1, 64), np.float32)
    q[0, 0, 0] = 8.0
    k[:, 0, 0] = 0.0
    k[3, 0, 0] = 17.0  # exp(-17) for each of the others
    v[3] = 0.0
    v[4:] = np.abs(v[4:])
    c = hip.PagedCache(1, 1, 64, 100, 1)
    ids = c.open(1)
    c.append(0, ids, [6000], k, v)
    got = check_attention(c, ids, [(k, v)], [1], 1, q=q, what="sink")
    kk, vv = P.held(k), P.held(v)
    want, _ = P.attention(q, kk, vv, [6000], 0.125)
    # The tail itself (2e-4): each of the 63 others in the sink's block is off by at most half a step of the fixed
    # point, 1 / (2 * 127 * 65536), relative to the sink; the other blocks' are relative to their own largest, so
    # what they add up to is off by the bound's share of itself.
    block = 63 * 0.5 / (127 * 65536) * np.max(np.abs(vv[:64]))
    assert (np.abs(got - want) < block + 1e-4 * want).all() and np.min(want) > 10 * block


@pytest.mark.parametrize("hd", [64, 128])
def test_nan_and_infinity_reach_who_sees_them(gpu, hd):
    print(f"case NaN hd={hd}", flush=True)
    n, rows = 64 + 40, 30
    k, v = rows_of(11, n, 2, hd)
    v[90, 0, 3] = np.nan  # in the open block, seen by the last rows only
    v[95, 1, 5] = np.inf
    k[100, 1, 7] = 1e6  # beyond f16
    c, q = hip.PagedCache(1, 2, hd, 2, 2), queries(12, rows, 4, hd)
    ids = c.open(2)
    c.append(0, ids[:1], [n], k, v)
    got = check_attention(c, ids[:1], [(k, v)], [rows], 4, q=q, what="open block")
    # v[90] reaches dim 3 of head 0's rows from token 90 on (the rows stand for tokens 74 .. 103).
    assert np.isfinite(got[:16, :2]).all() and np.isnan(got[16:, :2, 3]).all() and np.isfinite(got[16:, :2, 4]).all()
    assert np.isnan(got[26:, 2:]).all()
    # Full: the whole block of that head.
    k2, v2 = rows_of(13, 24, 2, hd)
    c.append(0, ids[:1], [24], k2, v2)
    k, v = np.concatenate([k, k2]), np.concatenate([v, v2])
    kk, vv = c.read(0, ids[:1], [0], [128])
    assert same(np.isnan(kk), np.isnan(P.held(k).reshape(128, -1)))
    assert np.isnan(vv[64:]).all() and np.isfinite(vv[:64]).all()
    assert np.isnan(kk[64:, hd:]).all() and np.isfinite(kk[:, :hd]).all()
    got = c.attention(0, ids[:1], [70], queries(14, 70, 4, hd), 4).reshape(70, 4, hd)
    # Rows 0 .. 5 stand for tokens 58 .. 63, before that block.
    assert np.isfinite(got[:6]).all() and np.isnan(got[6:]).all()
    # A sequence that takes over the rows and pages of one with NaN.
    c.close(ids[:1])
    fresh = c.open(1)
    k, v = rows_of(15, 70, 2, hd)
    c.append(0, fresh, [70], k, v)
    check_attention(c, fresh, [(k, v)], [9], 4, what="after NaN")
    # NaN and infinite queries stay in their own row and head.
    q = queries(16, 3, 4, hd)
    q[1, 2, 0], q[2, 0, hd - 1] = np.nan, np.inf
    got = c.attention(0, fresh, [3], q, 4).reshape(3, 4, hd)
    bad = np.zeros((3, 4), bool)
    bad[1, 2] = bad[2, 0] = True
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()


def test_zeros_and_magnitudes(gpu):
    """Blocks of zeros, blocks of the smallest and largest f16 values, queries of 0."""
    print("case magnitudes", flush=True)
    k, v = rows_of(21, 64 * 4 + 9, 1, 64)
    k[:64] = 0.0
    v[64:128] = 0.0
    v[128:192] *= 6e-8
    k[192:256] *= 1e-7
    v[200:256] = np.clip(v[200:256] * 3e4, -65504, 65504)
    c = hip.PagedCache(1, 1, 64, 4, 1)
    ids = c.open(1)
    c.append(0, ids, [len(k)], k, v)
    q = queries(22, 3, 2, 64)
    q[0, 0] = 0.0
    q[1, 1] *= 1e-20
    check_attention(c, ids, [(k, v)], [3], 2, q=q, what="magnitudes")


def test_fork_and_reorder(gpu):
    """Beams: forks share pages, go on apart, and change places."""
    print("case beams", flush=True)
    hd, kvh, heads = 64, 2, 4
    c, ids, data = filled(hd, kvh, [150], pages=40, sequences=6, layers=2)
    used = c.info()["used"]
    beams = np.concatenate([ids, c.fork([ids[0]] * 4)])
    assert c.info()["used"] == used
    held = [data[0]] * 5
    r = np.random.default_rng(3)
    for step in range(70):
        n = 5
        new = [rows_of(1000 + 10 * step + b, 1, kvh, hd) for b in range(n)]
        for layer in range(2):
            c.append(layer, beams, [1] * n, np.concatenate([k for k, _ in new]), np.concatenate([v for _, v in new]))
        held = [(np.concatenate([k, a]), np.concatenate([v, b])) for (k, v), (a, b) in zip(held, new)]
        if step % 8 == 0 or step > 66:
            check_attention(c, beams, held, [1] * n, heads, layer=step % 2, what=f"step {step}")
        parents = r.integers(0, n, n)
        c.reorder(beams, beams[parents])
        held = [held[p] for p in parents]
        if step % 20 == 7:
            c.compact()
    lens = [len(k) for k, _ in held]
    got = c.read(1, beams, [0] * 5, lens)
    for w in (0, 1):
        assert same(got[w], np.concatenate([flat(P.held(h[w])) for h in held]))
    c.close(beams)
    assert c.info()["used"] == 0


def test_reorder_from_outside(gpu):
    print("case reorder from outside", flush=True)
    c, ids, data = filled(64, 1, [70, 130, 5], pages=20, sequences=4)
    c.reorder(ids[1:], [ids[0], ids[1]])
    held = [data[0], data[0], data[1]]
    check_attention(c, ids, held, [1, 1, 1], 2, what="reordered")
    new = rows_of(77, 3, 1, 64)
    c.append(0, ids, [1, 1, 1], *new)
    held = [(np.concatenate([k, new[0][i:i + 1]]), np.concatenate([v, new[1][i:i + 1]]))
            for i, (k, v) in enumerate(held)]
    check_attention(c, ids, held, [2, 2, 2], 2, what="appended")


def test_copy_compact_resize(gpu):
    print("case copy, compact, resize", flush=True)
    lens = [200, 64, 33, 500]
    a, ids, data = filled(128, 2, lens, pages=64, sequences=12, layers=2)
    b = hip.PagedCache(2, 2, 128, 13, 5)
    twins = a.fork([ids[0], ids[0]])
    used = a.info()["used"]
    # Into another cache, what is shared stays shared: 3 + 1 + 0 + 7 pages.
    away = a.copy(np.concatenate([ids, twins[:1]]), into=b)
    assert b.info()["used"] == 11
    inside = a.copy(ids)
    assert a.info()["used"] == used + 11
    a.close(ids)
    a.close(twins)
    assert a.info()["used"] == 11
    assert a.compact() == 11
    a.resize(11)
    assert a.info()["pages"] == 11
    with pytest.raises(hip.TritError, match="in use"):
        a.resize(10)
    with pytest.raises(hip.TritError, match="pages"):
        a.append(0, inside[1:2], [64], *rows_of(1, 64, 2, 128))
    a.resize(30)
    more = rows_of(9, 64, 2, 128)
    for layer in range(2):
        a.append(layer, inside[1:2], [64], *more)
    held = [data[0], tuple(np.concatenate(x) for x in zip(data[1], more)), data[2], data[3]]
    for layer in range(2):
        check_attention(a, inside, held, [1, 3, 1, 2], 4, layer=layer, what="moved")
        check_attention(b, away, data + [data[0]], [1, 3, 1, 2, 1], 4, layer=layer, what="copied")
    b.close(away[:1])
    assert b.info()["used"] == 11
    b.close(away[4:])
    assert b.info()["used"] == 8
    with pytest.raises(hip.TritError, match="differ"):
        a.copy(inside, into=hip.PagedCache(2, 2, 64, 13, 5))
    assert a.info()["bytes"] > 0


def test_strides_streams_and_offsets(gpu):
    """Rows inside qkv rows at odd offsets, on streams that change from call to call, in the last layer of a pool of
    more than 4 GB."""
    print("case strides and streams", flush=True)
    import ctypes as C

    hd, kvh, heads, layers = 80, 3, 6, 24
    lens, rows = [100, 61, 130], [3, 1, 2]
    c = hip.PagedCache(layers, kvh, hd, 4000, 3)
    assert c.info()["bytes"] > 1 << 32
    ids = c.open(3)
    total, width, stride = sum(lens), kvh * hd, 1001
    data = [rows_of(31 + i, n, kvh, hd) for i, n in enumerate(lens)]
    host = np.full((total, stride), np.nan, np.float32)
    host[:, 7:7 + width] = np.concatenate([k for k, _ in data]).reshape(total, -1)
    host[:, 501:501 + width] = np.concatenate([v for _, v in data]).reshape(total, -1)
    q = queries(33, sum(rows), heads, hd)
    qs = heads * hd + 13
    hq = np.full((sum(rows), qs), np.nan, np.float32)
    hq[:, 1:1 + heads * hd] = q.reshape(sum(rows), -1)
    D = Device()
    streams = []
    try:
        for name in ("hipStreamCreate", "hipStreamDestroy"):
            getattr(D.L, name).restype = C.c_int
        for _ in range(2):
            s = C.c_void_p()
            assert D.L.hipStreamCreate(C.byref(s)) == 0
            streams.append(s)
        d, dq = D.upload(host), D.upload(hq)
        out = D.upload(np.full((sum(rows) + 1, heads * hd), 7.0, np.float32))
        for layer in (0, layers - 1):
            c.append_device(layer, ids, lens, d.value + 28, stride, d.value + 2004, stride, streams[0])
            c.attention_device(layer, ids, rows, dq.value + 4, qs, heads, out, stream=streams[1])
            got = D.download(out, (sum(rows) + 1, heads * hd))
            assert (got[-1] == 7.0).all()
            at = 0
            for i, n in enumerate(rows):
                k, v = (P.held(x) for x in data[i])
                want, off = P.attention(q[at:at + n], k, v, [lens[i] - n + r + 1 for r in range(n)],
                                        float(np.float32(1) / np.sqrt(np.float32(hd))))
                near(got[at:at + n].reshape(n, heads, hd), want, off, f"layer {layer} sequence {i}")
                at += n
            back = D.upload(np.full((total, stride), 5.0, np.float32))
            c.read_device(layer, ids, [0] * 3, lens, back.value + 12, stride, back.value + 2400, stride, streams[0])
            got = D.download(back, (total, stride))
            k, v = (np.concatenate([flat(P.held(x[w])) for x in data]) for w in (0, 1))
            assert same(got[:, 3:3 + width], k) and same(got[:, 600:600 + width], v)
            mask = np.ones(stride, bool)
            mask[3:3 + width] = mask[600:600 + width] = False
            assert (got[:, mask] == 5.0).all()
    finally:
        D.free()
        for s in streams:
            D.L.hipStreamDestroy(s)


def test_many_sequences(gpu):
    """More sequences than a launch takes, in a mixed order, some without rows."""
    print("case 300 sequences", flush=True)
    lens = [1 + (37 * i) % 150 for i in range(300)]
    c, ids, data = filled(64, 1, lens)
    order = np.random.default_rng(5).permutation(300)
    rows = [min(lens[i], int(i) % 3) for i in order]
    check_attention(c, ids[order], [data[i] for i in order], rows, 2, what="many")
    both = c.fork(ids[:0])
    assert both.size == 0
    c.close(ids[::2])
    again = c.fork(ids[1:300:2])
    k, v = c.read(0, again, [0] * 150, lens[1::2])
    assert same(k, np.concatenate([flat(P.held(data[i][0])) for i in range(1, 300, 2)]))


def test_calls_are_deterministic(gpu):
    print("case deterministic", flush=True)
    c, ids, _ = filled(128, 2, [3000, 10, 700])
    q = queries(8, 3, 8, 128)
    first = c.attention(0, ids, [1, 1, 1], q, 8)
    for _ in range(5):
        assert same(c.attention(0, ids, [1, 1, 1], q, 8), first)
    # A sequence's rows do not depend on what else the call holds... up to how its keys are split.
    one = c.attention(0, ids[2:], [1], q[2:], 8)
    assert np.max(np.abs(one - first[2:])) < 1e-5


def test_refusals(gpu):
    print("case refusals", flush=True)
    c, ids, _ = filled(64, 2, [70, 3], pages=2)
    x = np.zeros((200, 2, 64), np.float32)
    for what, call in [
        ("no sequence 2", lambda: c.append(0, [2], [1], x[:1], x[:1])),
        ("no sequence -1", lambda: c.attention(0, [-1], [1], x[:1], 2)),
        ("layer 1", lambda: c.append(1, ids, [1, 1], x[:2], x[:2])),
        ("layer -1", lambda: c.read(-1, ids, [0, 0], [1, 1])),
        ("twice", lambda: c.append(0, [ids[0]] * 2, [1, 1], x[:2], x[:2])),
        ("negative", lambda: c.append(0, ids, [2, -1], x[:1], x[:1])),
        ("pages", lambda: c.append(0, ids, [58, 125], x[:183], x[:183])),
        ("evenly", lambda: c.attention(0, ids, [1, 1], x[:3], 3)),
        ("evenly", lambda: c.attention(0, ids, [1, 1], x[:0], 0)),
        ("holds 3", lambda: c.attention(0, ids, [1, 4], np.zeros((5, 128), np.float32), 2)),
        ("scale", lambda: c.attention(0, ids, [1, 1], x[:2], 2, scale=-1.0)),
        ("scale", lambda: c.attention(0, ids, [1, 1], x[:2], 2, scale=float("nan"))),
        ("holds 70", lambda: c.read(0, ids, [70, 0], [1, 1])),
        ("holds 3", lambda: c.read(0, ids, [0, -1], [1, 1])),
        ("sequences", lambda: c.open(1)),
        ("values", lambda: c.append(0, ids, [1, 1], x[:1], x[:2])),
        ("counts", lambda: c.append(0, ids, [1], x[:1], x[:1])),
        ("stride", lambda: c.append_device(0, ids, [1, 1], 64, 127, 64, 128)),
        ("stride", lambda: c.attention_device(0, ids, [1, 1], 64, 127, 2, 64)),
        ("NULL", lambda: c.append_device(0, ids, [1, 1], None, 128, 64, 128)),
        ("NULL", lambda: c.attention_device(0, ids, [1, 1], 64, 128, 2, None)),
    ]:
        with pytest.raises(hip.TritError, match=what):
            call()
    assert [c.length(i) for i in ids] == [70, 3]
    # Calls of nothing.
    c.append(0, ids, [0, 0], x[:0], x[:0])
    assert c.attention(0, ids, [0, 0], x[:0], 2).shape == (0, 128)
    assert c.attention(0, ids[:0], [], x[:0], 2).shape == (0, 128)


def test_a_refused_attention_writes_nothing(gpu):
    """More query rows than a call takes, in a sequence behind more than one launch holds."""
    print("case refused attention", flush=True)
    lens = [1] * 140 + [2001]
    c, ids, _ = filled(1, 1, lens)
    q = np.ones((sum(lens), 400), np.float32)
    D = Device()
    try:
        dq, out = D.upload(q), D.upload(np.full_like(q, 7.0))
        with pytest.raises(hip.TritError, match="rows"):
            c.attention_device(0, ids, lens, dq, 400, 400, out)
        assert (D.download(out, q.shape) == 7.0).all()
        c.attention_device(0, ids, lens[:140] + [2000], dq, 400, 400, out)
        got = D.download(out, q.shape)
        assert (got[:2140] != 7.0).all() and (got[2140] == 7.0).all()
    finally:
        D.free()


def test_capture_is_refused(gpu):
    print("case capture", flush=True)
    import torch

    c, ids, _ = filled(64, 2, [70, 3])
    q = torch.ones(2, 256, device="cuda")
    out = torch.zeros(2, 256, device="cuda")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out.add_(1.0)
        with pytest.raises(hip.TritError, match="captured"):
            c.attention_device(0, ids, [1, 1], q.data_ptr(), 256, 4, out.data_ptr(), stream=s.cuda_stream)
        with pytest.raises(hip.TritError, match="captured"):
            c.fork(ids[:0], stream=s.cuda_stream)
    g.replay()
    torch.cuda.synchronize()
    assert (out == 1.0).all()


def test_a_failed_resize_leaves_the_cache_as_it_was(gpu):
    """More memory than the card has: refused, and the next calls know nothing of it."""
    print("case resize beyond the card", flush=True)
    c, ids, data = filled(128, 8, [70, 3], layers=4)
    before = c.info()
    with pytest.raises(hip.TritError, match="memory"):
        c.resize(1 << 24)  # 8 TB
    assert c.info() == before
    new = rows_of(41, 2, 8, 128)
    for layer in range(4):
        c.append(layer, ids, [1, 1], *new)
    held = [(np.concatenate([k, new[0][i:i + 1]]), np.concatenate([v, new[1][i:i + 1]])) for i, (k, v) in enumerate(data)]
    check_attention(c, ids, held, [1, 2], 16, layer=3, what="after")


def test_two_threads(gpu):
    """Calls of two threads, each on its own stream, take turns."""
    print("case two threads", flush=True)
    import threading

    c, ids, data = filled(64, 2, [700, 90], pages=60, sequences=8)
    q = queries(5, 2, 4, 64)
    want = c.attention(0, ids, [1, 1], q, 4)
    bad = []

    def work(mine):
        try:
            hip.init(0)
            for step in range(20):
                if not same(c.attention(0, ids, [1, 1], q, 4), want):
                    bad.append("attention")
                child = c.fork([ids[mine]])
                k, v = rows_of(100 * mine + step, 70, 2, 64)
                c.append(0, child, [70], k, v)
                n = len(data[mine][0])
                got = c.read(0, child, [n], [70])
                held = P.held(np.concatenate([data[mine][0], k]))[n:]
                if not same(got[0], flat(held)):
                    bad.append("append")
                c.close(child)
        except Exception as e:  # noqa: BLE001
            bad.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad[:3]


def test_a_step_of_a_batch(gpu):
    """A decoder layer's step as it is used: beams forked, a token appended, self attention, cross attention to their
    audio's states, the beams chosen again."""
    print("case a batch's steps", flush=True)
    hd, kvh, heads, audios, beams = 64, 4, 4, 3, 4
    states = [rows_of(200 + a, n, kvh, hd) for a, n in enumerate((150, 64, 31))]
    cross = hip.CrossStates(2, kvh, hd, audios, 150)
    cache = hip.PagedCache(2, kvh, hd, 60, audios * beams)
    prompt = [rows_of(210 + a, n, kvh, hd) for a, n in enumerate((60, 3, 127))]
    first = cache.open(audios)
    for layer in range(2):
        cross.set(layer, range(audios), [len(k) for k, _ in states], *(np.concatenate(x) for x in zip(*states)))
        cache.append(layer, first, [len(k) for k, _ in prompt], *(np.concatenate(x) for x in zip(*prompt)))
    ids = np.concatenate([np.concatenate([first[a:a + 1], cache.fork([first[a]] * (beams - 1))]) for a in range(audios)])
    held = [prompt[a] for a in range(audios) for _ in range(beams)]
    r = np.random.default_rng(8)
    n = audios * beams
    for step in range(8):
        new = rows_of(300 + step, n, kvh, hd)
        q = queries(400 + step, n, heads, hd)
        held = [(np.concatenate([k, new[0][i:i + 1]]), np.concatenate([v, new[1][i:i + 1]]))
                for i, (k, v) in enumerate(held)]
        for layer in range(2):
            cache.append(layer, ids, [1] * n, *new)
            check_attention(cache, ids, held, [1] * n, heads, layer=layer, q=q, what=f"step {step}")
            got = cross.attention(layer, range(audios), [beams] * audios, q, heads).reshape(n, heads, hd)
            for a, (k, v) in enumerate(states):
                rows = slice(a * beams, (a + 1) * beams)
                want, off = P.attention(q[rows], P.f16(k), P.f16(v), [len(k)] * beams, 0.125)
                near(got[rows], want, off, f"cross {step}")
        parents = np.concatenate([a * beams + r.integers(0, beams, beams) for a in range(audios)])
        cache.reorder(ids, ids[parents])
        held = [held[p] for p in parents]
