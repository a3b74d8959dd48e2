"""Serving many sequences at once, as cases that can be timed and compared: a
paged key/value cache held in 8 bits, the attention that reads it, its pages'
bookkeeping, and decoder rows' attention to an encoder's states.

A cache holds keys and values in blocks of 64 tokens of one key/value head. A
block that is not full holds its values as f16. A full one holds int8 codes
and an f32 scale: a / 127 with a the largest magnitude of the block's f16
values; the codes are round(127 * value / a), halves to the even one.

A case is a dict of plain values with a `family`:

- "attend": `rows` query rows of each of `seqs` sequences, at the ends of
  caches of `lo` to `hi` tokens.
- "write": `rows_lo` to `rows_hi` new rows of each of `seqs` sequences that
  hold `lo` to `hi` tokens, appended to forks of them; the blocks the rows
  touch are read back as the values they stand for.
- "beam": a decoder step of `seqs` beams over `layers` layers: each continues
  a fork of the beam it was chosen from, by one token; the last block of every
  beam is read back.
- "copy": sequences copied page by page, the originals freed, and the copies
  moved into the pages this leaves at the front; all values read back.
- "cross": `rows` rows of each of `slots` audios over `lo` to `hi` encoder
  positions, held as f16; with `fill` the keys and values are new and are
  laid out in the pass.

Outputs are f32, as everywhere in the library.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

BLOCK = 64


def listed():
    return [
        # The smallest call: one token of one sequence (the 0.6B decoder's heads).
        dict(name="attend_one", family="attend", seqs=1, lo=700, hi=700, rows=1, heads=16, kv_heads=8, head_dim=128),
        # A serving batch: 32 requests of very different lengths.
        dict(name="attend_ragged_32", family="attend", seqs=32, lo=100, hi=8001, rows=1, heads=16, kv_heads=8,
             head_dim=128),
        # Two very long contexts.
        dict(name="attend_long_2", family="attend", seqs=2, lo=130000, hi=131111, rows=1, heads=32, kv_heads=8,
             head_dim=128),
        # An audio LLM's prompt (1500 audio rows and 64 tokens) after 1000 cached tokens.
        dict(name="attend_prompt_1564", family="attend", seqs=1, lo=2564, hi=2564, rows=1564, heads=16, kv_heads=8,
             head_dim=128),
        # One token of each of 48 requests goes into the cache.
        dict(name="write_step_48", family="write", seqs=48, lo=1, hi=1500, rows_lo=1, rows_hi=1, kv_heads=8,
             head_dim=128),
        # Eight prompts go into the cache.
        dict(name="write_prompts_8", family="write", seqs=8, lo=0, hi=130, rows_lo=37, rows_hi=1564, kv_heads=8,
             head_dim=128),
        # Beam search with Whisper large-v3's heads, 5 beams, 4 of its layers.
        dict(name="beam_step_5", family="beam", seqs=5, layers=4, lo=447, hi=447, heads=20, kv_heads=20, head_dim=64),
        # Five beams for each of 12 audios, of different lengths.
        dict(name="beam_step_60", family="beam", seqs=60, layers=2, lo=30, hi=447, heads=16, kv_heads=8,
             head_dim=128),
        # Sequences moved within the pool, so that its end can be given back.
        dict(name="copy_compact_12", family="copy", seqs=12, layers=2, lo=200, hi=3001, kv_heads=8, head_dim=128),
        # One audio, 5 beams, a Whisper large-v3 decoder layer.
        dict(name="cross_beams_5", family="cross", slots=1, lo=1500, hi=1500, rows=5, heads=20, kv_heads=20,
             head_dim=64, fill=False),
        # A batch of audios of different lengths: new states, then the first rows (the start tokens of a transcript).
        dict(name="cross_first_16", family="cross", slots=16, lo=150, hi=1500, rows=4, heads=16, kv_heads=16,
             head_dim=64, fill=True),
        # Whole transcripts against their audios (scoring of known text).
        dict(name="cross_rows_448", family="cross", slots=8, lo=700, hi=1500, rows=448, heads=20, kv_heads=20,
             head_dim=64, fill=False),
    ]


def _log_int(rng, lo, hi):
    """A whole number in [lo, hi], uniform over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# (query heads, key/value heads, head_dim)
_HEADS = [(16, 8, 128), (16, 8, 128), (32, 8, 128), (20, 20, 64), (12, 12, 64), (8, 1, 128), (14, 2, 64), (10, 5, 96),
          (6, 6, 80), (9, 3, 40)]


def draw(rng):
    """One more case of the listed ones' ranges."""
    family = rng.choice(["attend", "attend", "attend", "write", "beam", "copy", "cross", "cross"])
    heads, kv_heads, head_dim = rng.choice(_HEADS)
    shape = dict(heads=heads, kv_heads=kv_heads, head_dim=head_dim)
    width = kv_heads * head_dim
    if family == "attend":
        kind = rng.choice(["step", "step", "few", "chunk"])
        if kind == "chunk":
            rows, seqs = _log_int(rng, 17, 1000), rng.randint(1, 2)
            hi = rows + _log_int(rng, 1, 2000)
            lo = rows + rng.randint(0, hi - rows)
        else:
            rows = 1 if kind == "step" else rng.randint(2, 8)
            seqs = _log_int(rng, 1, 60)
            hi = _log_int(rng, rows + 1, max(rows + 1, min(60000, (1 << 26) // (seqs * width))))
            lo = _log_int(rng, rows, hi)
        return dict(family=family, seqs=seqs, lo=lo, hi=hi, rows=rows, **shape)
    if family == "write":
        seqs = _log_int(rng, 1, 64)
        rows_hi = _log_int(rng, 1, max(1, min(3000, (1 << 23) // (seqs * width))))
        return dict(family=family, seqs=seqs, lo=rng.randint(0, 200), hi=rng.randint(200, 1500),
                    rows_lo=_log_int(rng, 1, rows_hi), rows_hi=rows_hi, kv_heads=kv_heads, head_dim=head_dim)
    if family == "beam":
        hi = _log_int(rng, 2, 1500)
        return dict(family=family, seqs=_log_int(rng, 2, 60), layers=rng.randint(1, 3), lo=_log_int(rng, 1, hi), hi=hi,
                    **shape)
    if family == "copy":
        seqs = _log_int(rng, 1, 32)
        hi = _log_int(rng, 1, max(2, min(6000, (1 << 24) // (seqs * width))))
        return dict(family=family, seqs=seqs, layers=rng.randint(1, 2), lo=rng.randint(0, hi), hi=hi,
                    kv_heads=kv_heads, head_dim=head_dim)
    slots = _log_int(rng, 1, 24)
    rows = rng.choice([1, rng.randint(1, 6), _log_int(rng, 7, 448)])
    cap = min(9000, (1 << 24) // (slots * width), (1 << 27) // (slots * rows * heads))
    hi = _log_int(rng, 1, max(1, cap))
    lo = rng.choice([0, _log_int(rng, 1, hi)])
    return dict(family=family, slots=slots, lo=lo, hi=hi, rows=rows, fill=rng.random() < 0.3, **shape)


# ---- sizes and inputs -------------------------------------------------------


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, even over their logarithm, in a mixed order."""
    at = np.linspace(0.0, 1.0, n) if n > 1 else np.ones(1)
    v = np.rint(np.exp((1.0 - at) * math.log(lo + 1) + at * math.log(hi + 1)) - 1).astype(np.int64)
    return v[(np.arange(n) * 7919 + 3) % n] if n % 7919 else v


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _channels(g, kv_heads, head_dim):
    """Keys have channels of very different size: a factor for each."""
    return torch.exp(0.5 * _randn(g, 1, 1, 1, kv_heads, head_dim))


def _inputs(case, seed):
    """Rows of keys and values as projections give them, with their counts:
    k, v (layers, seqs, tokens up to the longest, kv_heads, head_dim), the
    queries, and for families that append the new rows in `new_k`, `new_v`
    (layers, seqs, rows up to the most, kv_heads, head_dim)."""
    g = _gen(seed)
    family, kvh, hd = case["family"], case["kv_heads"], case["head_dim"]
    n = case["slots"] if family == "cross" else case["seqs"]
    layers = case.get("layers", 1)
    lens = _spread(n, case["lo"], case["hi"])
    d = dict(lens=lens)
    scale = _channels(g, kvh, hd)
    d["k"] = _randn(g, layers, n, int(lens.max()), kvh, hd) * scale
    d["v"] = _randn(g, layers, n, int(lens.max()), kvh, hd)
    rows = 1 if family == "beam" else case.get("rows", 0)
    if "heads" in case:
        # Sharp enough that some keys stand out, as trained heads' do.
        d["q"] = 1.5 * _randn(g, layers, n, rows, case["heads"], hd)
    if family in ("write", "beam"):
        new = _spread(n, case["rows_lo"], case["rows_hi"]) if family == "write" else np.ones(n, np.int64)
        d["rows"] = new
        d["new_k"] = _randn(g, layers, n, int(new.max()), kvh, hd) * scale
        d["new_v"] = _randn(g, layers, n, int(new.max()), kvh, hd)
    if family == "beam":
        # Every third beam goes on twice, the one after it not at all.
        beam = torch.arange(n, device="cuda")
        d["parents"] = beam - (beam % 3 == 2).long()
    return d


def _valid(counts, most):
    """(seqs, most): whether a row is one of its sequence's."""
    return torch.arange(most, device="cuda")[None, :] < torch.as_tensor(counts, device="cuda")[:, None]


def _stacked(rows, counts):
    """(layers, seqs, most, ...) to (layers, rows of all sequences, width)."""
    flat = rows.flatten(3)
    return flat[:, _valid(counts, rows.shape[2])].contiguous()


# ---- the cache, plain -------------------------------------------------------


def _quantized(h):
    """Codes and scales of full blocks: h (..., 64, head_dim) f16 values."""
    a = h.abs().amax(dim=(-2, -1), keepdim=True).float()
    # 127 h is exact in f32, and no quotient of two f16 values rounds onto a half it is not.
    codes = torch.round(127.0 * h.float() / torch.where(a > 0, a, torch.ones_like(a)))
    return codes.to(torch.int8), a / torch.full_like(a, 127.0)


def _blocks(rows, lens, extra):
    """Rows (layers, seqs, tokens, heads, hd) as f16 blocks (layers, seqs,
    blocks, heads, 64, hd), zero past each length, with `extra` blocks more."""
    layers, n, t, kvh, hd = rows.shape
    nb = t // BLOCK + 1 + extra
    held = torch.zeros(layers, n, nb * BLOCK, kvh, hd, dtype=torch.float16, device="cuda")
    held[:, :, :t] = torch.where(_valid(lens, t)[None, :, :, None, None], rows, torch.zeros((), device="cuda")).half()
    return held.view(layers, n, nb, BLOCK, kvh, hd).transpose(3, 4)


def _plain_cache(d, g, extra=0):
    """A pool of pages in mixed order, each sequence's table of them, and its open block."""
    pool = {}
    lens = torch.as_tensor(d["lens"], device="cuda")
    for name in ("k", "v"):
        blocks = _blocks(d[name], d["lens"], extra)
        layers, n, nb = blocks.shape[:3]
        if "table" not in pool:
            pool["table"] = torch.randperm(n * nb, generator=g, device="cuda").view(n, nb)
        codes, scales = _quantized(blocks)
        at = pool["table"].flatten()
        pool["codes_" + name] = torch.empty_like(codes.flatten(1, 2))
        pool["scales_" + name] = torch.empty_like(scales.flatten(1, 2))
        pool["codes_" + name][:, at] = codes.flatten(1, 2)
        pool["scales_" + name][:, at] = scales.flatten(1, 2)
        last = (lens // BLOCK)[None, :, None, None, None, None].expand(layers, n, 1, *blocks.shape[3:])
        pool["open_" + name] = blocks.gather(2, last).squeeze(2)
        del blocks, codes, scales
    pool["lens"] = lens
    return pool


def _values(pool, name, table, lens, open_blocks):
    """The values a cache holds: (layers, seqs, blocks, heads, 64, hd) f32,
    zero from each length on."""
    n, nb = table.shape
    v = pool["codes_" + name][:, table].float() * pool["scales_" + name][:, table]
    b = torch.arange(nb, device="cuda")[None, :]
    full, is_open = (b < lens[:, None] // BLOCK), (b == lens[:, None] // BLOCK)
    shape = (1, n, nb, 1, 1, 1)
    v = torch.where(full.view(shape), v, torch.zeros((), device="cuda"))
    filled = torch.arange(BLOCK, device="cuda")[None, :] < (lens % BLOCK)[:, None]
    part = torch.where(filled.view(1, n, 1, BLOCK, 1), open_blocks.float(), torch.zeros((), device="cuda"))
    return torch.where(is_open.view(shape), part.unsqueeze(2), v)


def _rows_of(values):
    """(layers, seqs, blocks, heads, 64, hd) to (layers, seqs, tokens, heads, hd)."""
    return values.transpose(3, 4).flatten(2, 3)


def _attention(q, k, v, seen):
    """q (layers, seqs, rows, heads, hd), k and v (layers, seqs, heads_kv,
    tokens, hd) f32; row r of sequence b sees its first seen[b, r] keys."""
    layers, n, rows, heads, hd = q.shape
    kvh = k.shape[2]
    group = heads // kvh
    qh = q.view(layers, n, rows, kvh, group, hd).permute(0, 1, 3, 4, 2, 5).reshape(layers, n, kvh, group * rows, hd)
    s = torch.matmul(qh * (1.0 / math.sqrt(hd)), k.transpose(-1, -2)).view(layers, n, kvh, group, rows, -1)
    sees = torch.arange(k.shape[3], device="cuda") < seen[:, :, None]
    s = s.masked_fill(~sees.view(1, n, 1, 1, rows, -1), -math.inf)
    m = s.amax(dim=-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    total = e.sum(dim=-1, keepdim=True)
    o = torch.matmul(e.view(layers, n, kvh, group * rows, -1), v).view(layers, n, kvh, group, rows, hd)
    o = torch.where(total > 0, o / total, torch.zeros((), device="cuda"))
    return o.permute(0, 1, 4, 2, 3, 5).reshape(layers, n * rows, heads * hd)


def _seen(lens, rows):
    return lens[:, None] - rows + 1 + torch.arange(rows, device="cuda")[None, :]


def _plain_write(pool, parents, d):
    """The caches of forks of `parents` with the new rows, as values of whole
    blocks from each fork's first touched one on: k and v (layers, seqs,
    blocks, heads, 64, hd), the first touched blocks, and the new lengths."""
    rows = d["rows_t"]
    old = pool["lens"][parents]
    most = d["new_k"].shape[2]
    nb = (most + BLOCK - 1) // BLOCK + 1
    out = []
    for name in ("k", "v"):
        new = d["new_" + name]
        layers, n, _, kvh, hd = new.shape
        held = torch.zeros(layers, n, nb * BLOCK, kvh, hd, dtype=torch.float16, device="cuda")
        held[:, :, :BLOCK] = pool["open_" + name][:, parents].transpose(2, 3)
        # New row i goes to place old % 64 + i; rows a sequence does not have go nowhere.
        at = (old % BLOCK)[:, None] + torch.arange(most, device="cuda")[None, :]
        b, i = torch.nonzero(_valid(rows, most), as_tuple=True)
        held[:, b, at[b, i]] = new[:, b, i].half()
        held = held.view(layers, n, nb, BLOCK, kvh, hd).transpose(3, 4)
        codes, scales = _quantized(held)
        full = torch.arange(nb, device="cuda")[None, :] < ((old % BLOCK + rows) // BLOCK)[:, None]
        out.append(torch.where(full.view(1, n, nb, 1, 1, 1), codes.float() * scales, held.float()))
    return out[0], out[1], old // BLOCK, old + rows


# ---- prepare and run --------------------------------------------------------


def _device_cache(case, d, slack):
    """The library's cache with every sequence's rows in it. It owns its pages,
    as a session does its caches, so a program keeps this handle between calls."""
    from trit_amd import hip

    layers = case.get("layers", 1)
    lens = d["lens"]
    pages = int((lens // BLOCK).sum()) + slack
    cache = hip.PagedCache(layers, case["kv_heads"], case["head_dim"], max(pages, 1), 2 * len(lens))
    ids = cache.open(len(lens))
    counts = lens.astype(np.int32)
    width = case["kv_heads"] * case["head_dim"]
    ks, vs = _stacked(d["k"], lens), _stacked(d["v"], lens)
    torch.cuda.synchronize()
    for layer in range(layers):
        cache.append_device(layer, ids, counts, ks[layer].data_ptr(), width, vs[layer].data_ptr(), width)
    torch.cuda.synchronize()
    return cache, ids


def prepare(case, seed):
    family, kvh, hd = case["family"], case["kv_heads"], case["head_dim"]
    d = _inputs(case, seed)
    lens = d["lens"]
    layers, n, width = case.get("layers", 1), len(lens), kvh * hd
    s = dict(family=family, layers=layers, kv_heads=kvh, head_dim=hd, heads=case.get("heads"), rows=case.get("rows", 1),
             counts=np.full(n, case.get("rows", 1), np.int32), host_lens=lens.astype(np.int32),
             lens=torch.as_tensor(lens, device="cuda"))
    if "q" in d:
        s["q"] = d["q"]
        s["out"] = torch.empty(layers, d["q"].shape[1] * d["q"].shape[2], case["heads"] * hd, device="cuda")
    if family == "cross":
        s["fill"] = case["fill"]
        s["ks"], s["vs"] = (_stacked(d[x], lens)[0] for x in ("k", "v"))
        if own:
            from trit_amd import hip

            s["cross"] = hip.CrossStates(1, kvh, hd, n, max(int(lens.max()), 1))
            s["slots"] = np.arange(n, dtype=np.int32)
            torch.cuda.synchronize()
            if not case["fill"]:
                s["cross"].set_device(0, s["slots"], s["host_lens"], s["ks"].data_ptr(), width, s["vs"].data_ptr(), width)
                torch.cuda.synchronize()
        elif not case["fill"]:
            s["k"], s["v"] = (_plain_states(s, s[x]) for x in ("ks", "vs"))
        if not case["fill"]:
            del s["ks"], s["vs"]
        s["at"] = torch.nonzero(_valid(lens, max(int(lens.max()), 1)), as_tuple=True)
        return s
    touched = 0
    if family in ("write", "beam"):
        s["new_rows"] = d["rows"].astype(np.int32)
        s["rows_t"] = torch.as_tensor(d["rows"], device="cuda")
        s["new_k"], s["new_v"] = d["new_k"], d["new_v"]
        s["parents"] = d.get("parents", torch.arange(n, device="cuda"))
        old = lens[s["parents"].cpu().numpy()]
        touched = (old % BLOCK + d["rows"]) // BLOCK
        s["from"] = (old // BLOCK * BLOCK).astype(np.int32)
        s["back"] = (old % BLOCK + d["rows"]).astype(np.int32)
    elif family == "copy":
        s["from"], s["back"] = np.zeros(n, np.int32), s["host_lens"]
        touched = lens // BLOCK
    if family != "attend":
        # The rows that are read back, as (sequence, token from the first one on).
        s["at"] = torch.nonzero(_valid(s["back"], max(int(s["back"].max()), 1)), as_tuple=True)
        total = int(s["back"].sum())
        s["read_k"], s["read_v"] = (torch.empty(layers, total, width, device="cuda") for _ in range(2))
    if own:
        s["cache"], s["ids"] = _device_cache(case, d, int(np.sum(touched)))
        if family in ("write", "beam"):
            s["stack_k"], s["stack_v"] = _stacked(d["new_k"], d["rows"]), _stacked(d["new_v"], d["rows"])
            s["parent_ids"] = s["ids"][s["parents"].cpu().numpy()]
    else:
        s["pool"] = _plain_cache(d, _gen(seed + 1))
        if family == "copy":
            pool = s["pool"]
            full = torch.arange(pool["table"].shape[1], device="cuda")[None, :] < (s["lens"] // BLOCK)[:, None]
            s["used"] = pool["table"][full]
    return s


def _plain_states(s, rows):
    """The stacked rows as padded f16 states (1, slots, heads, positions, hd)."""
    most = max(int(s["host_lens"].max()), 1)
    held = torch.zeros(len(s["host_lens"]), most, s["kv_heads"], s["head_dim"], dtype=torch.float16, device="cuda")
    held[_valid(s["lens"], most)] = rows.view(-1, s["kv_heads"], s["head_dim"]).half()
    return held.transpose(1, 2)[None]


def _plain(s):
    family = s["family"]
    if family == "cross":
        if s["fill"]:
            k, v = _plain_states(s, s["ks"]), _plain_states(s, s["vs"])
        else:
            k, v = s["k"], s["v"]
        return _attention(s["q"], k.float(), v.float(), s["lens"][:, None].expand(-1, s["rows"]))[0]
    pool = s["pool"]
    if family == "attend":
        k = _values(pool, "k", pool["table"], pool["lens"], pool["open_k"]).transpose(2, 3).flatten(3, 4)
        v = _values(pool, "v", pool["table"], pool["lens"], pool["open_v"]).transpose(2, 3).flatten(3, 4)
        return _attention(s["q"], k, v, _seen(pool["lens"], s["rows"]))[0]
    b, i = s["at"]
    if family == "copy":
        # Every page to a place of its own, then all of them to the front of a pool.
        codes = [pool["codes_" + x][:, s["used"]].clone() for x in ("k", "v")]
        scales = [pool["scales_" + x][:, s["used"]].clone() for x in ("k", "v")]
        opens = [pool["open_" + x].clone() for x in ("k", "v")]
        place = torch.zeros_like(pool["table"])
        full = torch.arange(place.shape[1], device="cuda")[None, :] < (pool["lens"] // BLOCK)[:, None]
        # Moving a sequence onto zero pages is nothing to gather.
        place[full] = torch.arange(s["used"].shape[0], device="cuda")
        if s["used"].shape[0] == 0:
            codes = [pool["codes_" + x][:, :1] for x in ("k", "v")]
            scales = [pool["scales_" + x][:, :1] for x in ("k", "v")]
        moved = dict(codes_k=codes[0], codes_v=codes[1], scales_k=scales[0], scales_v=scales[1])
        k = _rows_of(_values(moved, "k", place, pool["lens"], opens[0]))
        v = _rows_of(_values(moved, "v", place, pool["lens"], opens[1]))
        return dict(k=k[:, b, i].flatten(2), v=v[:, b, i].flatten(2))
    k, v, first, lens = _plain_write(pool, s["parents"], s)
    out = dict(k=_rows_of(k)[:, b, i].flatten(2), v=_rows_of(v)[:, b, i].flatten(2))
    if family == "beam":
        # The shared blocks of the parent, then the fork's last two.
        n, nb = s["parents"].shape[0], pool["table"].shape[1]
        table = pool["table"][s["parents"]]
        whole = first * BLOCK
        zeros = torch.zeros_like(pool["open_k"][:, s["parents"]])
        at = (first[:, None] + torch.arange(2, device="cuda")[None, :]).view(1, n, 2, 1, 1, 1)
        full = []
        for name, last in (("k", k), ("v", v)):
            base = _values(pool, name, table, whole, zeros)
            base = torch.cat([base, torch.zeros_like(base[:, :, :2])], dim=2)
            full.append(base.scatter(2, at.expand_as(last), last).transpose(2, 3).flatten(3, 4))
        out["att"] = _attention(s["q"], full[0], full[1], lens[:, None])
    return out


def run(state):
    if not own:
        return _plain(state)
    s, family = state, state["family"]
    width = s["kv_heads"] * s["head_dim"]
    if family == "cross":
        if s["fill"]:
            s["cross"].set_device(0, s["slots"], s["host_lens"], s["ks"].data_ptr(), width, s["vs"].data_ptr(), width)
        s["cross"].attention_device(0, s["slots"], s["counts"], s["q"].data_ptr(), s["heads"] * s["head_dim"],
                                    s["heads"], s["out"].data_ptr())
        return s["out"][0]
    cache = s["cache"]
    if family == "attend":
        cache.attention_device(0, s["ids"], s["counts"], s["q"].data_ptr(), s["heads"] * s["head_dim"], s["heads"],
                               s["out"].data_ptr())
        return s["out"][0]
    if family == "copy":
        ids = cache.copy(s["ids"])
        cache.close(s["ids"])
        s["ids"] = ids
        cache.compact()
    else:
        ids = cache.fork(s["parent_ids"])
        for layer in range(s["layers"]):
            cache.append_device(layer, ids, s["new_rows"], s["stack_k"][layer].data_ptr(), width,
                                s["stack_v"][layer].data_ptr(), width)
            if family == "beam":
                cache.attention_device(layer, ids, s["counts"], s["q"][layer].data_ptr(), s["heads"] * s["head_dim"],
                                       s["heads"], s["out"][layer].data_ptr())
    for layer in range(s["layers"]):
        cache.read_device(layer, ids, s["from"], s["back"], s["read_k"][layer].data_ptr(), width,
                          s["read_v"][layer].data_ptr(), width)
    out = dict(k=s["read_k"], v=s["read_v"])
    if family != "copy":
        cache.close(ids)
    if family == "beam":
        out["att"] = s["out"]
    return out


# ---- work -------------------------------------------------------------------


def work(case):
    family, kvh, hd = case["family"], case["kv_heads"], case["head_dim"]
    n = case["slots"] if family == "cross" else case["seqs"]
    lens = _spread(n, case["lo"], case["hi"]).astype(np.float64)
    width, layers = kvh * hd, case.get("layers", 1)
    # A full block's codes and two scales a head; two bytes a value of an open one.
    held = float((lens // BLOCK).sum()) * (2 * BLOCK * width + 8 * kvh) + float((lens % BLOCK).sum()) * 4 * width
    if family == "cross":
        rows, heads = case["rows"], case["heads"]
        # New states come as f32; kept ones are f16.
        nbytes = lens.sum() * width * (8 if case["fill"] else 4) + 8.0 * n * rows * heads * hd
        return dict(bytes=float(nbytes), flops=float(4 * rows * lens.sum() * heads * hd))
    if family == "attend":
        rows, heads = case["rows"], case["heads"]
        pairs = rows * lens.sum() - n * rows * (rows - 1) / 2
        return dict(bytes=held + 8.0 * n * rows * heads * hd, flops=float(4 * pairs * heads * hd))
    if family == "copy":
        return dict(bytes=float(layers * (held + 8.0 * lens.sum() * width)), flops=float(2 * layers * lens.sum() * width))
    new = _spread(n, case["rows_lo"], case["rows_hi"]) if family == "write" else np.ones(n)
    touched = float((lens % BLOCK + new).sum())
    # New rows in (f32), the open blocks in (f16), the touched blocks' values out (f32).
    nbytes = layers * width * (8.0 * new.sum() + 4.0 * (lens % BLOCK).sum() + 8.0 * touched)
    flops = 6.0 * layers * width * touched
    if family == "beam":
        heads = case["heads"]
        nbytes += layers * (held + 8.0 * n * heads * hd)
        flops += 4.0 * layers * (lens.sum() + n) * heads * hd
    return dict(bytes=float(nbytes), flops=float(flops))


# ---- float64 ----------------------------------------------------------------


def _held64(rows, length):
    """The values a cache holds of `length` rows (length, heads, hd), in float64."""
    h = rows[:length].half().double()
    out = h.clone()
    for at in range(0, length // BLOCK * BLOCK, BLOCK):
        block = h[at:at + BLOCK]
        a = block.abs().amax(dim=(0, 2), keepdim=True)
        out[at:at + BLOCK] = torch.round(127.0 * block / torch.where(a > 0, a, torch.ones_like(a))) * (a / 127.0)
    return out


def _attend64(q, k, v, seen):
    """q (rows, heads, hd), k and v (tokens, kv_heads, hd); row r sees seen[r] keys."""
    rows, heads, hd = q.shape
    out = torch.zeros(rows, heads, hd, dtype=torch.float64, device="cuda")
    if k.shape[0] == 0:
        return out
    hidden = torch.arange(k.shape[0], device="cuda")[None, :] >= seen[:, None]
    for h in range(heads):
        g = h // (heads // k.shape[1])
        s = (q[:, h].double() @ k[:, g].T.contiguous()) / math.sqrt(hd)
        out[:, h] = torch.softmax(s.masked_fill(hidden, -math.inf), dim=1) @ v[:, g].contiguous()
    return out


def exact(case, seed):
    d = _inputs(case, seed)
    family, lens = case["family"], d["lens"]
    layers, n = case.get("layers", 1), len(lens)
    if family in ("attend", "cross"):
        outs = []
        for b in range(n):
            t, rows = int(lens[b]), case["rows"]
            if family == "cross":
                k, v = (d[x][0, b, :t].half().double() for x in ("k", "v"))
                seen = torch.full((rows,), t, device="cuda")
            else:
                k, v = (_held64(d[x][0, b], t) for x in ("k", "v"))
                seen = torch.arange(t - rows + 1, t + 1, device="cuda")
            outs.append(_attend64(d["q"][0, b], k, v, seen).flatten(1))
        return torch.cat(outs)
    keys, values, atts = [], [], []
    for layer in range(layers):
        ks, vs, att = [], [], []
        for b in range(n):
            if family == "copy":
                t = int(lens[b])
                ks.append(_held64(d["k"][layer, b], t).flatten(1))
                vs.append(_held64(d["v"][layer, b], t).flatten(1))
                continue
            parent = int(d["parents"][b]) if family == "beam" else b
            old, new = int(lens[parent]), int(d["rows"][b])
            k, v = (_held64(torch.cat([d[x][layer, parent, :old], d["new_" + x][layer, b, :new]]), old + new)
                    for x in ("k", "v"))
            ks.append(k[old // BLOCK * BLOCK:].flatten(1))
            vs.append(v[old // BLOCK * BLOCK:].flatten(1))
            if family == "beam":
                att.append(_attend64(d["q"][layer, b], k, v, torch.tensor([old + new], device="cuda")).flatten(1))
        keys.append(torch.cat(ks))
        values.append(torch.cat(vs))
        if att:
            atts.append(torch.cat(att))
    out = dict(k=torch.stack(keys), v=torch.stack(values))
    if atts:
        out["att"] = torch.stack(atts)
    return out
