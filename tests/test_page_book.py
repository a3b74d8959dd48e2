"""The paged cache's books (trit_amd/csrc/page_book.h) on the host: random
calls against a model that keeps every sequence's tokens, with the device's
part (table entries, row copies, page moves) played on plain lists."""

import ctypes as C
import os
import random
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
BLOCK = 64


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("book") / "book.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-Wall", "-Werror",
                    "-o", out, os.path.join(HERE, "page_book_shim.cpp")], check=True)
    lib = C.CDLL(out)
    lib.book_new.restype = C.c_void_p
    lib.book_error.restype = C.c_char_p
    for name in ("book_free", "book_used", "book_row", "book_length", "book_open", "book_close", "book_fork",
                 "book_reorder", "book_append", "book_copy", "book_compact", "book_resize"):
        fn = getattr(lib, name)
        types = {"book_free": 1, "book_used": 1, "book_row": 2, "book_length": 3, "book_open": 3, "book_close": 3,
                 "book_fork": 5, "book_reorder": 5, "book_append": 6, "book_copy": 9, "book_compact": 4,
                 "book_resize": 2}[name]
        fn.argtypes = [C.c_void_p] + {
            "book_free": [], "book_used": [], "book_row": [C.c_int], "book_length": [C.c_int, C.c_int],
            "book_open": [C.c_int, C.c_void_p], "book_close": [C.c_void_p, C.c_int],
            "book_fork": [C.c_void_p, C.c_int, C.c_void_p, C.c_void_p],
            "book_reorder": [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p],
            "book_append": [C.c_int, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p],
            "book_copy": [C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p],
            "book_compact": [C.c_void_p, C.c_void_p, C.c_void_p], "book_resize": [C.c_int]}[name]
        assert len(fn.argtypes) == types
    return lib


def ints(values):
    return (C.c_int * max(len(values), 1))(*values)


class Played:
    """A book and the device arrays it speaks of: pages and open blocks as
    lists of tokens by layer, the page table."""

    def __init__(self, lib, layers, pages, sequences):
        self.lib, self.layers, self.sequences = lib, layers, sequences
        self.h = lib.book_new(layers, pages, sequences)
        self.pages = [[None] * layers for _ in range(pages)]
        self.open = [[[] for _ in range(layers)] for _ in range(sequences)]
        self.table = [[None] * pages for _ in range(sequences)]
        self.model = {}  # id -> tokens by layer

    def ok(self, rc):
        assert rc >= 0, self.lib.book_error()
        return rc

    def refused(self, rc, why):
        assert rc == -1 and why in self.lib.book_error().decode(), (rc, self.lib.book_error())
        self.check()

    def entries(self, e, n):
        for i in range(n):
            row, block, page = e[3 * i:3 * i + 3]
            self.table[row][block] = page

    def open_new(self, n):
        out = ints([0] * n)
        self.ok(self.lib.book_open(self.h, n, out))
        for i in out[:n]:
            assert i not in self.model
            self.model[i] = [[] for _ in range(self.layers)]
        return out[:n]

    def copy_rows(self, c, n, to):
        src = [[list(x) for x in self.open[c[4 * i]]] for i in range(n)]
        tables = [list(self.table[c[4 * i]]) for i in range(n)]
        assert not {c[4 * i] for i in range(n)} & {c[4 * i + 1] for i in range(n)} or to is not self
        assert len({c[4 * i + 1] for i in range(n)}) == n
        for i in range(n):
            dst, length, blocks = c[4 * i + 1:4 * i + 4]
            to.open[dst] = [x[:length % BLOCK] for x in src[i]]
            for b in range(blocks):
                to.table[dst][b] = tables[i][b]

    def fork(self, ids):
        out, c = ints([0] * len(ids)), ints([0] * (4 * len(ids)))
        n = self.ok(self.lib.book_fork(self.h, ints(ids), len(ids), out, c))
        self.copy_rows(c, n, self)
        for i, o in zip(ids, out[:len(ids)]):
            assert o not in self.model
            self.model[o] = [list(x) for x in self.model[i]]
        return out[:len(ids)]

    def reorder(self, ids, parents):
        c = ints([0] * (4 * len(ids)))
        n = self.ok(self.lib.book_reorder(self.h, ints(ids), ints(parents), len(ids), c))
        # One copy for each sequence whose parent already has an heir among the sequences.
        assert n == len(ids) - len({p for p in parents if p in ids})
        self.copy_rows(c, n, self)
        before = {p: [list(x) for x in self.model[p]] for p in parents}
        for i, p in zip(ids, parents):
            self.model[i] = [list(x) for x in before[p]]

    def copy(self, ids, into):
        total = sum(len(self.model[i][0]) // BLOCK for i in ids) + 1
        out, r, m, e, k = ints([0] * len(ids)), ints([0] * 4 * len(ids)), ints([0] * 2 * total), ints([0] * 3 * total), ints([0] * 3)
        self.ok(self.lib.book_copy(self.h, ints(ids), len(ids), into.h, out, r, m, e, k))
        self.move(m, k[1], into)
        self.copy_rows(r, k[0], into)
        into.entries(e, k[2])
        for i, o in zip(ids, out[:len(ids)]):
            into.model[o] = [list(x) for x in self.model[i]]
        return out[:len(ids)]

    def move(self, m, n, to):
        src, dst = [m[2 * i] for i in range(n)], [m[2 * i + 1] for i in range(n)]
        assert len(set(dst)) == n and (to is not self or not set(src) & set(dst))
        held = [list(self.pages[p]) for p in src]
        for p, x in zip(dst, held):
            to.pages[p] = x

    def close(self, ids):
        self.ok(self.lib.book_close(self.h, ints(ids), len(ids)))
        for i in ids:
            del self.model[i]

    def append(self, layer, ids, tokens):
        e = ints([0] * 3 * (sum(len(t) for t in tokens) // BLOCK + len(ids) + 1))
        old = [self.lib.book_length(self.h, i, layer) for i in ids]
        n = self.ok(self.lib.book_append(self.h, layer, ints(ids), ints([len(t) for t in tokens]), len(ids), e))
        self.entries(e, n)
        for i, t, at in zip(ids, tokens, old):
            row = self.lib.book_row(self.h, i)
            block = self.open[row][layer][:at % BLOCK] + t
            b = at // BLOCK
            while len(block) >= BLOCK:
                self.pages[self.table[row][b]][layer] = block[:BLOCK]
                block, b = block[BLOCK:], b + 1
            self.open[row][layer] = block
            self.model[i][layer] += t

    def compact(self):
        k = ints([0, 0])
        most = sum(max(len(x) for x in s) // BLOCK for s in self.model.values())
        m, e = ints([0] * 2 * len(self.pages)), ints([0] * 3 * (most + 1))
        used = self.ok(self.lib.book_compact(self.h, m, e, k))
        self.move(m, k[0], self)
        self.entries(e, k[1])
        for i in self.model:
            row = self.lib.book_row(self.h, i)
            for b in range(max(len(x) for x in self.model[i]) // BLOCK):
                assert self.table[row][b] < used

    def check(self):
        used = set()
        for i, layers in self.model.items():
            row = self.lib.book_row(self.h, i)
            assert 0 <= row < self.sequences
            for layer, want in enumerate(layers):
                assert self.lib.book_length(self.h, i, layer) == len(want)
                got = []
                for b in range(len(want) // BLOCK):
                    got += self.pages[self.table[row][b]][layer]
                assert got + self.open[row][layer][:len(want) % BLOCK] == want
            used |= {self.table[row][b] for b in range(max(len(x) for x in layers) // BLOCK)}
        assert len({self.lib.book_row(self.h, i) for i in self.model}) == len(self.model)
        assert self.lib.book_used(self.h) == len(used)


@pytest.mark.parametrize("seed", range(8))
def test_random_calls(shim, seed):
    rng = random.Random(seed)
    layers = rng.randint(1, 3)
    a, b = Played(shim, layers, 60, 12), Played(shim, layers, 40, 10)
    token = 0

    def fresh(n):
        nonlocal token
        token += n
        return list(range(token - n, token))

    for _ in range(250):
        x = rng.choice([a, a, b])
        ids = list(x.model)
        some = rng.sample(ids, rng.randint(0, len(ids))) if ids else []
        free_pages = len(x.pages) - shim.book_used(x.h)
        what = rng.choice(["open", "append", "append", "append", "fork", "reorder", "copy", "close", "compact"])
        if what == "open" and len(ids) < x.sequences:
            x.open_new(rng.randint(0, min(2, x.sequences - len(ids))))
        elif what == "append" and some:
            counts = [rng.choice([0, 1, 1, 5, 63, 64, 65, 130]) for _ in some]
            need = sum((len(x.model[i][0]) + c) // BLOCK - len(x.model[i][0]) // BLOCK for i, c in zip(some, counts))
            if need <= free_pages:
                for layer in rng.sample(range(layers), layers):
                    x.append(layer, some, [fresh(c) for c in counts])
        elif what == "fork" and ids:
            some = [rng.choice(ids) for _ in range(rng.randint(0, x.sequences - len(ids)))]
            x.fork(some)
        elif what == "reorder" and some:
            x.reorder(some, [rng.choice(ids) for _ in some])
        elif what == "copy" and some:
            y = rng.choice([a, b])
            pages = {x.table[shim.book_row(x.h, i)][k] for i in some for k in range(len(x.model[i][0]) // BLOCK)}
            if len(some) <= y.sequences - len(y.model) and len(pages) <= len(y.pages) - shim.book_used(y.h):
                x.copy(some, y)
        elif what == "close" and some:
            x.close(some)
        elif what == "compact":
            x.compact()
        a.check()
        b.check()


def test_forks_of_the_array_they_fill(shim):
    """The ids and their forks in one array."""
    x = Played(shim, 1, 4, 4)
    ids = ints(x.open_new(2))
    x.append(0, list(ids[:2]), [[1], [2]])
    c = ints([0] * 8)
    a, b = ids[0], ids[1]
    assert shim.book_fork(x.h, ids, 2, ids, c) == 2
    assert [c[0], c[4]] == [shim.book_row(x.h, a), shim.book_row(x.h, b)]


def test_refusals_change_nothing(shim):
    x = Played(shim, 2, 3, 3)
    p, q = x.open_new(2)
    for layer in range(2):
        x.append(layer, [p, q], [list(range(70)), list(range(100, 130))])
    x.check()
    out, scratch = ints([0] * 8), ints([0] * 64)
    x.refused(shim.book_open(x.h, 2, out), "sequences")
    x.refused(shim.book_open(x.h, -1, out), "negative")
    x.refused(shim.book_fork(x.h, ints([p, 2]), 2, out, scratch), "no sequence 2")
    x.refused(shim.book_fork(x.h, ints([p, -1]), 2, out, scratch), "no sequence -1")
    x.refused(shim.book_fork(x.h, ints([p, 7]), 2, out, scratch), "no sequence 7")
    x.refused(shim.book_fork(x.h, ints([p, p]), 2, out, scratch), "sequences")
    x.refused(shim.book_reorder(x.h, ints([p, p]), ints([q, q]), 2, scratch), "twice")
    x.refused(shim.book_reorder(x.h, ints([p]), ints([2]), 1, scratch), "no sequence 2")
    x.refused(shim.book_close(x.h, ints([p, p]), 2), "twice")
    x.refused(shim.book_close(x.h, ints([p, 2]), 2), "no sequence 2")
    x.refused(shim.book_append(x.h, 0, ints([p, p]), ints([1, 1]), 2, scratch), "twice")
    x.refused(shim.book_append(x.h, 0, ints([p, q]), ints([1, -1]), 2, scratch), "negative")
    x.refused(shim.book_append(x.h, 2, ints([p]), ints([1]), 1, scratch), "layer 2")
    x.refused(shim.book_append(x.h, 0, ints([p, q]), ints([64, 98]), 2, scratch), "pages")
    x.refused(shim.book_append(x.h, 0, ints([p]), ints([(1 << 31) - 1]), 1, scratch), "tokens")
    y = Played(shim, 2, 1, 1)
    x.refused(shim.book_copy(x.h, ints([p, q]), 2, y.h, out, scratch, scratch, scratch, ints([0] * 3)), "sequences")
    # Between the layers of a step a sequence cannot be forked, copied or reordered.
    x.append(0, [p], [[7]])
    x.refused(shim.book_fork(x.h, ints([p]), 1, out, scratch), "lengths")
    x.refused(shim.book_reorder(x.h, ints([q]), ints([p]), 1, scratch), "lengths")
    x.refused(shim.book_copy(x.h, ints([p]), 1, x.h, out, scratch, scratch, scratch, ints([0] * 3)), "lengths")
    x.append(1, [p], [[8]])
    x.fork([p])
    x.check()


def test_a_negative_number_of_sequences_is_refused(shim):
    x = Played(shim, 1, 4, 3)
    a, b = x.open_new(2)
    scratch = ints([0] * 64)
    x.refused(shim.book_reorder(x.h, ints([a]), ints([b]), -1, scratch), "negative")
    x.refused(shim.book_fork(x.h, ints([a]), -1, scratch, scratch), "negative")
