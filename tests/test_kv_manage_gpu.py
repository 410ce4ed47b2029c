"""The pool of pages on the GPU against the plain oracle: tables, users and bytes exactly; and a run of everything that a
long conversation over the paged cache calls."""
import math

import numpy as np
import pytest

from oracle import kv_pages as okv, long_context as olc
from tests._dev import down, empty, up
from tests.test_head_form_gpu import Form, check
from tests.test_kv_pages_gpu import attn_tolerance, matches, normal
from vte_amd.kernels import KVPages, KVRows, KVTables

pytestmark = pytest.mark.gpu


class Pools:
    """Layers' pools of random bytes, a table and users, on the device and for the oracle (a page's content: its bytes)."""

    def __init__(self, hip, K, rng, table, n_pages, page=16, n_layers=2, n_kv=2, hd=64, more=()):
        self.hip, self.K, self.page, self.n_pages = hip, K, page, n_pages
        table = np.array(table, np.int32)
        refs = np.zeros(n_pages, np.int32)
        np.add.at(refs, table[(table >= 0) & (table < n_pages)], 1)
        for p in more:
            refs[p] += 1
        shapes = [(n_kv, page, hd), (n_kv, page // 16, hd, 16), (n_kv, page // 16), (n_kv, page // 16)]
        self.host = [[rng.integers(0, 256, (n_pages, *s), dtype=np.uint8) for s in shapes] for _ in range(n_layers)]
        self.dev = [[up(hip, x) for x in layer] for layer in self.host]
        self.layers = (KVPages * n_layers)(*[KVPages.of(*d, n_pages, page, n_kv, hd) for d in self.dev])
        self.table, self.refs = up(hip, table), up(hip, refs)
        self.t = KVTables.of(self.table, self.refs, *table.shape, n_pages, page)
        self.missing = up(hip, np.full(1, -5, np.int32))
        self.ref = olc.Pool(table, refs, page, range(n_pages))

    def ints(self, x):
        return None if x is None else up(self.hip, np.array(x, np.int32))

    def free(self, seqs, n=None, **kw):
        end = kw.pop("end", None)
        self.ref.free(range(n) if seqs is None else seqs, end=end, **kw)
        self.K.kv_pages_free(self.t, n or len(seqs), seqs=self.ints(seqs), end=self.ints(end), stream=self.hip.stream, **kw)

    def reserve(self, seqs, start, count, stop=None):
        want = self.ref.reserve(range(len(start)) if seqs is None else seqs, start, count, stop)
        self.K.kv_pages_reserve(self.t, len(start), self.ints(start), count, self.missing, seqs=self.ints(seqs),
                                stop=self.ints(stop), stream=self.hip.stream)
        assert down(self.missing)[0] == want

    def fork(self, parents, children, lengths):
        want = self.ref.fork(parents, children, lengths)
        n = len(parents)
        size = self.K.kv_pages_fork_scratch_bytes(n)
        self.K.kv_pages_fork(self.layers, self.t, n, self.ints(parents), self.ints(children), self.ints(lengths), self.missing,
                             empty(self.hip, size, np.uint8), size, stream=self.hip.stream)
        assert down(self.missing)[0] == want

    def compact(self):
        where, used = self.ref.compact()
        n = self.K.kv_pages_compact_scratch_bytes(self.t)
        w, u = up(self.hip, np.full(self.n_pages, 77, np.int32)), up(self.hip, np.full(1, 77, np.int32))
        self.K.kv_pages_compact(self.layers, self.t, w, u, up(self.hip, np.full(n, 0xFF, np.uint8)), n, stream=self.hip.stream)
        assert np.array_equal(down(w), where) and down(u)[0] == used

    def check(self):
        assert np.array_equal(down(self.table), self.ref.table)
        assert np.array_equal(down(self.refs), self.ref.refs)
        for host, dev in zip(self.host, self.dev):
            for x, d in zip(host, dev):
                assert np.array_equal(down(d), x[self.ref.content])


def scattered(rng, rows, width, n_pages, used):
    """A table with `used` pages in any order and places."""
    t = np.full(rows * width, -1)
    t[rng.permutation(rows * width)[:used]] = rng.permutation(n_pages)[:used]
    return t.reshape(rows, width)


@pytest.mark.parametrize("page,n_kv,hd,n_layers,n", [(16, 1, 64, 1, 1), (64, 2, 128, 3, 17), (256, 3, 64, 2, 9),
                                                     (32, 5, 128, 70, 5), (4096, 2, 128, 1, 2)])
def test_copy(hip, K, page, n_kv, hd, n_layers, n):
    """Pairs in any order in every layer (more than one launch's), some of which are no pages."""
    rng = np.random.default_rng(page + n)
    n_pages = 2 * n + 3
    p = Pools(hip, K, rng, [[-1]], n_pages, page, n_layers, n_kv, hd)
    order = rng.permutation(n_pages)
    src, dst = order[:n].astype(np.int32), order[n:2 * n].astype(np.int32)
    if n > 4:
        src[1], dst[2], dst[3] = -1, n_pages, 2 ** 31 - 1
    K.kv_pages_copy(p.layers, up(hip, src), up(hip, dst), n, stream=hip.stream)
    for a, b in zip(src, dst):
        if 0 <= a < n_pages and 0 <= b < n_pages:
            p.ref.content[b] = p.ref.content[a]
    p.check()


@pytest.mark.parametrize("page", [16, 64])
def test_free(hip, K, page):
    """Whole sequences, those behind a window, from an end on; shared pages stay while one uses them; entries that are no
    page; sequences of no table; the same sequence twice."""
    rng = np.random.default_rng(page)
    table = scattered(rng, 6, 9, 60, 40)
    table[1, :4] = table[0, :4]       # shared (the pages that were there are free now)
    table[2, 5] = 10 ** 6
    p = Pools(hip, K, rng, table, 60, page, more=[int(table[0, 2])] if table[0, 2] >= 0 else [])
    p.free([0, 3, 77, -1])
    p.check()
    p.free(None, n=5, keep=page + 1, end=[5 * page, 5 * page + 3, -1, 9 * page + 100, 2], behind=2 * page)
    p.check()
    p.free([2, 2, 2], keep=2 * page)
    p.check()
    p.free([5], keep=2 ** 31 - 1)
    p.free([5], end=[2 ** 31 - 1], behind=2 ** 31 - 1)
    p.check()
    p.free(None, n=6)
    p.check()
    assert (down(p.table) == -1).all()


@pytest.mark.parametrize("free", [5, 60, 900])
def test_reserve(hip, K, free):
    """Decoded tokens, chunks from places inside pages, up to given ends, past the table; enough pages and too few."""
    rng = np.random.default_rng(free)
    used = 5000
    table = scattered(rng, 400, 20, used + free, used)
    p = Pools(hip, K, rng, table, used + free, n_layers=1, n_kv=1)
    p.reserve(None, [int(x) for x in rng.integers(0, 319, 40)], 1)
    p.check()
    p.reserve([3, 399, 400, -2, 7, 9], [0, 17, 0, 0, -1, 300], 100)
    p.check()
    p.reserve([11, 12, 13, 14], [5, 100, 40, 319], 2 ** 30, stop=[33, 90, 41, 2 ** 31 - 1])
    p.check()
    p.reserve([int(x) for x in rng.permutation(400)[:300]], [int(x) for x in rng.integers(0, 330, 300)], 60)
    p.check()


def test_reserve_for_more_slots_than_a_block_has_threads(hip, K):
    """1500 sequences of an empty table, 3 pages each, from a pool whose free pages lie far apart."""
    rng = np.random.default_rng(8)
    n_pages = 70001
    p = Pools(hip, K, rng, np.full((1500, 4), -1), n_pages, n_layers=1, n_kv=1, more=rng.permutation(n_pages)[:66000])
    p.reserve(None, [16] * 1500, 40)
    p.check()
    p.free(list(range(0, 1500, 2)), keep=30)
    p.reserve(None, [0] * 1500, 33)
    p.check()


@pytest.mark.parametrize("n_pages", [16383, 16386, 50003])
@pytest.mark.parametrize("shift", [1, 2, 3])
def test_reserve_from_unaligned_users(hip, K, n_pages, shift):
    """Users at any 4-byte address, pools around the pages that are looked at together, the last pages among the free."""
    rng = np.random.default_rng(n_pages + shift)
    refs = np.ones(n_pages, np.int32)
    free = np.sort(np.concatenate([rng.permutation(n_pages - 3)[:30], [n_pages - 1, n_pages - 2]]))
    refs[free] = 0
    refs[free[3]] = -7  # (counts below 0 are none)
    d = up(hip, np.concatenate([np.zeros(shift, np.int32), refs]))
    table, missing = up(hip, np.full((40, 2), -1, np.int32)), up(hip, np.zeros(1, np.int32))
    t = KVTables.of(table, d.ptr + 4 * shift, 40, 2, n_pages, 16)
    K.kv_pages_reserve(t, 40, up(hip, np.full(40, 20, np.int32)), 1, missing, stream=hip.stream)
    got, now = down(table), down(d)[shift:]
    assert np.array_equal(got[:32, 1], free) and (got[32:] == -1).all() and (got[:, 0] == -1).all() and down(missing)[0] == 8
    assert (now == 1).all() and not down(d)[:shift].any()


def test_the_same_sequence_twice_costs_no_page(hip, K):
    rng = np.random.default_rng(9)
    p = Pools(hip, K, rng, np.full((3, 4), -1), 40)
    K.kv_pages_reserve(p.t, 4, p.ints([0, 0, 0, 0]), 64, p.missing, seqs=p.ints([1, 1, 2, 1]), stream=hip.stream)
    t, refs = down(p.table), down(p.refs)
    assert (t[0] == -1).all() and (t[1:] >= 0).all() and len(np.unique(t[1:])) == 8
    assert refs.sum() == 8 and (refs[t[1:]] == 1).all()
    K.kv_pages_free(p.t, 3, seqs=p.ints([1, 1, 1]), stream=hip.stream)
    assert down(p.refs).sum() == 4 and (down(p.refs) >= 0).all()


@pytest.mark.parametrize("times", [300, 1500])
def test_a_sequence_many_times_keeps_its_lowest_pages(hip, K, times):
    """Two entries of one sequence asked for over and over, then those of others: the same pages every time.  (1024 slots
    are served together; later ones see what the earlier ones were given.)"""
    rng = np.random.default_rng(times)
    first = min(2 * times, 1024)  # pages taken for sequence 1
    for _ in range(5):
        p = Pools(hip, K, rng, [[-1, -1], [10 ** 6, -9], [-1, -1]], 4000, n_layers=1, n_kv=1)
        seqs = [1] * times + [2, 0]
        p.K.kv_pages_reserve(p.t, len(seqs), p.ints([0] * len(seqs)), 32, p.missing, seqs=p.ints(seqs), stream=hip.stream)
        assert np.array_equal(down(p.table), [[first + 2, first + 3], [0, 1], [first, first + 1]])
        refs = down(p.refs)
        assert refs.sum() == 6 and (refs[down(p.table)] == 1).all() and down(p.missing)[0] == 0


@pytest.mark.parametrize("page,n_layers,n_kv,hd", [(16, 1, 1, 64), (64, 3, 2, 128), (32, 66, 1, 64)])
def test_fork(hip, K, page, n_layers, n_kv, hd):
    """One parent and several, lengths of whole pages, of none, inside pages, past the parent's pages and the table's end,
    children that have pages, holes of the parent; a child that is its own parent, sequences of no table."""
    rng = np.random.default_rng(page)
    table = np.full((14, 6), -1)
    order = rng.permutation(70)
    table[0, :5], table[1, :3], table[2, :6] = order[:5], order[5:8], order[8:14]
    table[2, 3] = 99999
    table[5, :4], table[9, 2:5] = order[20:24], order[24:27]
    p = Pools(hip, K, rng, table, 70, page, n_layers, n_kv, hd)
    p.fork([0, 0, 1, 2, 2, 0], [3, 4, 5, 6, 7, 8], [4 * page + 1, 5 * page, 2 * page - 1, 3 * page + 2, 100 * page + 5, 0])
    p.check()
    p.fork([3, 3, 4, 77, 0, -1, 1], [9, 10, 11, 12, 0, 13, 1400], [4 * page + 1, page // 2, 5, 5, 5, 5, 5])
    p.check()
    p.fork([0], [12], [-3])
    p.free([0, 3, 4])
    p.check()


def test_forks_of_more_entries_than_a_block_has_threads(hip, K):
    """60 children of 3 parents in tables of 24 pages, a launch that shares before the one that finds pages; then the number
    of missing pages is not asked for."""
    rng = np.random.default_rng(19)
    table = np.full((70, 24), -1)
    order = rng.permutation(300)
    table[0, :20], table[1, :3], table[2, :24] = order[:20], order[20:23], order[23:47]
    table[5, 3:9], table[60, ::2] = order[50:56], order[60:72]
    p = Pools(hip, K, rng, table, 300, page=32, n_layers=2, n_kv=1)
    par = [i % 3 for i in range(60)]
    p.fork(par, list(range(3, 63)), [int(x) for x in rng.integers(0, 800, 60)])
    p.check()
    p.ref.fork([3, 0], [65, 66], [40, 639])
    K.kv_pages_fork(p.layers, p.t, 2, p.ints([3, 0]), p.ints([65, 66]), p.ints([40, 639]), None, empty(hip, 16, np.uint8), 16,
                    stream=hip.stream)
    p.ref.reserve([64], [5], 70)
    K.kv_pages_reserve(p.t, 1, p.ints([5]), 70, None, seqs=p.ints([64]), stream=hip.stream)
    p.check()


def test_forks_without_free_pages(hip, K):
    """The first children of the list get the pages there are; the others' last entry is none."""
    rng = np.random.default_rng(11)
    table = np.full((40, 3), -1)
    table[0, :2] = 7, 3
    p = Pools(hip, K, rng, table, 30, more=list(range(8, 21)))
    p.fork([0] * 39, list(range(1, 40)), [20] * 39)
    p.check()
    assert (down(p.table)[1:, 1] < 0).sum() == 39 - 15


@pytest.mark.parametrize("n_pages,used", [(1, 0), (1, 1), (10, 4), (300, 150), (1024, 1024), (1025, 700), (5000, 2048), (5000, 4999),
                                          (4096, 1024), (8192, 5000), (8193, 1024), (20001, 15000)])
def test_compact(hip, K, n_pages, used):
    """Pools from empty to full, their sizes and numbers of used pages at and beside the chunks' borders, shared pages,
    users that no table names; every block counting all pages, and a launch of counts before."""
    rng = np.random.default_rng(n_pages + used)
    rows = 1 + used // 13
    table = scattered(rng, rows, 14, n_pages, used - used // 9)
    table[0, 0] = table[0].max()      # twice, or no page
    rest = np.setdiff1d(np.arange(n_pages), table)
    p = Pools(hip, K, rng, table, n_pages, n_layers=2, n_kv=1, more=rest[:used // 9])
    p.compact()
    p.check()
    p.compact()
    p.check()
    p.free(None, n=min(rows, 3))
    p.compact()
    p.check()


def test_compact_of_many_layers_and_stray_entries(hip, K):
    """More layers than a launch takes; entries that are no page, or name a free one."""
    rng = np.random.default_rng(12)
    table = scattered(rng, 4, 10, 90, 30)
    p = Pools(hip, K, rng, table, 90, page=32, n_layers=67, n_kv=1)
    free = np.setdiff1d(np.arange(90), table)
    stray = np.array(p.ref.table)
    gaps = np.argwhere(stray == -1)
    for (r, c), x in zip(gaps, [int(free[-1]), 10 ** 8, -9, int(free[0])]):
        stray[r, c] = x
    p.ref.table = stray
    p.table.upload(stray.astype(np.int32))
    p.compact()
    p.check()


def test_random_lives(hip, K):
    """Forty rounds of everything, the oracle beside: users are the entries' numbers throughout."""
    rng = np.random.default_rng(13)
    p = Pools(hip, K, rng, np.full((24, 8), -1), 100, page=16, n_layers=2, n_kv=1)
    length = np.zeros(24, int)
    for step in range(40):
        seqs = [int(x) for x in rng.permutation(24)[:8]]
        start = [int(length[s]) for s in seqs]
        p.reserve(seqs, start, 30)
        length[seqs] = np.minimum(length[seqs] + 30, 128)
        a = rng.permutation(24)
        n = int(rng.integers(1, 6))
        par, kid = [int(x) for x in a[:n]], [int(x) for x in a[10:10 + n]]
        lens = [int(rng.integers(0, length[x] + 1)) for x in par]
        p.fork(par, kid, lens)
        length[kid] = lens
        gone = [int(x) for x in a[20:22]]
        p.free(gone)
        length[gone] = 0
        p.free(None, n=24, keep=4, end=[int(x) for x in length], behind=40)
        if step % 5 == 4:
            p.compact()
        p.check()
        count = np.zeros(100, int)
        np.add.at(count, p.ref.table[p.ref.table >= 0], 1)
        assert np.array_equal(count, p.ref.refs)


def test_captured_calls_follow_staged_arguments(hip, K):
    """Reserve, fork, free and compact as one graph, replayed four times with other arguments and eager work between."""
    rng = np.random.default_rng(15)
    p = Pools(hip, K, rng, scattered(rng, 12, 6, 60, 20), 60, page=16, n_layers=2, n_kv=1)
    start, par, kid, lens, gone = (p.ints([0] * 3) for _ in range(5))
    n, m = K.kv_pages_fork_scratch_bytes(3), K.kv_pages_compact_scratch_bytes(p.t)
    s1, s2, w, u = empty(hip, n, np.uint8), empty(hip, m, np.uint8), empty(hip, 60, np.int32), empty(hip, 1, np.int32)
    st = hip.stream
    hip.stream_synchronize()
    hip.stream_begin_capture()
    K.kv_pages_reserve(p.t, 3, start, 40, p.missing, stream=st)
    K.kv_pages_fork(p.layers, p.t, 3, par, kid, lens, p.missing, s1, n, stream=st)
    K.kv_pages_free(p.t, 3, seqs=gone, stream=st)
    K.kv_pages_compact(p.layers, p.t, w, u, s2, m, stream=st)
    g = hip.stream_end_capture()
    ge = hip.graph_instantiate(g)
    try:
        for _ in range(4):
            a = [int(x) for x in rng.permutation(12)]
            args = [[int(x) for x in rng.integers(0, 60, 3)], a[:3], a[3:6], [int(x) for x in rng.integers(0, 90, 3)], a[6:9]]
            for d, x in zip((start, par, kid, lens, gone), args):
                d.upload(np.array(x, np.int32))
            hip.graph_launch(ge)
            hip.synchronize()
            p.ref.reserve(range(3), args[0], 40)
            p.ref.fork(*args[1:4])
            p.ref.free(args[4])
            where, used = p.ref.compact()
            assert np.array_equal(down(w), where) and down(u)[0] == used
            p.check()
            p.free([a[10]])
            p.reserve([a[11]], [0], 50)
            p.check()
    finally:
        hip.graph_exec_destroy(ge)
        hip.graph_destroy(g)


def test_pages_beyond_32_bits(hip, K):
    """A pool of 5 GiB of K: pages beyond 2^32 bytes are copied and moved to and from their places."""
    page, n_kv, hd = 4096, 2, 128
    n_pages = 5 * 2 ** 30 // (page * n_kv * hd)
    size, blocks, one = n_pages * page * n_kv * hd, n_pages * n_kv * page // 16, page * n_kv * hd
    d = {n: hip.safe_malloc(s, "pool") for n, s in (("k", size), ("v", size), ("ke", blocks), ("ve", blocks))}
    try:
        rng = np.random.default_rng(16)
        pages = KVPages.of(d["k"], d["v"], d["ke"], d["ve"], n_pages, page, n_kv, hd)
        L = (KVPages * 1)(pages)
        # page n_pages - 1 gets rows through the append; copied to page 2, then compacted to page 0
        rows = [normal(rng, (33, n_kv, hd), "f16") for _ in "kv"]
        table, off = up(hip, np.array([[n_pages - 1]], np.int32)), up(hip, np.zeros(1, np.int32))
        r = KVRows.of(1, 33, 33, up(hip, np.array([0, 33], np.int32)), off, table, 1)
        K.kv_pages_append(pages, r, *[up(hip, x) for x in rows], stream=hip.stream)

        def read(entry):
            table.upload(np.array([[entry]], np.int32))
            out = [empty(hip, (1, 33, n_kv, hd), np.float16) for _ in "kv"]
            K.kv_pages_read(pages, r, *out, 33, stream=hip.stream)
            return [down(x).copy() for x in out]
        want = read(n_pages - 1)
        assert np.abs(want[0][0].astype(np.float64) - rows[0]).max() < 0.1
        K.kv_pages_copy(L, up(hip, np.array([n_pages - 1], np.int32)), up(hip, np.array([2], np.int32)), 1, stream=hip.stream)
        assert all(np.array_equal(a, b) for a, b in zip(read(2), want))

        def attend(entry):
            table.upload(np.array([[entry]], np.int32))
            out = []
            for new in (1, 20):
                rr = KVRows.of(1, new, new, up(hip, np.array([0, new], np.int32)), up(hip, np.array([33 - new], np.int32)), table, 1)
                n, o = K.attn_pages_window_scratch_bytes(pages, rr, 4, 9, 2), empty(hip, (new, 4, hd), np.float16)
                K.attn_pages_window(pages, rr, up(hip, q[:new]), o, 4, 0.1, 9, 2, empty(hip, n, np.uint8), n, stream=hip.stream)
                out.append(down(o).copy())
            return out
        q = normal(rng, (20, 4, hd), "f16")
        far, near = attend(n_pages - 1), attend(2)
        assert all(np.array_equal(a, b) and np.abs(a).max() > 0 for a, b in zip(far, near))
        table.upload(np.array([[n_pages - 1]], np.int32))
        refs = np.zeros(n_pages, np.int32)
        refs[-1] = 1
        t = KVTables.of(table, up(hip, refs), 1, 1, n_pages, page)
        m = K.kv_pages_compact_scratch_bytes(t)
        w, u = empty(hip, n_pages, np.int32), empty(hip, 1, np.int32)
        K.kv_pages_compact(L, t, w, u, empty(hip, m, np.uint8), m, stream=hip.stream)
        assert down(table)[0, 0] == 0 and down(u)[0] == 1 and down(w)[-1] == 0
        assert all(np.array_equal(a, b) for a, b in zip(read(0), want))
    finally:
        hip.synchronize()
        for x in d.values():
            hip.safe_free(x)


# ---------------------------------------------------------------------------- together
def test_a_long_conversation(hip, K):
    """Two layers.  A prompt is taken in in chunks (room, heads normed and rotated into the pages, windowed attention),
    three answers fork from it and decode 40 tokens as one captured graph that also makes room and gives back what falls out
    of the window; the pool is compacted now and then.  Every result is the oracle's on the device's own pages, the pages
    hold what was appended, users are what the tables say, and the pool stays small."""
    rng = np.random.default_rng(21)
    page, n_kv, n_q, hd, window, sinks, n_layers, B = 16, 2, 6, 64, 50, 5, 2, 4
    p = Pools(hip, K, rng, np.full((B, 24), -1), 40, page, n_layers, n_kv, hd)
    f = Form(hip, rng, hd, 32, True, amplitude=1.1)
    scale, st, prompt = 1 / math.sqrt(hd), hip.stream, 150
    rows_k = [[np.zeros((300, n_kv, hd)) for _ in range(B)] for _ in range(n_layers)]   # what each sequence was given
    tol_k = [[np.zeros((300, n_kv, hd)) for _ in range(B)] for _ in range(n_layers)]
    rows_v = [[np.zeros((300, n_kv, hd)) for _ in range(B)] for _ in range(n_layers)]

    def live(b, n):
        """Tokens of sequence b that have a page."""
        t = down(p.table)[b]
        return np.array([t[i // page] >= 0 for i in range(n)])

    def check_layer(l, b, first, q, out):
        """Rows of layer l from position `first` of sequence b: q as it was turned on the device, results, and pages."""
        table, (k, v, ke, ve) = down(p.table)[b], [down(x) for x in p.dev[l]]
        n = first + len(q)
        kc, kx = okv.unpool(k, ke.view(np.int8), table, page, False)
        vc, vx = okv.unpool(v, ve.view(np.int8), table, page, True)
        K_, V_ = (c * 2.0 ** np.repeat(x, 16, 0)[:, :, None] for c, x in ((kc, kx), (vc, vx)))
        have = live(b, n)
        lo = n - len(q) - window if n > window else 0
        for t in range(max(lo, 0), n):  # within a step (of raises as well) of what went in
            if have[t]:
                step = 2.0 ** np.array([kx[t // 16], vx[t // 16]])[:, :, None]
                assert (np.abs(K_[t] - rows_k[l][b][t]) <= step[0] + tol_k[l][b][t]).all(), (l, b, t)
                assert (np.abs(V_[t] - rows_v[l][b][t]) <= step[1]).all(), (l, b, t)
        for i in range(len(q)):
            seen = olc.sees(first + i, len(K_), window, sinks)
            assert have[seen[:n]].all()
            o, mag, big = okv.attention(q[i], K_, V_, first + i, scale, seen)
            assert matches("f16", out[i].astype(np.float64), o, attn_tolerance("f16", hd, o, mag, big, np.abs(V_[seen]).max())).all()

    # ---- the prompt, in chunks ----
    off = up(hip, np.zeros(B, np.int32))
    for lo in range(0, prompt, 60):
        n = min(60, prompt - lo)
        off.upload(np.array([lo, -1, -1, -1], np.int32))
        K.kv_pages_reserve(p.t, 1, off, n, p.missing, stream=st)
        assert down(p.missing)[0] == 0
        for l in range(n_layers):
            wide = normal(rng, (n, n_q + 2 * n_kv, hd), "f16")
            dw, do, size, ld = up(hip, wide), empty(hip, (n, n_q, hd), np.float16), 2, wide.shape[1] * hd
            r = KVRows.of(1, n, n, up(hip, np.array([0, n], np.int32)), off, p.table, 24)
            K.kv_pages_append_norm(p.layers[l], r, f.c, dw.ptr + n_q * hd * size, dw.ptr + (n_q + n_kv) * hd * size, q=dw, q_out=do,
                                   n_q=n_q, k_stride=ld, v_stride=ld, q_stride=ld, stream=st)
            q = down(do).copy()
            at = lo + np.arange(n)
            check("f16", q, *f.of(wide[:, :n_q], at, False))
            rows_k[l][0][at], tol_k[l][0][at] = f.of(wide[:, n_q:n_q + n_kv], at, True)
            rows_v[l][0][at] = wide[:, n_q + n_kv:]
            m = K.attn_pages_window_scratch_bytes(p.layers[l], r, n_q, window, sinks)
            K.attn_pages_window(p.layers[l], r, do, do, n_q, scale, window, sinks, empty(hip, m, np.uint8), m, stream=st)  # in place
            check_layer(l, 0, lo, q, down(do))
        off.upload(np.array([lo + n, -1, -1, -1], np.int32))
        K.kv_pages_free(p.t, B, keep=sinks, end=off, behind=window - 1, stream=st)
        assert (down(p.refs) > 0).sum() <= 1 + (window + n) // page + 2

    # ---- answers ----
    n = K.kv_pages_fork_scratch_bytes(3)
    K.kv_pages_fork(p.layers, p.t, 3, p.ints([0, 0, 0]), p.ints([1, 2, 3]), p.ints([prompt] * 3), p.missing,
                    empty(hip, n, np.uint8), n, stream=st)
    for l in range(n_layers):
        for b in (1, 2, 3):
            rows_k[l][b], tol_k[l][b], rows_v[l][b] = rows_k[l][0].copy(), tol_k[l][0].copy(), rows_v[l][0].copy()
    r = KVRows.of(B, B, 1, None, off, p.table, 24)
    wide = [empty(hip, (B, n_q + 2 * n_kv, hd), np.float16) for _ in range(n_layers)]
    qs, outs = ([empty(hip, (B, n_q, hd), np.float16) for _ in range(n_layers)] for _ in range(2))
    m = K.attn_pages_window_scratch_bytes(p.layers[0], r, n_q, window, sinks)
    scratch, ld = empty(hip, m, np.uint8), (n_q + 2 * n_kv) * hd
    hip.stream_synchronize()
    hip.stream_begin_capture()
    K.kv_pages_reserve(p.t, B, off, 1, p.missing, stream=st)
    for l in range(n_layers):
        x = wide[l].ptr
        K.kv_pages_append_norm(p.layers[l], r, f.c, x + n_q * hd * 2, x + (n_q + n_kv) * hd * 2, q=x, q_out=qs[l], n_q=n_q,
                               k_stride=ld, v_stride=ld, q_stride=ld, stream=st)
        K.attn_pages_window(p.layers[l], r, qs[l], outs[l], n_q, scale, window, sinks, scratch, m, stream=st)
    K.kv_pages_free(p.t, B, keep=sinks, end=off, behind=window, stream=st)  # (off: the row just written)
    g = hip.stream_end_capture()
    ge = hip.graph_instantiate(g)
    cm = K.kv_pages_compact_scratch_bytes(p.t)
    try:
        for step in range(40):
            pos = prompt + step
            off.upload(np.full(B, pos, np.int32))
            host = [normal(rng, (B, n_q + 2 * n_kv, hd), "f16", 2.0 ** rng.uniform(-3, 3)) for _ in range(n_layers)]
            for d, x in zip(wide, host):
                d.upload(x)
            hip.graph_launch(ge)
            hip.synchronize()
            assert down(p.missing)[0] == 0
            for l in range(n_layers):
                k, t = f.of(host[l][:, n_q:n_q + n_kv], [pos] * B, True)
                for b in range(B):
                    rows_k[l][b][pos], tol_k[l][b][pos], rows_v[l][b][pos] = k[b], t[b], host[l][b, n_q + n_kv:]
                check("f16", down(qs[l]), *f.of(host[l][:, :n_q], [pos] * B, False))
                if step % 3 == 0:
                    for b in range(B):
                        check_layer(l, b, pos, down(qs[l])[b:b + 1], down(outs[l])[b:b + 1])
            if step % 10 == 9:
                w, u = empty(hip, 40, np.int32), empty(hip, 1, np.int32)
                K.kv_pages_compact(p.layers, p.t, w, u, empty(hip, cm, np.uint8), cm, stream=st)
                used = int(down(u)[0])
                assert down(p.table).max() == used - 1
            t, refs = down(p.table), down(p.refs)
            count = np.zeros(40, int)
            np.add.at(count, t[t >= 0], 1)
            assert np.array_equal(count, refs) and (refs > 0).sum() <= 1 + B * (window // page + 2)
    finally:
        hip.graph_exec_destroy(ge)
        hip.graph_destroy(g)
