"""Room for tokens that follow others, where pages ran out meanwhile: tables and users against the plain oracle, and that
nothing of a page's former user is ever seen."""
import math

import numpy as np
import pytest

from oracle import kv_pages as okv, long_context as olc
from tests._dev import down, empty, up
from tests.test_kv_manage_gpu import Pools, scattered
from tests.test_kv_pages_gpu import attn_tolerance, matches, normal
from vte_amd.kernels import KVRows

pytestmark = pytest.mark.gpu


def extend(p, seqs, start, count, stop=None):
    want = p.ref.reserve(range(len(start)) if seqs is None else seqs, start, count, stop, follow=True)
    p.K.kv_pages_extend(p.t, len(start), p.ints(start), count, p.missing, seqs=p.ints(seqs), stop=p.ints(stop),
                        stream=p.hip.stream)
    assert down(p.missing)[0] == want
    p.check()


@pytest.mark.parametrize("free", [5, 60, 900])
def test_extend(hip, K, free):
    """Tokens and chunks from places inside pages and from their beginnings, up to given ends, past the table; enough pages
    and too few; entries that are no page; sequences of no table."""
    rng = np.random.default_rng(free)
    used = 5000
    table = scattered(rng, 400, 20, used + free, used)
    table[7, 3] = 10 ** 8
    p = Pools(hip, K, rng, table, used + free, n_layers=1, n_kv=1)
    extend(p, None, [int(x) for x in rng.integers(0, 319, 40)], 1)
    extend(p, [3, 399, 400, -2, 7, 9, 7], [0, 17, 0, 0, -1, 300, 50], 100)
    extend(p, [11, 12, 13, 14], [5, 96, 40, 319], 2 ** 30, stop=[33, 90, 41, 2 ** 31 - 1])
    extend(p, [int(x) for x in rng.permutation(400)[:300]], [int(x) for x in rng.integers(0, 330, 300)], 60)
    p.K.kv_pages_extend(p.t, 1, p.ints([5]), 1, None, stream=hip.stream)  # (the number is not asked for)
    p.ref.reserve([0], [5], 1, follow=True)
    p.check()


def test_extend_after_a_fork_without_pages(hip, K):
    """Children whose begun page could not be copied go on behind it when there are pages again."""
    rng = np.random.default_rng(5)
    table = np.full((12, 4), -1)
    table[0, :2] = 7, 3
    p = Pools(hip, K, rng, table, 12, more=[0, 1, 2, 4, 5, 6])
    p.fork([0] * 8, list(range(1, 9)), [20] * 8)
    assert (down(p.table)[1:9, 1] < 0).sum() == 4
    p.free([1, 2, 3])
    extend(p, list(range(4, 9)), [20] * 5, 1)
    assert (down(p.table)[5:9, 1] < 0).all()
    extend(p, list(range(4, 9)), [32] * 5, 1)
    p.free([4, 5])
    extend(p, list(range(4, 9)), [33] * 5, 16)


@pytest.mark.parametrize("left", ["large", "nan"])
@pytest.mark.parametrize("chunk", [1, 7])
def test_a_former_users_tokens_are_never_seen(hip, K, left, chunk):
    """A sequence runs out of pages inside its third one, and another one ends, whose pages hold huge values or NaN.  Tokens
    without a page are not seen, nor are the former user's, then or later; the next page is a whole one again."""
    rng = np.random.default_rng(6)
    page, n_kv, n_q, hd, window, sinks = 32, 2, 6, 64, 60, 3
    p = Pools(hip, K, rng, [[0, 1, -1, -1, -1], [2, 3, 4, -1, -1]], 5, page, 1, n_kv, hd)
    k, v, ke, ve = p.dev[0]
    for x, kind in ((k, 255), (v, 255), (ke, None), (ve, None)):
        h = down(x).copy()
        h[2:] = kind if kind else (np.uint8(60) if left == "large" else np.uint8(128))  # (-128: NaN)
        x.upload(h)
    rows = np.zeros((2, 160, n_kv, hd))
    given = np.zeros(160, bool)
    off, start = up(hip, np.array([0, -1], np.int32)), up(hip, np.array([0, 0, 0], np.int32))
    pos = 0
    while pos < 130:
        n = min(60 if pos == 0 else chunk, 130 - pos)
        if pos > 75 and down(p.table)[1, 0] >= 0:
            K.kv_pages_free(p.t, 1, seqs=p.ints([1]), stream=hip.stream)
        off.upload(np.array([pos, -1], np.int32))
        start.upload(np.array([0, n, n], np.int32))
        K.kv_pages_extend(p.t, 1, off, n, p.missing, stream=hip.stream)
        table = down(p.table)[0]
        here = np.array([table[t // page] >= 0 for t in range(pos, pos + n)])
        assert np.array_equal(here, [not 64 <= t < 96 for t in range(pos, pos + n)])
        assert down(p.missing)[0] == (not here.all())
        given[pos:pos + n] = here
        x = [normal(rng, (n, n_kv, hd), "f16") for _ in "kv"]
        rows[:, pos:pos + n] = x
        r = KVRows.of(2, n, n, start, off, p.table, 5)
        K.kv_pages_append(p.layers[0], r, *[up(hip, a) for a in x], stream=hip.stream)
        out = [empty(hip, (2, 160, n_kv, hd), np.float32) for _ in "kv"]
        K.kv_pages_read(p.layers[0], r, *out, 160, dtype="f32", stream=hip.stream)
        kv = [down(o)[0].astype(np.float64) for o in out]
        for got, want in zip(kv, rows):
            live = given[:pos + n]
            assert not got[:pos + n][~live].any()
            assert (np.abs(got - want)[:pos + n][live] <= 2 * np.abs(want).max() / 127).all()  # (a step, raises included)
        q = normal(rng, (n, n_q, hd), "f16")
        scale = 1 / math.sqrt(hd)
        for win in (None, window):
            o = empty(hip, q.shape, np.float16)
            if win is None:
                m = K.attn_pages_scratch_bytes(p.layers[0], r, n_q)
                K.attn_pages(p.layers[0], r, up(hip, q), o, n_q, scale, empty(hip, m, np.uint8), m, stream=hip.stream)
            else:
                m = K.attn_pages_window_scratch_bytes(p.layers[0], r, n_q, win, sinks)
                K.attn_pages_window(p.layers[0], r, up(hip, q), o, n_q, scale, win, sinks, empty(hip, m, np.uint8), m,
                                    stream=hip.stream)
            got = down(o).astype(np.float64)
            for i in range(n):
                seen = given & (olc.sees(pos + i, 160, win, sinks) if win else np.arange(160) <= pos + i)
                want, mag, big = okv.attention(q[i], *kv, pos + i, scale, seen)
                tol = attn_tolerance("f16", hd, want, mag, big, np.abs(kv[1][seen]).max())
                assert matches("f16", got[i], want, tol).all(), (pos, i, win)
        pos += n
    assert given.sum() == 130 - 32


# ---------------------------------------------------------------------------- a sequence twice in the list
@pytest.mark.parametrize("call", ["kv_pages_reserve", "kv_pages_extend"])
@pytest.mark.parametrize("free", [0, 1, 2, 3, 4, 8, 9, 40])
def test_a_sequence_twice_takes_no_page_from_others(hip, K, call, free):
    """With some ten entries to fill, one sequence many times over, those first in the list get the pages there are; the rest is
    missing, once for each time it is asked for."""
    rng = np.random.default_rng(free)
    seqs = [1, 1, 1, 2, 1, 3, 2, 2, 4, 1, 5, 5, 4, 0]
    start = [0, 5, 16, 0, 0, 20, 0, 16, 7, 16, 0, 0, 0, 33]
    p = Pools(hip, K, rng, np.full((6, 4), -1), 50, n_layers=1, n_kv=1, more=rng.permutation(50)[:50 - free])
    want = p.ref.reserve(seqs, start, 17, follow=call == "kv_pages_extend")
    getattr(K, call)(p.t, len(seqs), p.ints(start), 17, p.missing, seqs=p.ints(seqs), stream=hip.stream)
    table, refs = down(p.table), down(p.refs)
    assert np.array_equal(table >= 0, p.ref.table >= 0) and down(p.missing)[0] == want
    held = table[table >= 0]
    assert len(np.unique(held)) == len(held) == (p.ref.table >= 0).sum() and refs.sum() == 50 - free + len(held)
    assert (refs[held] == 1).all() and refs.max() == 1


@pytest.mark.parametrize("times,free", [(700, 3), (1500, 2), (3000, 700)])
def test_many_times_the_same_sequence_before_others(hip, K, times, free):
    """More repeats than a block has threads, and than there are free pages; the others come last."""
    rng = np.random.default_rng(times)
    seqs = [1] * times + [2, 0, 3]
    p = Pools(hip, K, rng, np.full((4, 2), -1), 900, n_layers=1, n_kv=1, more=rng.permutation(900)[:900 - free])
    want = p.ref.reserve(seqs, [0] * len(seqs), 32)
    p.K.kv_pages_reserve(p.t, len(seqs), p.ints([0] * len(seqs)), 32, p.missing, seqs=p.ints(seqs), stream=hip.stream)
    table, refs = down(p.table), down(p.refs)
    assert np.array_equal(table >= 0, p.ref.table >= 0) and down(p.missing)[0] == want
    assert refs.sum() == 900 - free + (table >= 0).sum() and (refs[table[table >= 0]] == 1).all()


def test_captured_extend_follows_staged_starts(hip, K):
    """A graph of one extend, replayed a token a time while pages run out, come back and are wanted twice; eager calls and
    synchronizations between."""
    rng = np.random.default_rng(31)
    p = Pools(hip, K, rng, np.full((6, 5), -1), 13, page=16, n_layers=1, n_kv=1)
    seqs = [4, 0, 1, 2, 0, 3]
    start, listed = p.ints([0] * 6), p.ints(seqs)
    at = {b: int(x) for b, x in enumerate(rng.integers(0, 16, 6))}
    hip.stream_synchronize()
    hip.stream_begin_capture()
    K.kv_pages_extend(p.t, 6, start, 9, p.missing, seqs=listed, stream=hip.stream)
    g = hip.stream_end_capture()
    ge = hip.graph_instantiate(g)
    short = 0
    try:
        for step in range(24):
            now = [at[b] for b in seqs]
            start.upload(np.array(now, np.int32))
            hip.graph_launch(ge)
            hip.synchronize()
            want = p.ref.reserve(seqs, now, 9, follow=True)
            table, refs = down(p.table), down(p.refs)
            assert down(p.missing)[0] == want and np.array_equal(table >= 0, p.ref.table >= 0)
            assert np.array_equal(np.bincount(table[table >= 0], minlength=13), refs)
            p.ref.table, p.ref.refs = np.array(table), np.array(refs)  # (which pages they are goes by the searches)
            short += want > 0
            for b in at:
                at[b] += 3
            if step % 6 == 5:
                gone = int(rng.integers(0, 6))
                p.free([gone])
                at[gone] = int(rng.integers(0, 8))
    finally:
        hip.graph_exec_destroy(ge)
        hip.graph_destroy(g)
    assert 0 < short < 24
