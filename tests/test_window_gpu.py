"""Attention with a sliding window and sinks over the 8-bit pages, on the GPU against the 64-bit oracle."""
import math

import numpy as np
import pytest

from oracle import kv_pages as okv, long_context as olc
from tests._dev import down, empty, up
from tests.test_kv_pages_gpu import NP, Batch, append_ref, attn_tolerance, filled, matches, normal

pytestmark = pytest.mark.gpu


def check_window(hip, K, bt, pos, new, n_q, dtype, rng, window, sinks, pad=0, row_start=True, before=None, q_scale=1.0):
    """Every row's result; ``before``: rows from that position on see something that is no ordinary number."""
    hd, R = bt.hd, sum(new)
    q = normal(rng, (R + pad, n_q, hd), dtype, q_scale)
    do = up(hip, np.full(q.shape, 5, NP[dtype]))
    r = bt.rows(pos, new if row_start else None, pad)
    n = K.attn_pages_window_scratch_bytes(bt.pages, r, n_q, window, sinks)
    scratch = up(hip, np.full(n, 0xFF, np.uint8))  # scratch holds NaNs: nothing reads what it did not write
    scale = 1 / math.sqrt(hd)
    K.attn_pages_window(bt.pages, r, up(hip, q), do, n_q, scale, window, sinks, scratch, n, dtype=dtype, stream=hip.stream)
    got = down(do).astype(np.float64)
    first = np.cumsum([0] + list(new))
    for b in range(len(pos)):
        kv = bt.ref.k[b].values(bt.ref.cap), bt.ref.v[b].values(bt.ref.cap)
        present = np.array([not bt.drop(b, t) for t in range(bt.ref.cap)])
        for i in range(new[b]):
            if before is not None and pos[b] + i >= before:
                continue
            p = pos[b] + i if pos[b] >= 0 else -1
            seen = present & olc.sees(p, bt.ref.cap, window, sinks)
            v = kv[1][seen]
            vmax = np.abs(v[np.isfinite(v)]).max(initial=0)
            o, mag, big = okv.attention(q[first[b] + i], *kv, p, scale, seen)
            g = got[first[b] + i]
            assert np.array_equal(np.isnan(g), np.isnan(o)), (b, i)
            ok = matches(dtype, g, o, attn_tolerance(dtype, hd, o, mag, big, vmax))
            if not ok.all():
                pytest.fail(f"sequence {b} row {i}: {float(np.abs(g - o)[~ok].max())} off, {int((~ok).sum())} values")
    assert (got[R:] == 5).all()
    return got


def poison(hip, bt, pos, new, window, sinks):
    """Pages that no row sees any more are given back: their entries are no page, or name one of NaN."""
    bad = int(np.setdiff1d(np.arange(bt.n_pages), bt.table)[-1])  # (a spare one)
    for b, p in enumerate(pos):
        for j in range(bt.width):
            if p >= 0 and j * bt.page >= sinks and (j + 1) * bt.page <= p + 1 - window:
                bt.table[b, j] = (-1, 10 ** 7, bad)[j % 3] if bad not in bt.table else -1
    bt.upload()
    for n in ("ke", "ve"):
        e = down(bt.d[n]).copy()
        e[[p for p in range(bt.n_pages) if p not in bt.table or p == bad]] = okv.E_NAN
        bt.d[n].upload(e)


WINDOWS = [(1, 0), (1, 1), (5, 0), (64, 4), (100, 17), (130, 0), (200, 100), (64, 64), (10 ** 6, 0), (2 ** 31 - 1, 2 ** 31 - 1)]


@pytest.mark.parametrize("hd,dtype,n_q,n_kv", [(128, "f16", 12, 2), (64, "f32", 4, 4), (128, "f32", 16, 1), (64, "f16", 7, 1)])
@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_decode(hip, K, hd, dtype, n_q, n_kv, window, sinks):
    """One row per sequence, lengths from one token on, across blocks, tiles and splits; one does not run."""
    rng = np.random.default_rng(hd + n_q)
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 200, 257, 700, 0, 1025]
    bt = filled(hip, K, rng, lens, n_kv, hd, 32)
    pos = [n - 1 for n in lens]
    check_window(hip, K, bt, pos, [1] * len(lens), n_q, dtype, rng, window, sinks, row_start=False)
    poison(hip, bt, pos, [1] * len(lens), window, sinks)
    check_window(hip, K, bt, pos, [1] * len(lens), n_q, dtype, rng, window, sinks, row_start=False)


@pytest.mark.parametrize("page", [16, 128, 1024])
@pytest.mark.parametrize("dtype,n_q,n_kv,hd", [("f16", 6, 2, 128), ("f32", 7, 1, 64)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 2), (70, 5), (150, 66)])
def test_few_rows(hip, K, page, dtype, n_q, n_kv, hd, window, sinks):
    """Several rows of a sequence at a time (0 to 5), one sequence alone, rows of nobody behind them."""
    rng = np.random.default_rng(page + hd)
    lens, new = [3, 70, 300, 5, 0, 1000], [3, 2, 5, 0, 1, 4]
    bt = filled(hip, K, rng, lens, n_kv, hd, page)
    check_window(hip, K, bt, [n - m for n, m in zip(lens, new)], new, n_q, dtype, rng, window, sinks, pad=3)
    bt = filled(hip, K, rng, [333], n_kv, hd, page)
    check_window(hip, K, bt, [332], [1], n_q, dtype, rng, window, sinks)


@pytest.mark.parametrize("dtype,n_q,n_kv,hd,page", [("f16", 12, 2, 128, 64), ("f32", 12, 2, 128, 16), ("f16", 7, 1, 64, 256),
                                                    ("f32", 4, 4, 64, 32), ("f16", 32, 2, 128, 32)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (30, 0), (64, 4), (100, 100), (300, 1), (2 ** 31 - 1, 0)])
def test_prompts(hip, K, dtype, n_q, n_kv, hd, page, window, sinks):
    """Ragged prompt chunks in one call: from the first token, after cached ones, a single row, a long one; then with the
    pages that no row sees given back."""
    rng = np.random.default_rng(hd + n_q + page)
    new, old = [130, 1, 0, 33, 64, 17], [0, 500, 3, 90, 64, 610]
    bt = filled(hip, K, rng, [a + b for a, b in zip(old, new)], n_kv, hd, page)
    check_window(hip, K, bt, old, new, n_q, dtype, rng, window, sinks, pad=2)
    poison(hip, bt, old, new, window, sinks)
    check_window(hip, K, bt, old, new, n_q, dtype, rng, window, sinks, pad=2)


@pytest.mark.parametrize("dtype,n_q,n_kv,hd,window,sinks", [("f16", 16, 4, 128, 40, 4), ("f32", 24, 4, 64, 7, 0),
                                                           ("f16", 8, 4, 64, 100, 70), ("f32", 12, 4, 128, 64, 1)])
def test_many_prompts(hip, K, dtype, n_q, n_kv, hd, window, sinks):
    """140 sequences with 0 to 90 new rows each: more row blocks than two a CU, so the wider ones."""
    rng = np.random.default_rng(hd + n_q)
    new = [int(x) for x in rng.integers(0, 6, 140)]
    new[3], new[77] = 90, 33
    old = [int(x) for x in rng.integers(0, 30, 140)]
    old[50], old[77] = 400, 131
    bt = filled(hip, K, rng, [a + b for a, b in zip(old, new)], n_kv, hd, 32)
    old[9] = -1
    check_window(hip, K, bt, old, new, n_q, dtype, rng, window, sinks, pad=1)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("hd,n_q,n_kv,lens,new,window,sinks", [
    (128, 32, 32, [1100], [1050], 40, 4),                             # four-wave blocks, two a CU
    (64, 32, 32, [1100], [1050], 40, 70),                             # three a CU
    (128, 256, 16, [700, 300], [125, 9], 100, 3),                     # 256-row blocks
    (128, 128, 8, [3500] + [30] * 39, [2] * 40, 1700, 0)],            # 128-row blocks of two groups
    ids=["four", "four64", "wide", "two"])
def test_forms_of_short_windows(hip, K, dtype, hd, n_q, n_kv, lens, new, window, sinks):
    """Each form that short windows over many row blocks take (by the cost of its rounds on 256 CUs)."""
    rng = np.random.default_rng(hd + n_q)
    bt = filled(hip, K, rng, lens, n_kv, hd, 64)
    pos = [n - m for n, m in zip(lens, new)]
    poison(hip, bt, pos, new, window, sinks)
    check_window(hip, K, bt, pos, new, n_q, dtype, rng, window, sinks, pad=1)


@pytest.mark.parametrize("batch", [64, 65, 300, 700])
@pytest.mark.parametrize("ragged", [False, True])
def test_many_sequences(hip, K, batch, ragged):
    """More sequences than a wave or a block has lanes, some of which do not run, with few rows and with many."""
    rng = np.random.default_rng(batch)
    new = [int(n) for n in (rng.integers(0, 7, batch) if ragged else [1] * batch)]
    new[batch // 2] = 6 if ragged else 1
    lens = [int(rng.integers(n, 350)) if n else 0 for n in new]
    bt = filled(hip, K, rng, lens, 1, 64, 16)
    pos = [x - n if b % 9 else -1 for b, (x, n) in enumerate(zip(lens, new))]
    check_window(hip, K, bt, pos, new, 4, "f16", rng, 70, 3, row_start=ragged)


@pytest.mark.parametrize("dtype,hd,window,sinks", [("f16", 128, 3000, 8), ("f32", 64, 4200, 0), ("f16", 64, 100, 1500)])
def test_long_windows(hip, K, dtype, hd, window, sinks):
    """Windows of many shares, in decoding, for some rows, and for a chunk."""
    rng = np.random.default_rng(14)
    bt = filled(hip, K, rng, [6000, 2050], 1, hd, 64)
    for new in (1, 3, 40):
        check_window(hip, K, bt, [6000 - new, 2050 - new], [new, new], 16, dtype, rng, window, sinks)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("window,sinks", [(20, 0), (90, 33), (300, 0)])
def test_holes_and_empty_rows(hip, K, dtype, new, window, sinks):
    """Pages that are not there, inside a window and as all of it, and windows partly and wholly behind the table's end."""
    rng = np.random.default_rng(new)
    lens = [300, 90, 64, 200, 260]
    bt = filled(hip, K, rng, lens, 2, 64, 32, width=6,
                holes=[(0, 1, -1), (0, 2, 10 ** 6), (1, 0, -1), (1, 1, -5), (1, 2, -1), (2, 0, -1), (3, 5, -1), (4, 0, -1)])
    got = check_window(hip, K, bt, [n - new for n in lens], [new] * 5, 4, dtype, rng, window, sinks)
    check_window(hip, K, bt, [2 ** 31 - 1, 2 ** 31 - new, 192, 191, 250], [new] * 5, 4, dtype, rng, window, sinks)
    assert (got[new:2 * new] == 0).all()


@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("window,sinks", [(40, 20), (130, 0)])
def test_not_finite_blocks(hip, K, dtype, new, window, sinks):
    """A NaN block makes NaN of the rows that see a token of it, and of no others: before a window, in it, in the sinks'
    tile behind the sinks."""
    rng = np.random.default_rng(7)
    lens = [200, 200, 200, 200]
    bt = filled(hip, K, rng, lens, 2, 128, 64)
    bt.ref.k[0].e[2, 1] = okv.E_NAN
    bt.ref.v[1].e[10, 0] = okv.E_NAN
    bt.ref.k[2].e[13:] = bt.ref.v[2].e[13:] = okv.E_NAN  # behind the last token
    bt.ref.k[3].e[9, 0] = bt.ref.v[3].e[1, 1] = okv.E_NAN
    bt.upload()
    check_window(hip, K, bt, [n - new for n in lens], [new] * 4, 4, dtype, rng, window, sinks)


@pytest.mark.parametrize("power", [20, 100])
@pytest.mark.parametrize("new,n_q,hd", [(4, 4, 128), (70, 2, 128), (150, 4, 64), (600, 16, 128)])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_huge_tokens_outside_the_window(hip, K, dtype, new, n_q, hd, power):
    """Tokens that a row does not see leave its result alone, however large they are: those before its window, in blocks of
    their own."""
    rng = np.random.default_rng(new + power)
    n, window, sinks = 1000, 96, 16
    bt = Batch(hip, K, rng, [n], 1, hd, 64)
    k, v = rng.standard_normal((2, n, 1, hd)).astype(np.float32)
    far = (n - new - window) // 16 * 16  # (the first row's window begins at far + 1 to far + 16)
    k[16:far] *= 2.0 ** power
    v[16:far] *= 2.0 ** power
    append_ref(bt, 0, 0, k, v)
    bt.upload()
    check_window(hip, K, bt, [n - new], [new], n_q, dtype, rng, window, sinks)


def test_a_window_of_everything_is_attention_without_one(hip, K):
    """What is left out of a window that leaves nothing out is nothing: the same bits with few rows.  With many, the same
    products, and the same weights' sums taken another way (of fp32 weights, not of their two fp16 parts, which are 2^-22 of
    a weight away): 700 additions of 2^-24 and 2^-22 make 2^-14 of a sum at most, less than half a step of fp16 (2^-11), so
    a result is the same or its neighbour, a step (2^-10 of it, 2^-24 at least) away."""
    rng = np.random.default_rng(9)
    bt = filled(hip, K, rng, [700, 40, 333], 2, 128, 64)
    for new in (1, 30):
        r = bt.rows([700 - new, 40 - new, 333 - new], [new] * 3)
        q = up(hip, normal(rng, (3 * new, 4, 128), "f16"))
        n = K.attn_pages_scratch_bytes(bt.pages, r, 4)
        a, b, s = empty(hip, (3 * new, 4, 128), np.float16), empty(hip, (3 * new, 4, 128), np.float16), empty(hip, n, np.uint8)
        K.attn_pages(bt.pages, r, q, a, 4, 0.09, s, n, stream=hip.stream)
        for window, sinks in ((10 ** 6, 0), (1, 10 ** 6)):
            assert K.attn_pages_window_scratch_bytes(bt.pages, r, 4, window, sinks) == n
            K.attn_pages_window(bt.pages, r, q, b, 4, 0.09, window, sinks, s, n, stream=hip.stream)
            x, y = down(a).astype(np.float64), down(b).astype(np.float64)
            assert np.array_equal(x, y) if new == 1 else (np.abs(x - y) <= 2.0 ** -10 * np.abs(x) + 2.0 ** -24).all()


@pytest.mark.parametrize("new", [1, 40])
def test_captured_windows_follow_staged_lengths(hip, K, new):
    """Lengths and pages are read on the device: one captured launch serves other lengths, replayed with eager work in
    between."""
    rng = np.random.default_rng(new)
    bt = filled(hip, K, rng, [300, 170, 64], 2, 128, 32)
    q = normal(rng, (3 * new, 4, 128), "f16")
    dq, do = up(hip, q), empty(hip, q.shape, np.float16)
    r = bt.rows([0, 0, 0], [new] * 3)
    off = bt.d["off"]
    n = K.attn_pages_window_scratch_bytes(bt.pages, r, 4, 50, 7)
    scratch = empty(hip, n, np.uint8)
    hip.stream_synchronize()
    hip.stream_begin_capture()
    K.attn_pages_window(bt.pages, r, dq, do, 4, 0.09, 50, 7, scratch, n, stream=hip.stream)
    g = hip.stream_end_capture()
    ge = hip.graph_instantiate(g)
    try:
        for pos in ([300 - new, 170 - new, 64 - new], [0, 0, 0], [17, -1, 5], [300 - new, 3, 0]):
            off.upload(np.array(pos, np.int32))
            hip.graph_launch(ge)
            got = down(do).copy()
            K.attn_pages_window(bt.pages, r, dq, do, 4, 0.09, 50, 7, scratch, n, stream=hip.stream)
            assert np.array_equal(down(do), got)
            for b in range(3):
                kv = bt.ref.k[b].values(bt.ref.cap), bt.ref.v[b].values(bt.ref.cap)
                present = np.array([not bt.drop(b, t) for t in range(bt.ref.cap)])
                for i in range(new):
                    p = pos[b] + i if pos[b] >= 0 else -1
                    o, mag, big = okv.attention(q[b * new + i], *kv, p, 0.09, present & olc.sees(p, bt.ref.cap, 50, 7))
                    tol = attn_tolerance("f16", 128, o, mag, big, 8.0)
                    assert matches("f16", got[b * new + i].astype(np.float64), o, tol).all(), (pos, b, i)
    finally:
        hip.graph_exec_destroy(ge)
        hip.graph_destroy(g)


def test_two_streams_at_once(hip, K):
    """Windows over a prompt chunk, windows of decoded tokens, heads and a pool's calls on three streams that are not the
    runtime's, each with memory of its own, together: the results of each alone."""
    import ctypes
    from tests.test_head_form_gpu import Form
    from tests.test_kv_manage_gpu import Pools
    rng = np.random.default_rng(41)
    streams = []
    for _ in range(3):
        s = ctypes.c_void_p()
        hip._check_error(hip._lib.hipStreamCreate(ctypes.byref(s)), "hipStreamCreate")
        streams.append(s)
    jobs, outs = [], []
    for new, s in zip((1, 150), streams):
        bt = filled(hip, K, rng, [900, 333], 2, 128, 64)
        q, r = up(hip, normal(rng, (2 * new, 8, 128), "f16")), bt.rows([900 - new, 333 - new], [new, new])
        n = K.attn_pages_window_scratch_bytes(bt.pages, r, 8, 200, 4)
        o, sc = empty(hip, (2 * new, 8, 128), np.float16), empty(hip, n, np.uint8)
        jobs.append(lambda bt=bt, r=r, q=q, o=o, sc=sc, n=n, s=s: K.attn_pages_window(bt.pages, r, q, o, 8, 0.1, 200, 4, sc, n, stream=s))
        outs.append(o)
    f, x, y = Form(hip, rng, 128, 128), up(hip, normal(rng, (200, 8, 128), "f16")), empty(hip, (200, 8, 128), np.float16)
    pos = up(hip, np.arange(200, dtype=np.int32))
    jobs.append(lambda: K.qk_norm_rope(f.c, 200, pos, q=x, q_out=y, n_q=8, stream=streams[2]))
    p = Pools(hip, K, rng, np.full((8, 6), -1), 60)
    start = p.ints([10] * 8)

    def pool():
        K.kv_pages_free(p.t, 8, stream=streams[2])
        K.kv_pages_reserve(p.t, 8, start, 60, None, stream=streams[2])
    jobs.append(pool)
    outs += [y, p.table, p.refs]
    try:
        for job in jobs:
            job()
            hip.synchronize()
        alone = [down(o).copy() for o in outs]
        for _ in range(10):
            for job in jobs:
                job()
        hip.synchronize()
        for o, a in zip(outs, alone):
            assert np.array_equal(down(o), a)
    finally:
        for s in streams:
            hip._lib.hipStreamDestroy(s)
