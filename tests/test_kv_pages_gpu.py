"""The 8-bit paged KV cache on the GPU against the 64-bit oracle: bytes and exponents exactly, attention within
bounds counted from the formats."""
import math

import numpy as np
import pytest

from oracle import kv_pages as okv
from tests._dev import down, empty, up
from vte_amd.core.rope_cache import build_rope_cache
from vte_amd.kernels import KVPages, KVRows

pytestmark = pytest.mark.gpu

NP = {"f16": np.float16, "f32": np.float32}


class Batch:
    """Sequences with pages in random order, the oracle's cache beside the device's."""

    def __init__(self, hip, K, rng, lens, n_kv, hd, page, spare=2, width=None, holes=()):
        self.hip, self.K, self.rng, self.n_kv, self.hd, self.page = hip, K, rng, n_kv, hd, page
        per = [max(1, -(-n // page)) for n in lens]
        self.width = width or max(per)
        self.n_pages = sum(per) + spare
        order, at = rng.permutation(self.n_pages), 0
        self.table = np.full((len(lens), self.width), -1, np.int32)
        for b, p in enumerate(per):
            m = min(p, self.width)
            self.table[b, :m] = order[at:at + m]
            at += p
        for b, j, entry in holes:
            self.table[b, j] = entry
        self.ref = okv.Cache(len(lens), n_kv, hd, self.width, page)
        self.d = {}
        self.upload()

    def upload(self):
        for is_v, n in ((False, "k"), (True, "v")):
            codes, exps = self.ref.pool(self.table, self.n_pages, is_v)
            self.d[n], self.d[n + "e"] = up(self.hip, codes), up(self.hip, exps)
        self.d["table"] = up(self.hip, self.table)
        self.pages = KVPages.of(self.d["k"], self.d["v"], self.d["ke"], self.d["ve"], self.n_pages, self.page,
                                self.n_kv, self.hd)

    def rows(self, pos, new=None, pad=0, max_rows=None):
        """New rows of each sequence from positions pos (new None: one each without row_start)."""
        self.d["off"] = up(self.hip, np.asarray(pos, np.int32))
        B = len(pos)
        if new is None:
            return KVRows.of(B, B, 1, None, self.d["off"], self.d["table"], self.width)
        start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.d["start"] = up(self.hip, start)
        return KVRows.of(B, int(start[-1]) + pad, max(new) if max_rows is None else max_rows, self.d["start"],
                         self.d["off"], self.d["table"], self.width)

    def drop(self, b, pos):
        """Whether a row at pos has no place."""
        return pos >= self.ref.cap or not 0 <= self.table[b, pos // self.page] < self.n_pages

    def check(self, rows):
        """The device's pages are the oracle's, byte for byte, where a sequence has live tokens."""
        for is_v, n in ((False, "k"), (True, "v")):
            codes, exps = down(self.d[n]), down(self.d[n + "e"])
            for b, parts in enumerate(self.ref.v if is_v else self.ref.k):
                c, e = okv.unpool(codes, exps, self.table[b], self.page, is_v)
                live = np.array([not self.drop(b, t) for t in range(rows[b])], bool)
                assert np.array_equal(c[:rows[b]][live], parts.c[:rows[b]][live]), (n, b)
                el = live[::okv.BLOCK]
                assert np.array_equal(e[:len(el)][el], parts.e[:len(el)][el]), (n, b)


def append_ref(batch, b, pos, k, v):
    """The oracle's append of rows whose places exist (a hole swallows whole blocks)."""
    n = min(len(k), batch.ref.cap - pos)
    t = 0
    while t < n:
        m = min(n - t, okv.BLOCK - (pos + t) % okv.BLOCK)
        if not batch.drop(b, pos + t):
            batch.ref.k[b].append(k[t:t + m], pos + t)
            batch.ref.v[b].append(v[t:t + m], pos + t)
        t += m


def normal(rng, shape, dtype, scale=1.0):
    return (scale * rng.standard_normal(shape)).astype(NP[dtype])


@pytest.mark.parametrize("hd,dtype,rope", [(128, "f16", 0), (128, "f16", 1), (128, "f32", 0), (64, "f16", 0),
                                           (64, "f32", 2), (128, "f16", 2), (128, "f16", None), (64, "f16", 1)])
def test_append_token_by_token(hip, K, hd, dtype, rope):
    """Three sequences from different places, magnitudes that climb by 2^12: the blocks' scales grow under tokens
    that are already in, and shrink again with a new block."""
    rng = np.random.default_rng(hd + 10 * (rope or 7))
    n_kv, n_q, start = 2, 6, [0, 15, 37]
    bt = Batch(hip, K, rng, [50, 66, 88], n_kv, hd, 32)
    for b, n in enumerate(start):
        for p in (bt.ref.k[b], bt.ref.v[b]):
            p.append(normal(rng, (n, n_kv, hd), "f16"), 0)
    bt.upload()
    rd = {None: 0, 2: hd // 2 + 4}.get(rope, hd)
    cos, sin = build_rope_cache(128, rd or hd, 1e4)
    dc, ds = up(hip, cos), up(hip, sin)
    for step in range(50):
        pos = [s + step for s in start]
        size = 2.0 ** rng.uniform(-6, 6)
        q, k, v = (normal(rng, (3, h, hd), dtype, size) for h in (n_q, n_kv, n_kv))
        dq, dk, dv, do = up(hip, q), up(hip, k), up(hip, v), empty(hip, q.shape, NP[dtype])
        r = bt.rows(pos)
        if rope is None:
            K.kv_pages_append(bt.pages, r, dk, dv, dtype=dtype, stream=hip.stream)
            kr = k.astype(np.float32)
        else:
            K.kv_pages_append(bt.pages, r, dk, dv, q=dq, q_out=do, n_q=n_q, rope_cos=dc, rope_sin=ds, rope_rows=128,
                              rope_type=rope, rotary_dim=rd, dtype=dtype, stream=hip.stream)
            kr = okv.rotate(k, pos, cos, sin, rope, rd)
            assert np.array_equal(down(do), okv.rotate(q, pos, cos, sin, rope, rd).astype(NP[dtype]))
        for b in range(3):
            append_ref(bt, b, pos[b], kr[b:b + 1], v[b:b + 1])
        if step % 7 == 0 or step == 49:
            bt.check([p + 1 for p in pos])


@pytest.mark.parametrize("page,hd,dtype", [(16, 128, "f16"), (64, 128, "f16"), (32, 64, "f32"), (256, 64, "f16")])
def test_append_ragged_prompts(hip, K, page, hd, dtype):
    """Chunks of 0 to 200 rows in one call, from places inside blocks, with a sequence that does not run, a table entry
    that is no page, rows past the table, rows of nobody, strided k, v and q; other memory stays as it was."""
    rng = np.random.default_rng(page + hd)
    n_kv, n_q = 3, 6
    pos, new = [0, 5, 31, -1, 16, 40, 3], [200, 0, 90, 4, 17, 60, 1]
    lens = [p + n if p >= 0 else 0 for p, n in zip(pos, new)]
    width = max(1, 208 // page)
    holes = [(2, 64 // page, -1), (4, 0, 10 ** 6)] if page <= 64 else [(4, 0, -7)]
    bt = Batch(hip, K, rng, lens, n_kv, hd, page, width=width, holes=holes)
    for b, p in enumerate(pos):
        if p > 0:
            old = [normal(rng, (p, n_kv, hd), "f16", 0.3) for _ in "kv"]
            append_ref(bt, b, 0, *old)
    bt.upload()
    before = {n: down(bt.d[n]).copy() for n in ("k", "v", "ke", "ve")}
    R, pad = sum(new), 5
    wide = normal(rng, (R + pad, n_q + 2 * n_kv, hd), dtype)  # q, k and v of one fused projection
    dw = up(hip, wide)
    size, ld = wide.itemsize, wide.shape[1] * hd
    out = np.full((R + pad, n_q, hd), 9, NP[dtype])
    do = up(hip, out)
    limit = 205 if page <= 64 else 230  # the rotation's table ends inside sequence 0's last page or past the capacity
    cos, sin = build_rope_cache(limit, hd, 1e4)
    r = bt.rows(pos, new, pad)
    K.kv_pages_append(bt.pages, r, dw.ptr + n_q * hd * size, dw.ptr + (n_q + n_kv) * hd * size, q=dw, q_out=do,
                      n_q=n_q, rope_cos=up(hip, cos), rope_sin=up(hip, sin), rope_rows=limit, dtype=dtype,
                      k_stride=ld, v_stride=ld, q_stride=ld, stream=hip.stream)
    got, first = down(do), np.cumsum([0] + new)
    written = set()
    for b in range(len(pos)):
        if pos[b] < 0:
            continue
        n = max(0, min(new[b], min(limit, bt.ref.cap) - pos[b]))
        w = wide[first[b]:first[b] + n]
        at = pos[b] + np.arange(n)
        append_ref(bt, b, pos[b], okv.rotate(w[:, n_q:n_q + n_kv], at, cos, sin), w[:, n_q + n_kv:].astype(np.float32))
        out[first[b]:first[b] + n] = okv.rotate(w[:, :n_q], at, cos, sin).astype(NP[dtype])
        written |= {(int(bt.table[b, t // page]), t % page // 16) for t in at if not bt.drop(b, t)}
    assert np.array_equal(got, out)
    bt.check([min(max(n, 0), bt.ref.cap, max(p, limit)) for n, p in zip(lens, pos)])
    for n, old in before.items():  # blocks that no new row fell into
        now = down(bt.d[n])
        for p in range(bt.n_pages):
            for i in range(page // 16):
                if (p, i) not in written:
                    sl = (p, slice(None), slice(16 * i, 16 * i + 16)) if n == "k" else (p, slice(None), i)
                    assert np.array_equal(now[sl], old[sl]), (n, p, i)


@pytest.mark.parametrize("batch", [70, 300])
def test_append_to_many_sequences(hip, K, batch):
    """A few rows of each of many sequences, some of none, with rows of nobody before the first one's."""
    rng = np.random.default_rng(batch)
    new = [int(n) for n in rng.integers(0, 4, batch)]
    pos = [int(p) if b % 7 else -1 for b, p in enumerate(rng.integers(0, 40, batch))]
    lens = [max(p, 0) + n for p, n in zip(pos, new)]
    bt = Batch(hip, K, rng, lens, 1, 64, 16, width=3)
    for b, p in enumerate(pos):
        if p > 0:
            append_ref(bt, b, 0, *[normal(rng, (p, 1, 64), "f16", 0.3) for _ in "kv"])
    bt.upload()
    r = bt.rows(pos, new, pad=2)
    start = (2 + np.concatenate([[0], np.cumsum(new)])).astype(np.int32)
    bt.d["start"] = up(hip, start)
    r.row_start = bt.d["start"].ptr
    R = int(start[-1])
    q, k, v = normal(rng, (R, 2, 64), "f16"), normal(rng, (R, 1, 64), "f16"), normal(rng, (R, 1, 64), "f16")
    cos, sin = build_rope_cache(64, 64, 1e4)
    out = np.full(q.shape, 9, np.float16)
    do = up(hip, out)
    K.kv_pages_append(bt.pages, r, up(hip, k), up(hip, v), q=up(hip, q), q_out=do, n_q=2, rope_cos=up(hip, cos),
                      rope_sin=up(hip, sin), rope_rows=64, stream=hip.stream)
    for b, n in enumerate(new):
        if pos[b] >= 0 and n:
            at, rows = pos[b] + np.arange(n), slice(start[b], start[b + 1])
            append_ref(bt, b, pos[b], okv.rotate(k[rows], at, cos, sin), v[rows].astype(np.float32))
            out[rows] = okv.rotate(q[rows], at, cos, sin).astype(np.float16)
    assert np.array_equal(down(do), out)
    bt.check([n if p >= 0 else 0 for n, p in zip(lens, pos)])


def test_append_not_finite(hip, K):
    """A block that receives an Inf or a NaN reads as NaN, and later ones of other heads and blocks do not."""
    rng = np.random.default_rng(5)
    bt = Batch(hip, K, rng, [40], 2, 64, 32)
    k, v = (normal(rng, (40, 2, 64), "f16") for _ in "kv")
    k[3, 0, 5], v[20, 1, 63], v[21, 0, 0] = np.inf, np.nan, -np.inf
    for lo, hi in ((0, 25), (25, 40)):
        K.kv_pages_append(bt.pages, bt.rows([lo], [hi - lo]), up(hip, k[lo:hi]), up(hip, v[lo:hi]), stream=hip.stream)
        append_ref(bt, 0, lo, k[lo:hi], v[lo:hi])
    bt.check([40])
    ko, vo = empty(hip, (1, 40, 2, 64), np.float32), empty(hip, (1, 40, 2, 64), np.float32)
    K.kv_pages_read(bt.pages, bt.rows([40], [0]), ko, vo, 40, dtype="f32", stream=hip.stream)
    for got, part, bad in ((ko, bt.ref.k[0], [(0, 0)]), (vo, bt.ref.v[0], [(1, 1), (1, 0)])):
        g = down(got)[0]
        assert np.array_equal(g, part.values(40).astype(np.float32), equal_nan=True)
        assert {(int(t) // 16, int(h)) for t, h, _ in zip(*np.nonzero(np.isnan(g)))} == set(bad)


@pytest.mark.parametrize("dtype,size", [("f16", 6e4), ("f16", 1e-7), ("f32", 1e38), ("f32", 1e-44), ("f32", 0.0)])
def test_append_and_read_extreme_magnitudes(hip, K, dtype, size):
    rng = np.random.default_rng(6)
    bt = Batch(hip, K, rng, [33], 1, 128, 16)
    k, v = ((size * rng.uniform(-1, 1, (33, 1, 128))).astype(NP[dtype]) for _ in "kv")
    K.kv_pages_append(bt.pages, bt.rows([0], [33]), up(hip, k), up(hip, v), dtype=dtype, stream=hip.stream)
    append_ref(bt, 0, 0, k, v)
    bt.check([33])
    ko, vo = empty(hip, (1, 33, 1, 128), NP[dtype]), empty(hip, (1, 33, 1, 128), NP[dtype])
    K.kv_pages_read(bt.pages, bt.rows([33], [0]), ko, vo, 33, dtype=dtype, stream=hip.stream)
    assert np.array_equal(down(ko)[0], bt.ref.k[0].values(33).astype(NP[dtype]))
    assert np.array_equal(down(vo)[0], bt.ref.v[0].values(33).astype(NP[dtype]))


@pytest.mark.parametrize("hd,dtype,page,out_rows", [(128, "f16", 16, 100), (64, "f32", 64, 37), (128, "f32", 128, 300),
                                                    (64, "f16", 32, 1)])
def test_read(hip, K, hd, dtype, page, out_rows):
    """Every sequence's rows, 0 where it has no page, the rest of the output as it was."""
    rng = np.random.default_rng(hd + page)
    lens, pos = [100, 1, 0, 64, 33], [100, 1, 0, 64, 30]
    bt = Batch(hip, K, rng, lens, 2, hd, page, holes=[(3, 1, -1)] if page <= 32 else [])
    for b, n in enumerate(lens):
        append_ref(bt, b, 0, *(normal(rng, (n, 2, hd), "f16") for _ in "kv"))
    bt.upload()
    new = [0, 0, 0, 0, 3]
    want = [np.full((5, out_rows, 2, hd), 7, NP[dtype]) for _ in "kv"]
    ko, vo = up(hip, want[0]), up(hip, want[1])
    pos[2] = -1
    K.kv_pages_read(bt.pages, bt.rows(pos, new), ko, vo, out_rows, dtype=dtype, stream=hip.stream)
    for w, parts in zip(want, (bt.ref.k, bt.ref.v)):
        for b in range(5):
            n = min(lens[b], out_rows) if pos[b] >= 0 else 0
            x = parts[b].values(n)
            for t in range(n):
                w[b, t] = 0 if bt.drop(b, t) else x[t]
    assert np.array_equal(down(ko), want[0]) and np.array_equal(down(vo), want[1])


# ---------------------------------------------------------------------------- attention
def attn_tolerance(dtype, hd, out, mag, big, vmax):
    """|error| of one result.  fp16: the probabilities are rounded (2^-11 of each, so of the weighted |V|) and the
    result is (2^-11); fp32: two fp16 parts of q and of the probabilities (2^-21 each: a rounded part and a rounded
    rest of at most 2^-11 of it), the result 2^-24.  Both: scores are fp32 sums of hd + 3 roundings at most (2^-24 of
    the sum of |q k| each), which e^x carries into both sums (twice); exponentials, sums and the rescaling by running
    maxima add 2^-19 at most (2^-24 a rounding, below 32 of them in a chain); half the smallest fp16 is 2^-25, of
    probabilities scaled by 2^14 2^-39 of the largest for each of at most 2^16 tokens, of a prompt's scaled by 2^9 2^-34
    for each of at most 2^13 (2^-21 together).  fp16 results below 2^-14 are
    rounded to steps of 2^-24 (2^-25 at most)."""
    p, r = (2.0 ** -11, 2.0 ** -11) if dtype == "f16" else (2.0 ** -20, 2.0 ** -24)
    q = 0.0 if dtype == "f16" else 2.0 ** -21
    score = big[:, None] * (q + (hd + 3) * 2.0 ** -24)
    return (p + 2 * score + 2.0 ** -19) * mag + r * np.abs(out) + 2.0 ** -21 * vmax + (2.0 ** -25 if dtype == "f16" else 0)


def matches(dtype, got, out, tol):
    """Within the tolerance; an fp16 result from 65520 on (half a step past the largest, 65504) is Inf."""
    with np.errstate(invalid="ignore"):
        ok = np.isnan(out) | (np.abs(got - out) <= tol)
        return ok | (np.isinf(got) & (np.abs(out) + tol >= 65520) & (got * out > 0)) if dtype == "f16" else ok


def check_attention(hip, K, bt, pos, new, n_q, dtype, rng, pad=0, q_scale=1.0, row_start=True, zero_dims=0, before=None):
    B, hd = len(pos), bt.hd
    R = sum(new)
    q = normal(rng, (R + pad, n_q, hd), dtype, q_scale)
    q[:, :, :zero_dims] = 0
    out = np.full(q.shape, 5, NP[dtype])
    do = up(hip, out)
    r = bt.rows(pos, new if row_start else None, pad)
    n = K.attn_pages_scratch_bytes(bt.pages, r, n_q)
    scratch = up(hip, np.full(n, 0xFF, np.uint8))  # scratch holds NaNs: nothing reads what it did not write
    scale = 1 / math.sqrt(hd)
    K.attn_pages(bt.pages, r, up(hip, q), do, n_q, scale, scratch, n, dtype=dtype, stream=hip.stream)
    got = down(do).astype(np.float64)
    first = np.cumsum([0] + list(new))
    for b in range(B):
        kv = bt.ref.k[b].values(bt.ref.cap), bt.ref.v[b].values(bt.ref.cap)
        present = np.array([not bt.drop(b, t) for t in range(bt.ref.cap)])
        for i in range(new[b]):
            if before is not None and pos[b] + i >= before:
                continue
            seen = kv[1][:max(pos[b] + i + 1, 0)]
            vmax = np.abs(seen[np.isfinite(seen)]).max(initial=0)
            o, mag, big = okv.attention(q[first[b] + i], *kv, pos[b] + i if pos[b] >= 0 else -1, scale, present)
            g = got[first[b] + i]
            assert np.array_equal(np.isnan(g), np.isnan(o)), (b, i)
            tol = attn_tolerance(dtype, hd, o, mag, big, vmax)
            ok = matches(dtype, g, o, tol)
            if not ok.all():
                pytest.fail(f"sequence {b} row {i}: {float(np.abs(g - o)[~ok].max())} off, {int((~ok).sum())} values")
    assert (got[R:] == 5).all()
    return got


def filled(hip, K, rng, lens, n_kv, hd, page, v_sizes=None, **kw):
    bt = Batch(hip, K, rng, lens, n_kv, hd, page, **kw)
    for b, n in enumerate(lens):
        n = min(n, bt.ref.cap)
        v = rng.standard_normal((n, n_kv, hd))
        if v_sizes is not None:
            v *= 2.0 ** rng.uniform(*v_sizes, (n, n_kv, 1))
        append_ref(bt, b, 0, rng.standard_normal((n, n_kv, hd)).astype(np.float16), v.astype(np.float32))
    bt.upload()
    return bt


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("n_q,n_kv", [(12, 2), (1, 1), (16, 1), (4, 4), (14, 2)])
def test_attention_decode(hip, K, hd, dtype, n_q, n_kv):
    """One row per sequence, lengths from one token on, across blocks, tiles and splits; one does not run."""
    rng = np.random.default_rng(hd + n_q)
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 200, 257, 700, 0, 1025]
    bt = filled(hip, K, rng, lens, n_kv, hd, 32)
    check_attention(hip, K, bt, [n - 1 for n in lens], [1] * len(lens), n_q, dtype, rng, row_start=False)


@pytest.mark.parametrize("page", [16, 64, 128, 1024])
@pytest.mark.parametrize("dtype,n_q,n_kv,hd", [("f16", 6, 2, 128), ("f32", 7, 1, 64)])
def test_attention_few_rows(hip, K, page, dtype, n_q, n_kv, hd):
    """Several rows of a sequence at a time (0 to 5), one sequence alone, rows of nobody behind them."""
    rng = np.random.default_rng(page + hd)
    lens, new = [3, 70, 300, 5, 0, 1000], [3, 2, 5, 0, 1, 4]
    bt = filled(hip, K, rng, lens, n_kv, hd, page)
    check_attention(hip, K, bt, [n - m for n, m in zip(lens, new)], new, n_q, dtype, rng, pad=3)
    bt = filled(hip, K, rng, [333], n_kv, hd, page)
    check_attention(hip, K, bt, [332], [1], n_q, dtype, rng)


@pytest.mark.parametrize("dtype,n_q,n_kv,hd,page", [("f16", 12, 2, 128, 64), ("f32", 12, 2, 128, 16),
                                                    ("f16", 7, 1, 64, 256), ("f32", 4, 4, 64, 32),
                                                    ("f16", 32, 2, 128, 32)])
def test_attention_prompts(hip, K, dtype, n_q, n_kv, hd, page):
    """Ragged prompt chunks in one call: from the first token, after cached ones, a single row, a long one."""
    rng = np.random.default_rng(hd + n_q + page)
    new = [130, 1, 0, 33, 64, 17]
    old = [0, 500, 3, 90, 64, 1]
    bt = filled(hip, K, rng, [a + b for a, b in zip(old, new)], n_kv, hd, page)
    check_attention(hip, K, bt, old, new, n_q, dtype, rng, pad=2)


@pytest.mark.parametrize("batch", [64, 65, 300, 700])
@pytest.mark.parametrize("ragged", [False, True])
def test_attention_of_many_sequences(hip, K, batch, ragged):
    """More sequences than a wave or a block has lanes, some of which do not run, with few rows and with many."""
    rng = np.random.default_rng(batch)
    new = [int(n) for n in (rng.integers(0, 7, batch) if ragged else [1] * batch)]
    new[batch // 2] = 6 if ragged else 1
    lens = [int(rng.integers(n, 150)) if n else 0 for n in new]
    bt = filled(hip, K, rng, lens, 1, 64, 16)
    pos = [x - n if b % 9 else -1 for b, (x, n) in enumerate(zip(lens, new))]
    check_attention(hip, K, bt, pos, new, 4, "f16", rng, row_start=ragged)


@pytest.mark.parametrize("dtype,hd", [("f16", 128), ("f32", 64)])
def test_attention_of_some_rows_over_a_long_cache(hip, K, dtype, hd):
    """More rows than one tile has columns, tokens for more shares than are joined at once."""
    rng = np.random.default_rng(14)
    bt = filled(hip, K, rng, [5000, 2050], 1, hd, 64)
    check_attention(hip, K, bt, [4997, 2047], [3, 3], 16, dtype, rng)


@pytest.mark.parametrize("dtype,n_q,n_kv,hd", [("f16", 16, 4, 128), ("f32", 24, 4, 64), ("f16", 8, 4, 64),
                                               ("f32", 12, 4, 128)])
def test_attention_many_prompts(hip, K, dtype, n_q, n_kv, hd):
    """140 sequences with 0 to 90 new rows each: more row blocks than two a CU, so the wider ones."""
    rng = np.random.default_rng(hd + n_q)
    new = [int(x) for x in rng.integers(0, 6, 140)]
    new[3], new[77] = 90, 33
    old = [int(x) for x in rng.integers(0, 30, 140)]
    old[50], old[77] = 400, 131
    bt = filled(hip, K, rng, [a + b for a, b in zip(old, new)], n_kv, hd, 32)
    old[9] = -1
    check_attention(hip, K, bt, old, new, n_q, dtype, rng, pad=1)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_holes_and_empty_rows(hip, K, dtype, new):
    """Pages that are not there, all of a sequence's among them, and rows past the table's end."""
    rng = np.random.default_rng(new)
    lens = [300, 90, 64, 200]
    bt = filled(hip, K, rng, lens, 2, 64, 32, width=6,
                holes=[(0, 1, -1), (0, 2, 10 ** 6), (1, 0, -1), (1, 1, -5), (1, 2, -1), (2, 0, -1)])
    check_attention(hip, K, bt, [n - new for n in lens], [new] * 4, 4, dtype, rng)


@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_not_finite_blocks(hip, K, dtype, new):
    """A NaN block makes NaN of the rows that see a token of it, and of no others; dead places hold anything."""
    rng = np.random.default_rng(7)
    lens = [200, 200, 200]
    bt = filled(hip, K, rng, lens, 2, 128, 64)
    bt.ref.k[0].e[2, 1] = okv.E_NAN
    bt.ref.v[1].e[11, 0] = okv.E_NAN
    bt.ref.k[2].e[13:] = okv.E_NAN  # behind the last token of sequence 2
    bt.ref.v[2].e[13:] = okv.E_NAN
    bt.upload()
    got = check_attention(hip, K, bt, [n - new for n in lens], [new] * 3, 4, dtype, rng)
    assert np.isnan(got).any() and not np.isnan(got[2 * new:]).any()


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("v_sizes,q_scale", [((-20, 20), 1.0), ((0, 0), 30.0), ((-3, 3), 1e-3)])
def test_attention_scales_and_peaks(hip, K, dtype, new, v_sizes, q_scale):
    """V blocks of very different scales, sharply peaked scores, and small queries."""
    rng = np.random.default_rng(8)
    bt = filled(hip, K, rng, [900, 71], 1, 128, 64, v_sizes=v_sizes)
    check_attention(hip, K, bt, [900 - new, 71 - new], [new, new], 6, dtype, rng, q_scale=q_scale)


@pytest.mark.parametrize("power", [20, 40, 100])
@pytest.mark.parametrize("new,n_q,hd", [(4, 4, 128), (70, 2, 128), (150, 4, 64), (600, 16, 128)])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_of_rows_before_huge_tokens(hip, K, dtype, new, n_q, hd, power):
    """Tokens that a row does not see leave its result alone, however large they are (those of blocks of their own: a
    block has one scale)."""
    rng = np.random.default_rng(new + power)
    n, at = 800, 800 - new // 2 - (800 - new // 2) % 16
    bt = Batch(hip, K, rng, [n], 1, hd, 64)
    k, v = rng.standard_normal((2, n, 1, hd)).astype(np.float32)
    k[at:] *= 2.0 ** power
    v[at:] *= 2.0 ** power
    append_ref(bt, 0, 0, k, v)
    bt.upload()
    check_attention(hip, K, bt, [n - new], [new], n_q, dtype, rng, before=at)


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_beside_huge_keys_in_other_dims(hip, K, dtype, new):
    """Keys of one block are 2^60 times the others', in dims that no query has: scores of both are ordinary."""
    rng = np.random.default_rng(12)
    bt = Batch(hip, K, rng, [300], 2, 128, 64)
    k, v = rng.standard_normal((2, 300, 2, 128)).astype(np.float32)
    k[112:128, :, :4] *= 2.0 ** 60
    append_ref(bt, 0, 0, k, v)
    bt.upload()
    check_attention(hip, K, bt, [300 - new], [new], 6, dtype, rng, zero_dims=4)


@pytest.mark.parametrize("new", [1, 70])
def test_attention_of_scores_far_below_zero(hip, K, new):
    """Equal keys, so equal weights, at scores of -6e32: the mean of V."""
    rng = np.random.default_rng(15)
    bt = Batch(hip, K, rng, [200], 1, 64, 64)
    v = rng.standard_normal((200, 1, 64)).astype(np.float32)
    append_ref(bt, 0, 0, np.full((200, 1, 64), 1e14, np.float32), v)
    bt.upload()
    r = bt.rows([200 - new], [new])
    q, out = up(hip, np.full((new, 4, 64), -1e18, np.float32)), empty(hip, (new, 4, 64), np.float32)
    need = K.attn_pages_scratch_bytes(bt.pages, r, 4)
    K.attn_pages(bt.pages, r, q, out, 4, 0.1, empty(hip, need, np.uint8), need, dtype="f32", stream=hip.stream)
    got, v = down(out), bt.ref.v[0].values(200)[:, 0]
    for i in range(new):
        # weights of 1 and sums of up to 200 of them: 200 roundings of 2^-24 of the largest |V| at most
        assert np.abs(got[i] - v[:201 - new + i].mean(0)).max() <= 200 * 2.0 ** -24 * np.abs(v).max()


@pytest.mark.parametrize("new", [2, 70])
def test_attention_of_positions_at_the_end_of_int(hip, K, new):
    """Positions behind the table see all of it, up to the largest int; what they append has no place."""
    rng = np.random.default_rng(13)
    bt = filled(hip, K, rng, [128, 128], 2, 64, 64)
    check_attention(hip, K, bt, [2 ** 31 - 1, 2 ** 31 - new], [new, new], 4, "f32", rng)
    r = bt.rows([2 ** 31 - 1, 2 ** 31 - new], [new, new])
    x = up(hip, normal(rng, (2 * new, 2, 64), "f16"))
    K.kv_pages_append(bt.pages, r, x, x, stream=hip.stream)
    bt.check([128, 128])
    ko, vo = empty(hip, (2, 128, 2, 64), np.float32), empty(hip, (2, 128, 2, 64), np.float32)
    K.kv_pages_read(bt.pages, r, ko, vo, 128, dtype="f32", stream=hip.stream)
    for b in range(2):
        assert np.array_equal(down(ko)[b], bt.ref.k[b].values(128)) and np.array_equal(down(vo)[b], bt.ref.v[b].values(128))


@pytest.mark.parametrize("new", [1, 30])
def test_attention_does_not_depend_on_the_batch(hip, K, new):
    """Equal bits for a sequence alone, in a batch and in other pages."""
    rng = np.random.default_rng(9)
    lens = [700, 40, 333]
    bt = filled(hip, K, rng, lens, 2, 128, 64)
    alone = Batch(hip, K, rng, [700], 2, 128, 64, spare=9)
    alone.ref.k[0], alone.ref.v[0] = bt.ref.k[0], bt.ref.v[0]
    alone.upload()
    q = normal(rng, (3 * new, 4, 128), "f16")
    res = []
    for b, pos, n in ((bt, [x - new for x in lens], [new] * 3), (alone, [700 - new], [new])):
        r = b.rows(pos, n)
        need = K.attn_pages_scratch_bytes(b.pages, r, 4)
        do = empty(hip, (sum(n), 4, 128), np.float16)
        K.attn_pages(b.pages, r, up(hip, q[:sum(n)]), do, 4, 0.09, empty(hip, need, np.uint8), need, stream=hip.stream)
        res.append(down(do)[:new].astype(np.float64))
    assert np.abs(res[0] - res[1]).max() <= 2.0 ** -9 * np.abs(res[1]).max()


# ---------------------------------------------------------------------------- together, captured, on other streams
def test_captured_decode_loop(hip, K):
    """Embedding (q, k and v rows of a token), append, attention, LM head, draw and feedback as one captured graph,
    replayed 30 times over ragged sequences that cross blocks and pages: every replay's cache is the oracle's, its
    logits within the attention's bounds of the oracle's, its tokens the draws from these logits."""
    from oracle import sampling as osm
    from oracle.dequant import dequantize_matrix
    from vte_amd import synthetic as syn
    rng = np.random.default_rng(31)
    n_q, n_kv, hd, V, start = 6, 2, 64, 1000, [0, 13, 30, 47]
    B, width, qd = 4, (n_q + 2 * n_kv) * hd, n_q * hd
    bt = Batch(hip, K, rng, [s + 31 for s in start], n_kv, hd, 16)
    for b, n in enumerate(start):
        append_ref(bt, b, 0, *(normal(rng, (n, n_kv, hd), "f16") for _ in "kv"))
    bt.upload()
    table, head = syn.random_matrix("q8_0", rng, V, width), syn.random_matrix("q8_0", rng, V, qd)
    rows_f = dequantize_matrix("q8_0", table, V, width).astype(np.float16)
    head_f = dequantize_matrix("q8_0", head, V, qd).astype(np.float64)
    cos, sin = build_rope_cache(96, hd, 1e4)
    steps = 30
    us = rng.random((steps, B))
    d = {n: up(hip, v) for n, v in dict(table=table, head=head, cos=cos, sin=sin, tok=np.arange(B, dtype=np.int32),
                                        step=np.zeros(1, np.int32), T=np.full(B, 0.8, np.float32),
                                        p=np.full(B, 0.9, np.float32), u=us[0]).items()}
    x, att, logits = empty(hip, (B, width), np.float16), empty(hip, (B, n_q, hd), np.float16), empty(hip, (B, V), np.float32)
    nxt, hist = empty(hip, B, np.int32), empty(hip, (steps, B), np.int32)
    r = bt.rows(start)
    off = bt.d["off"]
    need, sneed = K.attn_pages_scratch_bytes(bt.pages, r, n_q), K.sample_scratch_bytes(B)
    scratch, sscratch = empty(hip, need, np.uint8), empty(hip, sneed, np.uint8)
    st, scale = hip.stream, 1 / math.sqrt(hd)

    def step():
        K.embedding("q8_0", d["tok"], d["table"], x, B, width, stream=st)
        K.kv_pages_append(bt.pages, r, x.ptr + 2 * qd, x.ptr + 2 * (qd + n_kv * hd), q=x, q_out=att, n_q=n_q,
                          rope_cos=d["cos"], rope_sin=d["sin"], rope_rows=96, k_stride=width, v_stride=width,
                          q_stride=width, stream=st)
        K.attn_pages(bt.pages, r, att, att, n_q, scale, scratch, need, stream=st)  # in place
        K.gemv("q8_0", att, d["head"], logits, B, qd, V, in_dtype="f16", out_dtype="f32", stream=st)
        K.sample(logits, B, V, nxt, sscratch, temperature=d["T"], top_p=d["p"], u=d["u"], stream=st)
        K.greedy_advance(nxt, 1, B, d["tok"], off, 95, hist, steps, d["step"], stream=st)

    hip.stream_synchronize()
    hip.stream_begin_capture()
    try:
        step()
    finally:
        g = hip.stream_end_capture()
    ge = hip.graph_instantiate(g)
    toks, pos = np.arange(B), list(start)
    try:
        for i in range(steps):
            d["u"].upload(us[i])
            hip.graph_launch(ge)
            hip.synchronize()
            got = down(logits).astype(np.float64)
            w = rows_f[toks].astype(np.float32).reshape(B, n_q + 2 * n_kv, hd)
            for b in range(B):
                q = okv.rotate(w[b:b + 1, :n_q], [pos[b]], cos, sin).astype(np.float16)[0]
                append_ref(bt, b, pos[b], okv.rotate(w[b:b + 1, n_q:n_q + n_kv], [pos[b]], cos, sin), w[b:b + 1, n_q + n_kv:])
                kv = bt.ref.k[b].values(pos[b] + 1), bt.ref.v[b].values(pos[b] + 1)
                o, mag, big = okv.attention(q, *kv, pos[b], scale)
                tol = attn_tolerance("f16", hd, o, mag, big, np.abs(kv[1]).max()).reshape(-1)
                want = head_f @ o.reshape(-1)
                # the head's products and sums in fp32: 2^-24 of the sum of |products| for each of qd + 8 roundings
                slack = np.abs(head_f) @ tol + (qd + 8) * 2.0 ** -24 * (np.abs(head_f) @ (np.abs(o.reshape(-1)) + tol))
                assert (np.abs(got[b] - want) <= slack).all(), (i, b)
                t, near = osm.sample(got[b], float(np.float32(0.8)), 0, float(np.float32(0.9)), 0.0, us[i, b])
                drawn = int(down(d["tok"])[b])
                assert drawn == t or near < V * 2.0 ** -44
            toks, pos = down(d["tok"]).copy(), [p + 1 for p in pos]
            if i % 10 == 0:
                bt.check(pos)
                check_attention(hip, K, bt, [p - 3 for p in pos], [2] * B, n_q, "f32", rng)  # eager work in between
                off.upload(np.array(pos, np.int32))
                r.kv_offset = off.ptr  # (the check staged its own offsets elsewhere)
                bt.d["off"] = off
        bt.check(pos)
        assert (down(hist) >= 0).all()
    finally:
        hip.graph_exec_destroy(ge)
        hip.graph_destroy(g)


@pytest.mark.parametrize("new", [1, 40])
def test_captured_attention_follows_staged_lengths(hip, K, new):
    """Lengths, rows and pages are read on the device: one captured launch serves other lengths and tables."""
    rng = np.random.default_rng(new)
    bt = filled(hip, K, rng, [300, 170, 64], 2, 128, 32)
    q = normal(rng, (3 * new, 4, 128), "f16")
    dq, do = up(hip, q), empty(hip, q.shape, np.float16)
    r = bt.rows([0, 0, 0], [new] * 3)
    off = bt.d["off"]
    n = K.attn_pages_scratch_bytes(bt.pages, r, 4)
    scratch = empty(hip, n, np.uint8)
    hip.stream_synchronize()
    hip.stream_begin_capture()
    K.attn_pages(bt.pages, r, dq, do, 4, 0.09, scratch, n, stream=hip.stream)
    g = hip.stream_end_capture()
    ge = hip.graph_instantiate(g)
    try:
        for pos in ([300 - new, 170 - new, 64 - new], [0, 0, 0], [17, -1, 5], [300 - new, 3, 0]):
            off.upload(np.array(pos, np.int32))
            hip.graph_launch(ge)
            got = down(do).astype(np.float64)
            for b in range(3):
                kv = bt.ref.k[b].values(bt.ref.cap), bt.ref.v[b].values(bt.ref.cap)
                for i in range(new):
                    o, mag, big = okv.attention(q[b * new + i], *kv, pos[b] + i if pos[b] >= 0 else -1, 0.09,
                                                np.array([not bt.drop(b, t) for t in range(bt.ref.cap)]))
                    tol = attn_tolerance("f16", 128, o, mag, big, 8.0)
                    assert matches("f16", got[b * new + i], o, tol).all(), (pos, b, i)
    finally:
        hip.graph_exec_destroy(ge)
        hip.graph_destroy(g)


def test_two_streams_at_once(hip, K):
    """Prompt and decode attention on two streams that are not the runtime's, each with its own scratch, in turn and
    together: the results of each alone."""
    import ctypes
    rng = np.random.default_rng(41)
    streams = []
    for _ in range(2):
        s = ctypes.c_void_p()
        hip._check_error(hip._lib.hipStreamCreate(ctypes.byref(s)), "hipStreamCreate")
        streams.append(s)
    jobs = []
    for new in (1, 150):
        bt = filled(hip, K, rng, [900, 333], 2, 128, 64)
        q = up(hip, normal(rng, (2 * new, 8, 128), "f16"))
        r = bt.rows([900 - new, 333 - new], [new, new])
        n = K.attn_pages_scratch_bytes(bt.pages, r, 8)
        jobs.append((bt, r, q, empty(hip, (2 * new, 8, 128), np.float16), empty(hip, n, np.uint8), n))
    try:
        alone = []
        for (bt, r, q, o, sc, n), s in zip(jobs, streams):
            K.attn_pages(bt.pages, r, q, o, 8, 0.1, sc, n, stream=s)
            hip.synchronize()
            alone.append(down(o).copy())
        for _ in range(10):
            for (bt, r, q, o, sc, n), s in zip(jobs, streams):
                K.attn_pages(bt.pages, r, q, o, 8, 0.1, sc, n, stream=s)
        hip.synchronize()
        for (_, _, _, o, _, _), a in zip(jobs, alone):
            assert np.array_equal(down(o), a)
    finally:
        for s in streams:
            hip._lib.hipStreamDestroy(s)


def test_offsets_past_32_bits(hip, K):
    """A pool of 5 GiB of K: pages beyond 2^32 bytes are written and read in their places."""
    rng = np.random.default_rng(51)
    page, n_kv, hd = 4096, 2, 128
    n_pages = 5 * 2 ** 30 // (page * n_kv * hd)
    size, blocks = n_pages * page * n_kv * hd, n_pages * n_kv * page // 16
    d = {n: empty_raw(hip, s) for n, s in (("k", size), ("v", size), ("ke", blocks), ("ve", blocks))}
    table = np.array([[n_pages - 1], [1], [n_pages - 2]], np.int32)
    lens = [70, 33, 20]
    ref = okv.Cache(3, n_kv, hd, 1, page)
    new = [up(hip, normal(rng, (sum(lens), n_kv, hd), "f16")) for _ in "kv"]
    k, v = (down(x).astype(np.float32) for x in new)
    first = np.cumsum([0] + lens)
    for b, n in enumerate(lens):
        ref.k[b].append(k[first[b]:first[b + 1]], 0)
        ref.v[b].append(v[first[b]:first[b + 1]], 0)
    dt, off, start = up(hip, table), up(hip, np.zeros(3, np.int32)), up(hip, first.astype(np.int32))
    pages = KVPages.of(d["k"], d["v"], d["ke"], d["ve"], n_pages, page, n_kv, hd)
    rows = KVRows.of(3, sum(lens), max(lens), start, off, dt, 1)
    K.kv_pages_append(pages, rows, *new, stream=hip.stream)
    ko, vo = empty(hip, (3, 80, n_kv, hd), np.float16), empty(hip, (3, 80, n_kv, hd), np.float16)
    K.kv_pages_read(pages, rows, ko, vo, 80, stream=hip.stream)
    for got, parts in ((down(ko), ref.k), (down(vo), ref.v)):
        for b, n in enumerate(lens):
            assert np.array_equal(got[b, :n], parts[b].values(n).astype(np.float16))
    one = KVRows.of(3, 3, 1, None, up(hip, np.array([n - 1 for n in lens], np.int32)), dt, 1)
    for r, q in ((one, normal(rng, (3, 4, hd), "f16")), (rows, normal(rng, (sum(lens), 4, hd), "f16"))):
        n = K.attn_pages_scratch_bytes(pages, r, 4)
        do = empty(hip, q.shape, np.float16)
        K.attn_pages(pages, r, up(hip, q), do, 4, 0.1, empty(hip, n, np.uint8), n, stream=hip.stream)
        got = down(do).astype(np.float64)
        for b, m in enumerate(lens):
            for i in ([m - 1] if r is one else range(m)):
                row = b if r is one else first[b] + i
                o, mag, big = okv.attention(q[row], ref.k[b].values(m), ref.v[b].values(m), i, 0.1)
                assert matches("f16", got[row], o, attn_tolerance("f16", hd, o, mag, big, 8.0)).all()
    for p in d.values():
        hip.safe_free(p)


def empty_raw(hip, nbytes):
    return hip.safe_malloc(nbytes, "pool")
