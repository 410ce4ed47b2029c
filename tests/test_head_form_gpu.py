"""Heads normed and rotated by position on the GPU against the 64-bit oracle: rows of q and k, and on their way into the
8-bit pages."""
import numpy as np
import pytest

from oracle import kv_pages as okv, long_context as olc
from tests._dev import down, empty, up
from tests.test_kv_pages_gpu import NP, Batch, append_ref, normal
from vte_amd.core.rope_cache import rope_frequencies
from vte_amd.kernels import HeadForm

pytestmark = pytest.mark.gpu


class Form:
    """A model's form, on the device and for the oracle."""

    def __init__(self, hip, rng, hd, rot=None, interleaved=False, norms=(True, True), amplitude=1.0, theta=1e6, eps=1e-6):
        self.hip, self.hd, self.eps = hip, hd, eps
        self.w = [(1 + 0.2 * rng.standard_normal(hd)).astype(np.float16) if n else None for n in norms]
        self.turn = dict(freq=None)
        d = [None if w is None else up(hip, w) for w in self.w]
        if rot is not None:
            f, _ = rope_frequencies(rot, theta)
            self.turn = dict(freq=f, rotary_dim=rot, interleaved=interleaved, amplitude=amplitude)
            d.append(up(hip, f))
        else:
            d.append(None)
        self.kept = d
        self.c = HeadForm.of(d[2], rot or 0, interleaved, amplitude, d[0], d[1], eps)

    def of(self, x, pos, is_k):
        return olc.head_form(x, pos, self.w[int(is_k)], self.eps, **self.turn)


def rounded(dtype, y, tol):
    """The bound with the result's own rounding: 2^-11 of it (fp16; steps of 2^-24 below 2^-14), 2^-24 (fp32)."""
    return tol * (1 + 2.0 ** -11) + np.abs(y) * (2.0 ** -11 if dtype == "f16" else 2.0 ** -24) + (2.0 ** -25 if dtype == "f16" else 0)


def check(dtype, got, y, tol, what=""):
    off, most = np.abs(got.astype(np.float64) - y), rounded(dtype, y, tol)
    if not (off <= most).all():
        pytest.fail(f"{what}: {float((off / most).max())} times the bound, {int((~(off <= most)).sum())} values")


FORMS = [(128, 128, False), (128, 64, False), (128, 128, True), (128, 32, True), (64, 64, False), (64, 16, True), (256, 256, False),
         (256, 64, False), (256, 2, True), (128, None, False),
         (128, 24, False), (128, 2, False), (64, 62, False), (256, 200, False), (64, 6, True)]  # (halves of no 8 dims: a pair a lane)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("hd,rot,inter", FORMS)
def test_rows(hip, K, hd, rot, inter, dtype):
    """q and k of ragged row counts, with positions far out, some rows of none, at both ends of the range of sizes."""
    rng = np.random.default_rng(hd + (rot or 1))
    for rows, n_q, n_kv in ((1, 12, 2), (37, 7, 1), (130, 28, 4)):
        f = Form(hip, rng, hd, rot, inter, amplitude=1.2)
        pos = rng.integers(0, 1 << 20, rows).astype(np.int32)
        pos[rows // 3] = 0
        pos[rows // 2 + 1:: 9] = -1
        q, k = normal(rng, (rows, n_q, hd), dtype, 3.0), normal(rng, (rows, n_kv, hd), dtype, 0.01)
        qo, ko = up(hip, np.full_like(q, 7)), up(hip, np.full_like(k, 7))
        K.qk_norm_rope(f.c, rows, up(hip, pos), q=up(hip, q), q_out=qo, n_q=n_q, k=up(hip, k), k_out=ko, n_kv=n_kv, head_dim=hd,
                       dtype=dtype, stream=hip.stream)
        runs = pos >= 0
        for x, out, is_k in ((q, qo, False), (k, ko, True)):
            got = down(out)
            assert (got[~runs] == 7).all()
            check(dtype, got[runs], *f.of(x[runs], pos[runs], is_k), f"{rows} rows, k {is_k}")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("norms", [(True, True), (True, False), (False, True), (False, False)])
def test_rows_without_some_norms_or_positions(hip, K, norms, dtype):
    """A norm of q, of k or of neither; no rotation, and no positions then; q or k alone."""
    rng = np.random.default_rng(3)
    q, k = normal(rng, (9, 5, 128), dtype), normal(rng, (9, 2, 128), dtype)
    for rot in (None, 128):
        f = Form(hip, rng, 128, rot, norms=norms)
        pos = np.arange(9, dtype=np.int32) * 1000
        qo, ko = empty(hip, q.shape, NP[dtype]), empty(hip, k.shape, NP[dtype])
        dp = up(hip, pos) if rot else None
        K.qk_norm_rope(f.c, 9, dp, q=up(hip, q), q_out=qo, n_q=5, dtype=dtype, stream=hip.stream)
        K.qk_norm_rope(f.c, 9, dp, k=up(hip, k), k_out=ko, n_kv=2, dtype=dtype, stream=hip.stream)
        for x, out, is_k in ((q, qo, False), (k, ko, True)):
            if rot is None and not norms[is_k]:
                assert np.array_equal(down(out), x)
            check(dtype, down(out), *f.of(x, pos, is_k))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("rot,inter", [(128, False), (40, False), (96, True)])
def test_rows_in_place_strided_and_misaligned(hip, K, dtype, rot, inter):
    """q and k inside one projection's rows, written in place; the same an element off 16-byte alignment."""
    rng = np.random.default_rng(rot)
    n_q, n_kv, hd, rows = 6, 2, 128, 21
    f = Form(hip, rng, hd, rot, inter)
    pos = np.arange(5, 5 + rows).astype(np.int32)
    width = (n_q + 2 * n_kv) * hd
    for shift in (0, 1):
        flat = normal(rng, rows * (width + shift) + shift, dtype)
        d = up(hip, flat)
        size, ld = flat.itemsize, width + shift
        pq = d.ptr + shift * size
        pk = pq + n_q * hd * size
        K.qk_norm_rope(f.c, rows, up(hip, pos), q=pq, q_out=pq, n_q=n_q, k=pk, k_out=pk, n_kv=n_kv, dtype=dtype, q_stride=ld,
                       k_stride=ld, stream=hip.stream)
        got = down(d)
        x, y = flat[shift:].reshape(rows, ld), got[shift:].reshape(rows, ld)
        assert np.array_equal(got[:shift], flat[:shift])
        assert np.array_equal(y[:, (n_q + n_kv) * hd:], x[:, (n_q + n_kv) * hd:])
        for lo, n, is_k in ((0, n_q, False), (n_q * hd, n_kv, True)):
            part = slice(lo, lo + n * hd)
            check(dtype, y[:, part].reshape(rows, n, hd), *f.of(x[:, part].reshape(rows, n, hd), pos, is_k), f"shift {shift}")


@pytest.mark.parametrize("dtype,hd,rot,rows", [("f16", 64, 24, 2 ** 23 + 1), ("f32", 256, 64, 2 ** 20 + 3)])
def test_rows_of_more_heads_than_a_launch_has_in_one_dimension(hip, K, dtype, hd, rot, rows):
    """8 GiB of heads in place: 2^26 of a pair a lane, 2^23 of 16-byte runs; the rows at the ends, and around where blocks
    begin a second time."""
    rng = np.random.default_rng(rot)
    n_q = 8
    f, size = Form(hip, rng, hd, rot), np.dtype(NP[dtype]).itemsize
    row = n_q * hd * size
    per = 4 if rot == 24 else 8192 // (hd * size)
    again = 2 ** 20 * per // n_q  # (the row at which block 2^20 begins)
    at = sorted({0, 1, rows // 3, again - 1, again, again + 1, min(4 * again, rows - 3), rows - 2, rows - 1})
    assert at[-1] * n_q > 2 ** 20 * per
    d = hip.safe_malloc(rows * row, "rows")
    try:
        x = normal(rng, (len(at), n_q, hd), dtype, 3.0)
        pos = np.full(rows, -1, np.int32)
        pos[at] = rng.integers(0, 1 << 20, len(at))
        pos[at[2]] = -1
        for i, r in enumerate(at):
            hip.safe_memcpy_host_to_device(d.value + r * row, x[i])
        K.qk_norm_rope(f.c, rows, up(hip, pos), q=d, q_out=d, n_q=n_q, head_dim=hd, dtype=dtype, stream=hip.stream)
        hip.synchronize()
        got = np.empty_like(x)
        for i, r in enumerate(at):
            hip.safe_memcpy_device_to_host(got[i], d.value + r * row)
    finally:
        hip.synchronize()
        hip.safe_free(d)
    assert np.array_equal(got[2], x[2])
    live = np.arange(len(at)) != 2
    check(dtype, got[live], *f.of(x[live], pos[at][live], False))


@pytest.mark.parametrize("rot,inter", [(64, False), (64, True), (40, False)])
def test_not_finite_values_stay_in_their_pairs(hip, K, rot, inter):
    """Without a norm an Inf or a NaN reaches its partner in a pair that turns, and nothing else; a row of zeros stays zero
    under a norm."""
    rng = np.random.default_rng(4)
    q = normal(rng, (4, 2, 128), "f32")
    q[0, 0, 3], q[1, 1, 100], q[2, 0, 127] = np.inf, np.nan, -np.inf
    f = Form(hip, rng, 128, rot, inter, norms=(False, False))
    pos = np.arange(1, 5, dtype=np.int32)
    out = empty(hip, q.shape, np.float32)
    K.qk_norm_rope(f.c, 4, up(hip, pos), q=up(hip, q), q_out=out, n_q=2, dtype="f32", stream=hip.stream)
    with np.errstate(invalid="ignore"):
        want, tol = f.of(q, pos, False)
    got, fine = down(out), np.isfinite(want)
    assert np.array_equal(np.isfinite(got), fine)
    assert (np.abs(got - want)[fine] <= rounded("f32", want, tol)[fine]).all()
    f = Form(hip, rng, 128, rot, inter)
    q = np.zeros((2, 2, 128), np.float16)
    out = up(hip, q + np.float16(1))
    K.qk_norm_rope(f.c, 2, up(hip, pos), q=up(hip, q), q_out=out, n_q=2, stream=hip.stream)
    assert (down(out) == 0).all()


def test_positions_up_to_the_end_of_int(hip, K):
    """Angles of positions near 2^30 are off by 2^-51 of them at most: 2^-21 of a radian."""
    rng = np.random.default_rng(5)
    f = Form(hip, rng, 128, 128, norms=(False, False))
    pos = np.array([2 ** 30, 2 ** 30 - 1, 2 ** 31 - 1, 123456789], np.int32)
    q = normal(rng, (4, 3, 128), "f32")
    out = empty(hip, q.shape, np.float32)
    K.qk_norm_rope(f.c, 4, up(hip, pos), q=up(hip, q), q_out=out, n_q=3, dtype="f32", stream=hip.stream)
    check("f32", down(out), *f.of(q, pos, False))


# ---------------------------------------------------------------------------- into the pages
def check_pages_of(bt, b, first, want, tol, name):
    """The device's values of tokens first .. of sequence b: each within half a step of its block's scale (and the value's
    own error) of the oracle's, the scale the smallest that fits (or its neighbour, where the largest value is within its
    error of the border)."""
    codes, exps = down(bt.d[name]), down(bt.d[name + "e"])
    c, e = okv.unpool(codes, exps, bt.table[b], bt.page, name == "v")
    n = first + len(want)
    for blk in range(first // 16, -(-n // 16)):
        lo, hi = max(first, 16 * blk), min(n, 16 * blk + 16)
        w, t = want[lo - first:hi - first], tol[lo - first:hi - first]
        for h in range(w.shape[1]):
            step = 2.0 ** e[blk, h]
            top = np.abs(w[:, h]) - t[:, h], np.abs(w[:, h]) + t[:, h]
            at_least, at_most = okv.exponent(max(top[0].max(), 0.0)), okv.exponent(top[1].max())
            if lo % 16 == 0:  # (else tokens before these have a say)
                assert at_least <= e[blk, h] <= at_most, (name, b, blk, h)
            assert e[blk, h] >= at_least
            off = np.abs(c[lo:hi, h] * step - w[:, h])
            assert (off <= step / 2 + t[:, h]).all(), (name, b, blk, h, float((off - t[:, h]).max() / step))


@pytest.mark.parametrize("page,hd,rot,inter,dtype", [(16, 128, 128, False, "f16"), (64, 128, 64, True, "f32"),
                                                     (32, 64, 32, False, "f16"), (256, 64, 64, True, "f16"),
                                                     (32, 128, 40, False, "f16"), (64, 64, 10, False, "f32"),
                                                     (64, 128, None, False, "f32")])
def test_append_ragged_prompts(hip, K, page, hd, rot, inter, dtype):
    """Chunks of 0 to 200 rows from places inside blocks, a sequence that does not run, pages that are not there, rows past
    the table, rows of nobody, strided rows; q beside; then a token each; other memory stays as it was."""
    rng = np.random.default_rng(page + hd)
    n_kv, n_q = 3, 6
    pos, new = [0, 5, 31, -1, 16, 40, 3], [200, 0, 90, 4, 17, 60, 1]
    lens = [p + n if p >= 0 else 0 for p, n in zip(pos, new)]
    width = max(1, 208 // page)
    holes = [(2, 64 // page, -1), (4, 0, 10 ** 6)] if page <= 64 else [(4, 0, -7)]
    bt = Batch(hip, K, rng, lens, n_kv, hd, page, width=width, holes=holes)
    for b, p in enumerate(pos):
        if p > 0:
            append_ref(bt, b, 0, *[normal(rng, (p, n_kv, hd), "f16", 0.3) for _ in "kv"])
    bt.upload()
    before = {n: down(bt.d[n]).copy() for n in ("k", "v", "ke", "ve")}
    f = Form(hip, rng, hd, rot, inter, amplitude=0.7)
    for new, pad in ((new, 5), ([1] * 7, 0)):
        R = sum(new)
        wide = normal(rng, (R + pad, n_q + 2 * n_kv, hd), dtype)  # q, k and v of one fused projection
        dw, out = up(hip, wide), np.full((R + pad, n_q, hd), 9, NP[dtype])
        do = up(hip, out)
        size, ld = wide.itemsize, wide.shape[1] * hd
        K.kv_pages_append_norm(bt.pages, bt.rows(pos, new, pad), f.c, dw.ptr + n_q * hd * size,
                               dw.ptr + (n_q + n_kv) * hd * size, q=dw, q_out=do, n_q=n_q, dtype=dtype, k_stride=ld, v_stride=ld,
                               q_stride=ld, stream=hip.stream)
        got, first = down(do), np.cumsum([0] + new)
        written = set()
        for b in range(len(pos)):
            n = max(0, min(new[b], bt.ref.cap - pos[b])) if pos[b] >= 0 else 0
            mine = slice(first[b], first[b] + n)
            at = pos[b] + np.arange(n)
            assert (got[first[b] + n:first[b + 1]] == 9).all()
            check(dtype, got[mine], *f.of(wide[mine, :n_q], at, False), f"q of {b}")
            k, tol = f.of(wide[mine, n_q:n_q + n_kv], at, True)
            v = wide[mine, n_q + n_kv:].astype(np.float64)
            runs = np.array([not bt.drop(b, t) for t in at], bool)
            written |= {(int(bt.table[b, t // page]), t % page // 16) for t in at[runs]}
            for lo in np.nonzero(runs & ~np.concatenate([[False], runs[:-1]]))[0]:  # runs of places that exist
                hi = lo + int(np.argmin(np.append(runs[lo:], False)))
                check_pages_of(bt, b, int(at[lo]), k[lo:hi], tol[lo:hi], "k")
                check_pages_of(bt, b, int(at[lo]), v[lo:hi], 0 * v[lo:hi], "v")
        assert (got[R:] == 9).all()
        for n, old in before.items():  # blocks that no new row fell into
            now = down(bt.d[n])
            for p in range(bt.n_pages):
                for i in range(page // 16):
                    if (p, i) not in written:
                        sl = (p, slice(None), slice(16 * i, 16 * i + 16)) if n == "k" else (p, slice(None), i)
                        assert np.array_equal(now[sl], old[sl]), (n, p, i)
        before = {n: down(bt.d[n]).copy() for n in before}
        pos = [p + n if p >= 0 else p for p, n in zip(pos, new)]


@pytest.mark.parametrize("hd,dtype,rot", [(128, "f16", 128), (64, "f32", 20)])
def test_append_token_by_token(hip, K, hd, dtype, rot):
    """Tokens one by one: old ones move by half a step of each raise of their block's scale and no further."""
    rng = np.random.default_rng(hd)
    n_kv, n_q, start = 2, 6, [0, 15, 37]
    bt = Batch(hip, K, rng, [50, 66, 88], n_kv, hd, 32)
    for b, n in enumerate(start):
        for p in (bt.ref.k[b], bt.ref.v[b]):
            p.append(normal(rng, (n, n_kv, hd), "f16"), 0)
    bt.upload()
    f = Form(hip, rng, hd, rot)
    want = [{"k": [], "v": [], "t": []} for _ in start]
    for step in range(50):
        pos = [s + step for s in start]
        size = 2.0 ** rng.uniform(-6, 6)
        q, k, v = (normal(rng, (3, h, hd), dtype, size) for h in (n_q, n_kv, n_kv))
        do = empty(hip, q.shape, NP[dtype])
        K.kv_pages_append_norm(bt.pages, bt.rows(pos), f.c, up(hip, k), up(hip, v), q=up(hip, q), q_out=do, n_q=n_q, dtype=dtype,
                               stream=hip.stream)
        check(dtype, down(do), *f.of(q, pos, False))
        kk, tol = f.of(k, pos, True)
        for b in range(3):
            for n, x in (("k", kk[b]), ("v", v[b]), ("t", tol[b])):
                want[b][n].append(x)
    for n in "kv":
        codes, exps = down(bt.d[n]), down(bt.d[n + "e"])
        for b in range(3):
            c, e = okv.unpool(codes, exps, bt.table[b], bt.page, n == "v")
            at = start[b] + np.arange(50)
            step = 2.0 ** e[at // 16][:, :, None]
            off = np.abs(c[at] * step - np.array(want[b][n], np.float64))
            assert (off <= step + (np.array(want[b]["t"]) if n == "k" else 0)).all()  # 1/2 + 1/4 + ... of the last step


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("rot,inter", [(128, False), (64, True), (24, False)])
def test_append_from_unaligned_rows(hip, K, dtype, rot, inter):
    """q, k and v inside rows of an odd length, an element off 16-byte alignment, weights 2 bytes off."""
    rng = np.random.default_rng(rot)
    n_q, n_kv, hd, n = 5, 2, 128, 37
    bt = Batch(hip, K, rng, [n + 11], n_kv, hd, 32)
    f = Form(hip, rng, hd, rot, inter)
    w = [up(hip, np.concatenate([np.zeros(1, np.float16), x])) for x in f.w]
    f.c.q_norm, f.c.k_norm = w[0].ptr + 2, w[1].ptr + 2
    ld = (n_q + 2 * n_kv) * hd + 3
    flat = normal(rng, n * ld + 1, dtype)
    d, do = up(hip, flat), empty(hip, (n, n_q, hd), NP[dtype])
    size = flat.itemsize
    K.kv_pages_append_norm(bt.pages, bt.rows([11], [n]), f.c, d.ptr + size * (1 + n_q * hd), d.ptr + size * (1 + (n_q + n_kv) * hd),
                           q=d.ptr + size, q_out=do, n_q=n_q, dtype=dtype, k_stride=ld, v_stride=ld, q_stride=ld,
                           stream=hip.stream)
    x = flat[1:].reshape(n, ld)[:, :-3].reshape(n, n_q + 2 * n_kv, hd)
    at = 11 + np.arange(n)
    check(dtype, down(do), *f.of(x[:, :n_q], at, False))
    k, tol = f.of(x[:, n_q:n_q + n_kv], at, True)
    # (what stood in the first block's pages before has a say in its scale)
    check_pages_of(bt, 0, 16, k[5:], tol[5:], "k")
    check_pages_of(bt, 0, 16, x[5:, n_q + n_kv:].astype(np.float64), 0 * tol[5:], "v")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_append_with_an_empty_form(hip, K, dtype):
    """No norms and no rotation: the plain append's bytes, and q as it was; 200 sequences of none to three rows, in place."""
    rng = np.random.default_rng(20)
    new = [int(x) for x in rng.integers(0, 4, 200)]
    pos = [int(p) if b % 7 else -1 for b, p in enumerate(rng.integers(0, 40, 200))]
    lens = [max(p, 0) + n for p, n in zip(pos, new)]
    a = Batch(hip, K, rng, lens, 1, 64, 16, width=3)
    R = sum(new)
    q, k, v = normal(rng, (R, 2, 64), dtype), up(hip, normal(rng, (R, 1, 64), dtype)), up(hip, normal(rng, (R, 1, 64), dtype))
    r = a.rows(pos, new)
    K.kv_pages_append(a.pages, r, k, v, dtype=dtype, stream=hip.stream)
    want = [down(a.d[n]).copy() for n in ("k", "v", "ke", "ve")]
    a.upload()
    r = a.rows(pos, new)
    f, dq = Form(hip, rng, 64, None, norms=(False, False)), up(hip, q)
    K.kv_pages_append_norm(a.pages, r, f.c, k, v, q=dq, q_out=dq, n_q=2, dtype=dtype, stream=hip.stream)
    assert all(np.array_equal(down(a.d[n]), w) for n, w in zip(("k", "v", "ke", "ve"), want))
    assert np.array_equal(down(dq), q)


@pytest.mark.parametrize("batch", [3, 64, 65, 200])
def test_append_to_many_sequences(hip, K, batch):
    """A few rows of each of many sequences, some of none, some that do not run, rows of nobody before the first one's."""
    rng = np.random.default_rng(batch)
    new = [int(n) for n in rng.integers(0, 4, batch)]
    new[1] = 3
    pos = [int(p) if b % 7 else -1 for b, p in enumerate(rng.integers(0, 40, batch))]
    bt = Batch(hip, K, rng, [max(p, 0) + n for p, n in zip(pos, new)], 2, 64, 16, width=3)
    r = bt.rows(pos, new, pad=2)
    start = (2 + np.concatenate([[0], np.cumsum(new)])).astype(np.int32)
    bt.d["start"] = up(hip, start)
    r.row_start = bt.d["start"].ptr
    R = int(start[-1])
    for n_q in (1, 6):
        f = Form(hip, rng, 64, 64)
        q, k, v = normal(rng, (R, n_q, 64), "f16"), normal(rng, (R, 2, 64), "f16"), normal(rng, (R, 2, 64), "f16")
        do = up(hip, np.full(q.shape, 9, np.float16))
        K.kv_pages_append_norm(bt.pages, r, f.c, up(hip, k), up(hip, v), q=up(hip, q), q_out=do, n_q=n_q, stream=hip.stream)
        got = down(do)
        assert (got[:2] == 9).all()
        for b, n in enumerate(new):
            mine = slice(int(start[b]), int(start[b + 1]))
            if pos[b] < 0:
                assert (got[mine] == 9).all()
            elif n:
                at = pos[b] + np.arange(n)
                check("f16", got[mine], *f.of(q[mine], at, False), f"{n_q} heads, sequence {b}")
                kk, tol = f.of(k[mine], at, True)
                check_pages_of(bt, b, pos[b], kk, tol, "k")
                check_pages_of(bt, b, pos[b], v[mine].astype(np.float64), 0 * tol, "v")


def test_captured_heads_follow_staged_positions(hip, K):
    """Rows in place and an append as one graph, replayed with other positions, eager work between."""
    rng = np.random.default_rng(22)
    bt = Batch(hip, K, rng, [60, 60], 2, 128, 32)
    f = Form(hip, rng, 128, 64, True)
    q, k, v = (normal(rng, (2, h, 128), "f16") for h in (4, 2, 2))
    dq, do, dk, dv, ko = up(hip, q), empty(hip, q.shape, np.float16), up(hip, k), up(hip, v), empty(hip, k.shape, np.float16)
    r = bt.rows([0, 0])
    off = bt.d["off"]
    hip.stream_synchronize()
    hip.stream_begin_capture()
    K.kv_pages_append_norm(bt.pages, r, f.c, dk, dv, q=dq, q_out=do, n_q=4, stream=hip.stream)
    K.qk_norm_rope(f.c, 2, off, k=dk, k_out=ko, n_kv=2, stream=hip.stream)
    g = hip.stream_end_capture()
    ge = hip.graph_instantiate(g)
    try:
        for pos in ([0, 3], [17, 40], [33, 0], [59, 48]):
            off.upload(np.array(pos, np.int32))
            hip.graph_launch(ge)
            hip.synchronize()
            check("f16", down(do), *f.of(q, pos, False))
            kk, tol = f.of(k, pos, True)
            check("f16", down(ko), kk, tol)
            eager = empty(hip, k.shape, np.float16)
            K.qk_norm_rope(f.c, 2, off, k=dk, k_out=eager, n_kv=2, stream=hip.stream)
            assert np.array_equal(down(eager), down(ko))
            for b in range(2):
                if pos[b] % 16 == 0:
                    check_pages_of(bt, b, pos[b], kk[b:b + 1], tol[b:b + 1], "k")
    finally:
        hip.graph_exec_destroy(ge)
        hip.graph_destroy(g)


def test_append_not_finite(hip, K):
    """A row of k with an Inf or a NaN makes its block read as NaN, and no other."""
    rng = np.random.default_rng(6)
    bt = Batch(hip, K, rng, [40], 2, 128, 16)
    k, v = (normal(rng, (40, 2, 128), "f16") for _ in "kv")
    k[3, 0, 5], k[36, 1, 0], v[20, 1, 63] = np.inf, np.nan, -np.inf
    f = Form(hip, rng, 128, 128)
    K.kv_pages_append_norm(bt.pages, bt.rows([0], [40]), f.c, up(hip, k), up(hip, v), stream=hip.stream)
    for n, bad in (("k", {(0, 0), (2, 1)}), ("v", {(1, 1)})):
        _, e = okv.unpool(down(bt.d[n]), down(bt.d[n + "e"]), bt.table[0], 16, n == "v")
        assert {(int(i), int(h)) for i, h in zip(*np.nonzero(e[:3] == okv.E_NAN))} == bad
