"""Paged 8-bit attention where tokens' sizes lie far apart: every result within bounds counted from what each token
contributes (its weight times its |V|), not from the largest |V|."""
import math

import numpy as np
import pytest

from oracle import kv_pages as okv
from tests._dev import down, empty, up
from tests.test_kv_pages_gpu import NP, Batch, append_ref, filled, normal

pytestmark = pytest.mark.gpu


def weighted(q, k, v, unit, pos, scale, dtype, chain, small):
    """(result, bound of its error) of rows q [rows, hd] of one head over values k, v [tokens, hd] whose V blocks have
    scales ``unit`` [tokens], row i at pos[i]; 64 bits.

    The result's rounding: 2^-11 of it (fp16; 2^-25 below 2^-14), 2^-24 (fp32).  A weight: two fp16 parts, a rounded
    one and a rounded rest of at most 2^-11 of it (2^-22), 2^-20 with the exponential's own rounding; where the rest is
    below the normal fp16 numbers, ``small`` of the largest weight times scale, for each of n tokens of 127 steps at most.
    A score: sums of hd + 3 roundings of 2^-24 of the sum of |q k| (fp32 q as two fp16 parts: 2^-21 more), which
    reach the result by the token's weight, in both sums.  Sums: ``chain`` roundings of 2^-24 one after the other."""
    s = q @ k.T * scale
    s[np.arange(len(k))[None] > np.asarray(pos)[:, None]] = -np.inf
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    err = p * (np.abs(q) @ np.abs(k).T * scale * ((q.shape[1] + 3) * 2.0 ** -24 + (2.0 ** -21 if dtype == "f32" else 0)))
    out, mag = p @ v, p @ np.abs(v)
    n = np.minimum(np.asarray(pos) + 1, len(k))
    tol = (2.0 ** -20 + chain * 2.0 ** -24) * mag + err @ np.abs(v) + err.sum(1)[:, None] * np.abs(out)
    tol += (n * 127 * small * (p * unit).max(1))[:, None]
    return out, tol + (2.0 ** -11 * np.abs(out) + 2.0 ** -25 if dtype == "f16" else 2.0 ** -24 * np.abs(out))


def run(hip, K, bt, pos, new, n_q, dtype, q, scale):
    r = bt.rows(pos, new)
    need = K.attn_pages_scratch_bytes(bt.pages, r, n_q)
    scratch, out = up(hip, np.full(need, 0xFF, np.uint8)), empty(hip, q.shape, NP[dtype])
    K.attn_pages(bt.pages, r, up(hip, q), out, n_q, scale, scratch, need, dtype=dtype, stream=hip.stream)
    return down(out).astype(np.float64)


def check(hip, K, bt, b, pos, new, n_q, dtype, q, before=None, chain=None, small=2.0 ** -38, what=()):
    """Rows of sequence b of a batch (those at positions below ``before``).  ``small``: probabilities as 2^14 of the
    heaviest token's, half the smallest fp16 is 2^-25, and a power of two between."""
    scale = 1 / math.sqrt(bt.hd)
    got = run(hip, K, bt, pos, new, n_q, dtype, q, scale)[sum(new[:b]):sum(new[:b + 1])]
    got = got[:new[b] if before is None else min(new[b], before - pos[b])]
    n = pos[b] + len(got)
    k, v = bt.ref.k[b].values(n), bt.ref.v[b].values(n)
    unit = 2.0 ** np.repeat(bt.ref.v[b].e, okv.BLOCK, 0)[:n].astype(np.float64)
    for h in range(n_q):
        j = h // (n_q // bt.n_kv)
        o, tol = weighted(q[sum(new[:b]):][:len(got), h].astype(np.float64), k[:, j], v[:, j], unit[:, j],
                          pos[b] + np.arange(len(got)), scale, dtype, n + 32 if chain is None else chain, small)
        off = np.abs(got[:, h] - o)
        if not (off <= tol).all():
            pytest.fail(f"{what} head {h}: {float((off / tol).max())} times the bound, {int((~(off <= tol)).sum())} values")


@pytest.mark.parametrize("new,n_q,n_kv,hd", [(1, 12, 2, 128), (3, 4, 1, 64), (130, 12, 2, 128), (300, 7, 1, 64),
                                             (70, 32, 2, 128)])
def test_fp16_results_are_off_by_their_own_rounding(hip, K, new, n_q, n_kv, hd):
    """fp16 in and out: the probabilities' rounding is not seen beside the result's.  (A prompt's probabilities are 2^9
    of the largest, V of ordinary blocks of one scale: 2^-34 of it for half the smallest fp16.)"""
    rng = np.random.default_rng(new + hd)
    bt = filled(hip, K, rng, [700, 331], n_kv, hd, 64)
    pos = [700 - new, 331 - new]
    q = normal(rng, (2 * new, n_q, hd), "f16")
    for b in range(2):
        # sums: 16 tokens an instruction, two parts of each, 32 for exponentials and rescaling
        check(hip, K, bt, b, pos, [new, new], n_q, "f16", q, chain=2 * 700 // 16 + 32,
              small=2.0 ** -38 if new * n_q // n_kv <= 16 else 2.0 ** -33)


def sized(hip, K, rng, n, n_kv, hd, v_size, batch=1, **kw):
    """Sequence 0 of n tokens whose V are v_size [n] times normal ones (``batch`` - 1 empty ones behind it)."""
    bt = Batch(hip, K, rng, [n] + [0] * (batch - 1), n_kv, hd, 64, **kw)
    k, v = rng.standard_normal((2, n, n_kv, hd)).astype(np.float32)
    append_ref(bt, 0, 0, k, v * np.asarray(v_size, np.float32)[:, None, None])
    bt.upload()
    return bt


@pytest.mark.parametrize("new,n_q,n_kv,hd,batch", [(128, 1, 1, 128, 1), (70, 2, 1, 64, 1), (600, 16, 1, 128, 1),
                                                   (130, 16, 4, 64, 160), (4, 4, 1, 128, 1)])
@pytest.mark.parametrize("at", [448, 704, 720])
def test_values_of_2_to_130_times_behind_a_row(hip, K, new, n_q, n_kv, hd, batch, at):
    """V of tokens that a row does not see are 2^130 times those that it sees, from a border of a step on and inside one:
    groups and shares of which a row sees nothing leave its result alone."""
    rng = np.random.default_rng(new + at)
    n = min(800, at + new // 2)
    bt = sized(hip, K, rng, n, n_kv, hd, np.where(np.arange(n) < at, 2.0 ** -10, 2.0 ** 120), batch)
    q = normal(rng, (new, n_q, hd), "f32")
    check(hip, K, bt, 0, [n - new] + [-1] * (batch - 1), [new] + [0] * (batch - 1), n_q, "f32", q, before=at)


@pytest.mark.parametrize("n_kv,batch", [(4, 160), (1, 1)])
def test_values_that_grow_twice_behind_a_row(hip, K, n_kv, batch):
    """V grow by 2^80 and, a step later, by 2^80 again, each less than fp32 holds, together more: rows before the first
    growth, and those between the two.  (Of 160 sequences the row blocks are 256 rows, which span both.)"""
    rng = np.random.default_rng(n_kv)
    n, new = 900, 300
    bt = sized(hip, K, rng, n, n_kv, 64, 2.0 ** np.repeat([-80.0, 0.0, 80.0], [704, 64, 132]), batch)
    q = normal(rng, (new, n_kv, 64), "f32")
    pos, rows = [n - new] + [-1] * (batch - 1), [new] + [0] * (batch - 1)
    check(hip, K, bt, 0, pos, rows, n_kv, "f32", q, before=704)
    check(hip, K, bt, 0, pos, rows, n_kv, "f32", q, before=768)


@pytest.mark.parametrize("new,n_q", [(1, 4), (4, 4), (70, 2), (150, 16)])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("at", [0, 64, 96, 128])
def test_a_huge_value_of_vanishing_weight(hip, K, dtype, new, n_q, at):
    """A block's V is 2^power times the others', its tokens' probability 2^-drop of theirs: what the others contribute
    stays, whichever is heavier, wherever the block lies."""
    hd, n = 128, 300
    for power, drop in ((40, 100), (120, 160), (60, 60), (20, 26), (20, 33), (14, 30), (30, 45), (12, 40), (110, 100)):
        rng = np.random.default_rng(power + drop)
        bt = Batch(hip, K, rng, [n], 1, hd, 64)
        k, v = rng.standard_normal((2, n, 1, hd)).astype(np.float32)
        k[:, :, 0] = 0
        k[at:at + 16, :, 0] = -drop * math.log(2) * math.sqrt(hd) / 16
        v[at:at + 16] *= 2.0 ** power
        append_ref(bt, 0, 0, k, v)
        bt.upload()
        q = normal(rng, (new, n_q, hd), dtype)
        q[:, :, 0] = 16
        few = n_q * new <= 16
        check(hip, K, bt, 0, [n - new], [new], n_q, dtype, q, chain=2 * n // 16 + 32 if few else None,
              small=2.0 ** -38 if power > 12 or few else 2.0 ** -22, what=(power, drop))


def test_equal_bits_in_other_pages(hip, K):
    """The same batch in other pages: its sums are cut at the same places, so its bits are equal.  (In another batch they
    are cut elsewhere, and equal within the bounds only.)"""
    for new in (1, 30):
        rng = np.random.default_rng(new)
        bt = filled(hip, K, rng, [700, 40, 333], 2, 128, 64)
        other = Batch(hip, K, rng, [700, 40, 333], 2, 128, 64, spare=9)
        other.ref = bt.ref
        other.upload()
        q = normal(rng, (3 * new, 4, 128), "f16")
        pos = [700 - new, 40 - new, 333 - new]
        a, b = (run(hip, K, x, pos, [new] * 3, 4, "f16", q, 0.09) for x in (bt, other))
        assert np.array_equal(a, b)
        alone = Batch(hip, K, rng, [700], 2, 128, 64, spare=5)
        alone.ref.k[0], alone.ref.v[0] = bt.ref.k[0], bt.ref.v[0]
        alone.upload()
        for x, p in ((bt, pos), (alone, pos[:1])):
            check(hip, K, x, 0, p, [new] * len(p), 4, "f16", q[:new * len(p)], small=2.0 ** -33)
