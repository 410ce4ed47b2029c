"""Oracle of the 8-bit paged KV cache: append, read and attention in 64 bits, block by block (test oracle only).

``Cache`` keeps each sequence as whole numbers [tokens][n_kv][hd] and exponents [blocks][n_kv] for K and V;
``pool`` lays them out in pages as the kernels do, ``unpool`` takes them back out.
"""
from __future__ import annotations

import numpy as np

BLOCK, E_MIN, E_NAN = 16, -126, -128


def exponent(amax: float) -> int:
    """The smallest e >= E_MIN with amax <= 127 * 2^e."""
    if amax == 0:
        return E_MIN
    e = int(np.ceil(np.log2(amax / 127.0)))
    while amax > 127.0 * 2.0 ** e:
        e += 1
    while e > E_MIN and amax <= 127.0 * 2.0 ** (e - 1):
        e -= 1
    return max(e, E_MIN)


def rotate(x, pos, cos, sin, rope_type=0, rotary_dim=0):
    """x [n, heads, hd] (fp32 values) at positions pos; products and sums rounded to fp32 one by one."""
    x = np.asarray(x, np.float32)
    out = x.copy()
    hd = x.shape[2]
    n = rotary_dim if rope_type == 2 else hd
    i = np.arange(n // 2)
    a, b = (2 * i, 2 * i + 1) if rope_type == 1 else (i, i + n // 2)
    c = np.asarray(cos, np.float32)[pos][:, None, :n // 2]
    s = np.asarray(sin, np.float32)[pos][:, None, :n // 2]
    with np.errstate(invalid="ignore", over="ignore"):
        out[:, :, a] = x[:, :, a] * c - x[:, :, b] * s
        out[:, :, b] = x[:, :, a] * s + x[:, :, b] * c
    return out


class Part:
    """K or V of one sequence."""

    def __init__(self, n_kv, hd, capacity):
        self.c = np.zeros((capacity, n_kv, hd), np.int64)
        self.e = np.full((capacity // BLOCK, n_kv), E_MIN, np.int64)

    def append(self, x, pos):
        """Rows x [n, n_kv, hd] (exact values) at pos, pos + 1, ...; the caller cuts them to the capacity."""
        x = np.asarray(x, np.float64)
        n, n_kv, _ = x.shape
        for blk in range(pos // BLOCK, (pos + n - 1) // BLOCK + 1) if n else ():
            t0 = blk * BLOCK
            j0, j1 = max(pos - t0, 0), min(pos + n - t0, BLOCK)
            new = x[t0 + j0 - pos:t0 + j1 - pos]
            for h in range(n_kv):
                old = int(self.e[blk, h]) if j0 else E_MIN
                if not np.isfinite(new[:, h]).all() or old == E_NAN:
                    self.e[blk, h] = E_NAN
                    self.c[t0 + j0:t0 + j1, h] = 0
                    continue
                e = max(old, exponent(np.abs(new[:, h]).max()))
                if j0 and e > old:
                    self.c[t0:t0 + j0, h] = np.rint(self.c[t0:t0 + j0, h] * 2.0 ** (old - e))
                self.c[t0 + j0:t0 + j1, h] = np.rint(np.ldexp(new[:, h], -e))
                self.e[blk, h] = e

    def values(self, n):
        e = np.repeat(self.e, BLOCK, 0)[:n, :, None]
        return np.where(e == E_NAN, np.nan, np.ldexp(self.c[:n].astype(np.float64), np.maximum(e, E_MIN)))


class Cache:
    def __init__(self, batch, n_kv, hd, max_pages, page):
        self.page, self.cap = page, max_pages * page
        self.k = [Part(n_kv, hd, self.cap) for _ in range(batch)]
        self.v = [Part(n_kv, hd, self.cap) for _ in range(batch)]

    def pool(self, table, n_pages, is_v, fill=77):
        """Pages of bytes and exponents; memory that belongs to nobody holds ``fill``."""
        parts = self.v if is_v else self.k
        _, n_kv, hd = parts[0].c.shape
        bp = self.page // BLOCK
        codes = np.full((n_pages, n_kv, bp, hd, BLOCK) if is_v else (n_pages, n_kv, self.page, hd), fill, np.uint8)
        exps = np.full((n_pages, n_kv, bp), fill, np.int8)
        for b, part in enumerate(parts):
            for j, p in enumerate(table[b]):
                if 0 <= p < n_pages:
                    c = (part.c[j * self.page:(j + 1) * self.page] + 128).astype(np.uint8).transpose(1, 0, 2)
                    codes[p] = c.reshape(n_kv, bp, BLOCK, hd).transpose(0, 1, 3, 2) if is_v else c
                    exps[p] = part.e[j * bp:(j + 1) * bp].T
        return codes, exps


def unpool(codes, exps, row, page, is_v):
    """(whole numbers [tokens][n_kv][hd], exponents [blocks][n_kv]) of one table row; 0 where there is no page."""
    n_pages, n_kv, hd = codes.shape[0], codes.shape[1], codes.shape[3]
    c = np.zeros((len(row) * page, n_kv, hd), np.int64)
    e = np.full((len(row) * page // BLOCK, n_kv), E_MIN, np.int64)
    for j, p in enumerate(row):
        if 0 <= p < n_pages:
            x = codes[p].transpose(0, 1, 3, 2).reshape(n_kv, page, hd) if is_v else codes[p]
            c[j * page:(j + 1) * page] = x.transpose(1, 0, 2).astype(np.int64) - 128
            e[j * page // BLOCK:(j + 1) * page // BLOCK] = exps[p].T
    return c, e


def attention(q, k, v, pos, scale, present=None):
    """Row q [n_q, hd] over values k, v [tokens, n_kv, hd] at positions 0..pos (those ``present``): (result, the
    softmax-weighted |V|, the largest sum of |q k| * scale of a seen token), 64 bits.  Sees nothing: zeros."""
    n_q, hd = q.shape
    n_kv = k.shape[1]
    out, mag, big = np.zeros((n_q, hd)), np.zeros((n_q, hd)), np.zeros(n_q)
    seen = np.arange(len(k)) <= pos
    if present is not None:
        seen &= present
    if not seen.any():
        return out, mag, big
    with np.errstate(invalid="ignore"):
        for h in range(n_q):
            kk, vv = k[seen, h // (n_q // n_kv)], v[seen, h // (n_q // n_kv)]
            s = kk @ q[h].astype(np.float64) * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[h], mag[h] = p @ vv, p @ np.abs(vv)
            big[h] = (np.abs(kk) @ np.abs(q[h].astype(np.float64))).max() * scale
    return out, mag, big
