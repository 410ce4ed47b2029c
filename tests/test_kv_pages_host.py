"""The 8-bit paged cache and the device draw without a GPU: refusals of the C ABI (nothing is launched), and the
oracles against closed forms."""
import ctypes

import numpy as np
import pytest

from oracle import kv_pages as okv, sampling as osm
from vte_amd.bridge.hip_runtime import HIPSafetyError
from vte_amd.kernels import KVPages, KVRows, kernels

P = 4096  # a 16-byte aligned address that nothing dereferences


def pages(**kw):
    a = dict(k=P, v=P, k_exp=P, v_exp=P, n_pages=4, page_tokens=64, n_kv=2, head_dim=128) | kw
    return KVPages.of(**a)


def rows(**kw):
    a = dict(batch=3, rows=3, max_rows=1, row_start=None, kv_offset=P, page_table=P, max_pages=2) | kw
    return KVRows.of(**a)


BAD_PAGES = [dict(head_dim=96), dict(head_dim=0), dict(n_kv=0), dict(n_pages=0), dict(page_tokens=8),
             dict(page_tokens=48), dict(page_tokens=8192), dict(page_tokens=0)]
BAD_ROWS = [dict(batch=0), dict(batch=65536, rows=65536), dict(rows=2), dict(max_rows=2), dict(rows=-1),
            dict(max_pages=0), dict(max_pages=(1 << 30) // 64 + 1), dict(rows=4, row_start=P, max_rows=5),
            dict(rows=(1 << 24) + 1, row_start=P)]
BAD_MEMORY = [dict(k=None), dict(v=None), dict(k_exp=None), dict(v_exp=None), dict(k=P + 8), dict(v=P + 1)]


def calls(c, r):
    K = kernels()
    return [lambda: K.kv_pages_append(c, r, P, P), lambda: K.kv_pages_read(c, r, P, P, 64),
            lambda: K.attn_pages(c, r, P, P, 4, 0.1, P, 1 << 40)]


@pytest.mark.parametrize("bad", BAD_PAGES + BAD_MEMORY, ids=str)
def test_bad_caches_are_refused(bad):
    for call in calls(pages(**bad), rows()):
        with pytest.raises(HIPSafetyError):
            call()


@pytest.mark.parametrize("bad", BAD_ROWS + [dict(kv_offset=None), dict(page_table=None), dict(kv_offset=P + 2)], ids=str)
def test_bad_rows_are_refused(bad):
    for call in calls(pages(), rows(**bad)):
        with pytest.raises(HIPSafetyError):
            call()


def test_no_rows_read_but_neither_append_nor_attend():
    c, r = pages(), rows(rows=0, max_rows=0)
    for call in (calls(c, r)[0], calls(c, r)[2]):
        with pytest.raises(HIPSafetyError, match="no rows"):
            call()


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(k=P + 1), dict(k_stride=255), dict(v_stride=-256),
                                 dict(q=P), dict(q=P, q_out=P, n_q=4), dict(rope_cos=P), dict(dtype="f32", k=P + 2),
                                 dict(rope_cos=P, rope_sin=P, rope_rows=0), dict(q=P, q_out=P, n_q=0, rope=1),
                                 dict(rope=1, rope_type=3), dict(rope=1, rope_type=2, rotary_dim=3),
                                 dict(rope=1, rope_type=2, rotary_dim=130), dict(q=P, q_out=P, n_q=4, q_stride=511, rope=1),
                                 dict(q=P, q_out=P, n_q=4, q_stride=1024, rope=1),
                                 dict(q=P, q_out=P + 8, n_q=65535, r=dict(batch=1, rows=1 << 10, row_start=P), rope=1)], ids=str)
def test_append_refusals(bad):
    a = dict(k=P, v=P) | bad
    r = a.pop("r", {})
    if a.pop("rope", 0):
        a = dict(rope_cos=P, rope_sin=P, rope_rows=10) | a
    with pytest.raises(HIPSafetyError):
        kernels().kv_pages_append(pages(), rows(**r), **a)


def test_read_and_attention_refusals():
    K, c, r = kernels(), pages(), rows()
    need = K.attn_pages_scratch_bytes(c, r, 12)
    assert need > 0
    for call in (lambda: K.kv_pages_read(c, r, None, P, 64), lambda: K.kv_pages_read(c, r, P, P, 0),
                 lambda: K.kv_pages_read(c, r, P + 2, P, 64),
                 lambda: K.kv_pages_read(pages(n_kv=4, page_tokens=4096), rows(max_pages=1 << 14), P, P, (1 << 25) + 1),
                 lambda: K.attn_pages(c, r, P, P, 12, 0.1, P, need - 1),
                 lambda: K.attn_pages(c, r, P, P, 12, 0.1, None, need),
                 lambda: K.attn_pages(c, r, P, P, 12, 0.1, P + 4, need),
                 lambda: K.attn_pages(c, r, P + 2, P, 12, 0.1, P, need),
                 lambda: K.attn_pages(c, r, P, P, 12, 0.0, P, need),
                 lambda: K.attn_pages(c, r, P, P, 12, float("nan"), P, need),
                 lambda: K.attn_pages(c, r, P, P, 13, 0.1, P, need),   # no multiple of n_kv
                 lambda: K.attn_pages(c, r, P, P, 34, 0.1, P, 1 << 40),  # 17 heads of one KV head
                 lambda: K.attn_pages_scratch_bytes(c, r, 34),
                 lambda: K.attn_pages_scratch_bytes(pages(n_kv=16), rows(rows=(1 << 21) + 1, max_rows=9, row_start=P), 16),
                 lambda: K.attn_pages_scratch_bytes(pages(n_kv=32), rows(batch=32769, rows=32769), 32)):
        with pytest.raises(HIPSafetyError):
            call()
    lib, ref = K.lib, ctypes.byref
    assert lib.vte_attn_pages(ref(c), ref(r), 2, P, P, 12, ctypes.c_float(0.1), P, need, None) == -1
    assert lib.vte_attn_pages(None, ref(r), 1, P, P, 12, ctypes.c_float(0.1), P, need, None) == -1
    assert lib.vte_kv_pages_read(ref(c), None, 1, P, P, 4, None) == -1


@pytest.mark.parametrize("bad", [dict(logits=None), dict(u=None), dict(tokens=None), dict(scratch=None), dict(rows=0),
                                 dict(rows=65536), dict(vocab=0), dict(vocab=262145), dict(logits=P + 2),
                                 dict(u=P + 4), dict(scratch=P + 8), dict(tokens=P + 2), dict(temperature=P + 1),
                                 dict(top_k=P + 2), dict(top_p=P + 3), dict(min_p=P + 2)], ids=str)
def test_sample_refusals(bad):
    a = dict(logits=P, rows=2, vocab=100, tokens=P, scratch=P, u=P) | bad
    with pytest.raises(HIPSafetyError):
        kernels().sample(**a)


# ---------------------------------------------------------------------------- the oracles
@pytest.mark.parametrize("amax,e", [(0.0, -126), (127.0, 0), (127.5, 1), (254.0, 1), (1.0, -6), (0.9921875, -7),
                                    (0.99218756, -6), (1e-45, -126), (65504.0, 10), (3.3e38, 121), (3.4e38, 122)])
def test_exponent(amax, e):
    assert okv.exponent(float(np.float32(amax))) == e
    assert e == okv.E_MIN or np.float32(amax) > 127 * 2.0 ** (e - 1)


def test_append_one_by_one_stays_within_one_step():
    """Every raise of a block's scale rounds its tokens again: 1/2 step of the last scale, 1/4 from the one before, ..."""
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((48, 2, 64)) * 2.0 ** rng.uniform(-6, 6, (48, 1, 1))).astype(np.float16).astype(np.float64)
    one, all_ = okv.Part(2, 64, 64), okv.Part(2, 64, 64)
    for t in range(48):
        one.append(x[t:t + 1], t)
    all_.append(x, 0)
    step = 2.0 ** np.repeat(one.e, 16, 0)[:48, :, None]
    assert (np.abs(one.values(48) - x) < step).all()
    assert (np.abs(all_.values(48) - x) <= 2.0 ** np.repeat(all_.e, 16, 0)[:48, :, None] / 2).all()
    assert np.array_equal(one.e, all_.e)


def test_pool_and_unpool_are_inverse():
    rng = np.random.default_rng(2)
    c = okv.Cache(2, 3, 64, 2, 32)
    for b in range(2):
        c.k[b].append(rng.standard_normal((50, 3, 64)), 0)
        c.v[b].append(rng.standard_normal((50, 3, 64)), 0)
    table = np.array([[3, 0], [1, -1]])
    for is_v, parts in ((False, c.k), (True, c.v)):
        codes, exps = c.pool(table, 4, is_v)
        for b in range(2):
            got, e = okv.unpool(codes, exps, table[b], 32, is_v)
            n = 64 if b == 0 else 32
            assert np.array_equal(got[:n], parts[b].c[:n]) and np.array_equal(e[:n // 16], parts[b].e[:n // 16])


def test_sampling_oracle_equals_the_host_sampler():
    """0 < top_p < 1: the host sampler's draw for the same random number (its masses are fp32)."""
    from vte_amd.core.sampler import Sampler
    rng = np.random.default_rng(3)
    agree = 0
    for i in range(40):
        x = (3 * rng.standard_normal(500)).astype(np.float32)
        state = np.random.default_rng(100 + i)
        u = np.random.default_rng(100 + i).random()
        want = Sampler.sample(x, 0.7, 0.9, 40, 1.0, rng=state)
        got, near = osm.sample(x, 0.7, 40, 0.9, 0.0, u)
        assert got == want or near < 1e-5
        agree += got == want
    assert agree >= 38


@pytest.mark.parametrize("u,token", [(0.0, 1), (0.49, 1), (0.51, 0), (0.74, 0), (0.76, 2), (0.999, 3), (1.0, 3)])
def test_sampling_oracle_closed_form(u, token):
    x = np.log(np.array([2, 4, 1, 1], np.float32))
    assert osm.sample(x, u=u)[0] == token
    assert osm.sample(x, top_k=1, u=u)[0] == 1 and osm.sample(x, temperature=0, u=u)[0] == 1
    assert osm.sample(x, min_p=0.4, u=u)[0] in (0, 1) and osm.sample(x, top_p=0.4, u=u)[0] == 1


def test_sample_scratch_of_more_rows_serves_fewer():
    """Memory sized for the largest batch is enough as sequences end: the size never falls with the rows, at the borders
    of 8 parts a row and fewer (32, 36, 42, 51, 64, 85 and 128 rows on 256 compute units) and elsewhere."""
    K = kernels()
    size = [K.sample_scratch_bytes(r) for r in range(1, 3000)] + [K.sample_scratch_bytes(65535)]
    assert size[0] > 0 and all(a <= b for a, b in zip(size, size[1:]))


def test_sample_scratch_of_fewer_bytes_is_refused():
    K = kernels()
    with pytest.raises(HIPSafetyError, match="scratch"):
        K.sample(P, 33, 100, P, P, u=P, scratch_bytes=K.sample_scratch_bytes(33) - 1)
