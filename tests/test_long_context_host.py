"""Normed and rotated heads, windows and the pool of pages without a GPU: refusals of the C ABI (nothing is launched),
rotation frequencies, and the oracles against closed forms."""
import ctypes

import numpy as np
import pytest

from oracle import long_context as olc
from tests.test_kv_pages_host import BAD_MEMORY, BAD_PAGES, BAD_ROWS, P, pages, rows
from vte_amd.bridge.hip_runtime import HIPSafetyError
from vte_amd.core.rope_cache import rope_frequencies
from vte_amd.kernels import HeadForm, KVPages, KVTables, kernels


def form(**kw):
    return HeadForm.of(**(dict(freq=P, rotary_dim=128, q_norm=P, k_norm=P) | kw))


def tables(**kw):
    return KVTables.of(**(dict(page_table=P, refs=P, batch=3, max_pages=2, n_pages=4, page_tokens=64) | kw))


def layers(*c):
    return (KVPages * len(c))(*c)


def refused(*calls):
    for call in calls:
        with pytest.raises(HIPSafetyError):
            call()


def paged_calls(c, r):
    K = kernels()
    return [lambda: K.kv_pages_append_norm(c, r, form(), P, P),
            lambda: K.attn_pages_window(c, r, P, P, 4, 0.1, 100, 4, P, 1 << 40)]


@pytest.mark.parametrize("bad", BAD_PAGES + BAD_MEMORY, ids=str)
def test_bad_caches_are_refused(bad):
    refused(*paged_calls(pages(**bad), rows()))


@pytest.mark.parametrize("bad", BAD_ROWS + [dict(kv_offset=None), dict(page_table=None), dict(rows=0, max_rows=0)], ids=str)
def test_bad_rows_are_refused(bad):
    refused(*paged_calls(pages(), rows(**bad)))


def test_window_refusals():
    K, c, r = kernels(), pages(), rows()
    need = K.attn_pages_window_scratch_bytes(c, r, 12, 100, 4)
    assert need > 0
    a = (c, r, P, P, 12, 0.1, 100, 4, P, need)
    refused(*[lambda i=i, x=x: K.attn_pages_window(*a[:i], x, *a[i + 1:])
              for i, x in ((2, None), (2, P + 2), (3, None), (3, P + 8), (4, 13), (4, 34), (5, 0.0), (5, float("nan")), (6, 0),
                           (6, -1), (7, -1), (8, None), (8, P + 4), (9, need - 1))],
            lambda: K.attn_pages_window_scratch_bytes(c, r, 12, 0, 4), lambda: K.attn_pages_window_scratch_bytes(c, r, 13, 1, 0),
            lambda: K.attn_pages_window(c, r, P, P, 12, 2e6, 1, 0, P, need))


def test_window_scratch_goes_by_the_window():
    """A table for 2^20 tokens asks for no more than one for the window's."""
    K, r = kernels(), rows(batch=1, rows=1, max_pages=1 << 14)
    c = pages(n_pages=1 << 14)
    assert K.attn_pages_window_scratch_bytes(c, r, 4, 128, 4) < K.attn_pages_scratch_bytes(c, r, 4)
    assert K.attn_pages_window_scratch_bytes(c, r, 4, 2 ** 31 - 1, 2 ** 31 - 1) == K.attn_pages_scratch_bytes(c, r, 4)


BAD_FORMS = [dict(freq=P + 4), dict(q_norm=P + 1), dict(k_norm=P + 1), dict(eps=0.0), dict(eps=9e-31), dict(eps=-1.0), dict(eps=float("nan")),
             dict(eps=2.0), dict(rotary_dim=3), dict(rotary_dim=-2), dict(rotary_dim=130), dict(amplitude=float("inf")),
             dict(amplitude=float("nan"))]


@pytest.mark.parametrize("bad", BAD_FORMS, ids=str)
def test_bad_forms_are_refused(bad):
    K = kernels()
    refused(lambda: K.qk_norm_rope(form(**bad), 1, P, q=P, q_out=P, n_q=2),
            lambda: K.kv_pages_append_norm(pages(), rows(), form(**bad), P, P))


@pytest.mark.parametrize("bad", [dict(q=None), dict(q_out=None), dict(k=P), dict(positions=None), dict(rows=0),
                                 dict(rows=(1 << 24) + 1), dict(n_q=0), dict(n_q=65536), dict(q_stride=255), dict(q_stride=1 << 31),
                                 dict(q=P + 1), dict(dtype="f32", q_out=P + 2), dict(head_dim=96), dict(head_dim=512),
                                 dict(positions=P + 2), dict(rows=1 << 24, n_q=9), dict(q=None, q_out=None),
                                 dict(k=P, k_out=P, n_kv=0), dict(k=P, k_out=P, n_kv=2, k_stride=100)], ids=str)
def test_qk_norm_rope_refusals(bad):
    a = dict(rows=2, positions=P, q=P, q_out=P, n_q=2) | bad
    refused(lambda: kernels().qk_norm_rope(form(), **a))


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(k=P + 1), dict(k_stride=255), dict(v_stride=-256), dict(q=P),
                                 dict(dtype="f32", v=P + 2), dict(q=P, q_out=P, n_q=0), dict(q=P, q_out=P, n_q=4, q_stride=511),
                                 dict(q=P, q_out=P, n_q=4, q_stride=1024)], ids=str)
def test_append_norm_refusals(bad):
    refused(lambda: kernels().kv_pages_append_norm(pages(), rows(), form(), **(dict(k=P, v=P) | bad)))


BAD_TABLES = [dict(page_table=None), dict(refs=None), dict(page_table=P + 2), dict(refs=P + 1), dict(batch=0), dict(batch=65536),
              dict(n_pages=0), dict(n_pages=(1 << 24) + 1), dict(page_tokens=8), dict(page_tokens=48), dict(page_tokens=8192),
              dict(max_pages=0), dict(max_pages=(1 << 30) // 64 + 1)]


@pytest.mark.parametrize("bad", BAD_TABLES, ids=str)
def test_bad_tables_are_refused(bad):
    K, t, L = kernels(), tables(**bad), layers(pages())
    refused(lambda: K.kv_pages_free(t, 1), lambda: K.kv_pages_reserve(t, 1, P, 1, P),
            lambda: K.kv_pages_fork(L, t, 1, P, P, P, P, P, 1 << 20),
            lambda: K.kv_pages_compact(L, t, P, P, P, 1 << 40), lambda: K.kv_pages_compact_scratch_bytes(t))


@pytest.mark.parametrize("bad", BAD_PAGES + BAD_MEMORY + [dict(n_pages=5), dict(page_tokens=32), dict(n_kv=65535, page_tokens=4096)],
                         ids=str)
def test_bad_layers_are_refused(bad):
    """The second layer of two is bad, or differs from the first."""
    K, t, L = kernels(), tables(), layers(pages(), pages(**bad))
    refused(lambda: K.kv_pages_copy(L, P, P, 1), lambda: K.kv_pages_fork(L, t, 1, P, P, P, P, P, 1 << 20),
            lambda: K.kv_pages_compact(L, t, P, P, P, 1 << 40))


def test_pool_refusals():
    K, t, L = kernels(), tables(), layers(pages())
    need, most = K.kv_pages_compact_scratch_bytes(t), layers(*[pages()] * 513)
    assert need >= 4 * 2 * 4 and K.kv_pages_fork_scratch_bytes(3) == 24 and K.kv_pages_fork_scratch_bytes(0) == 0
    refused(lambda: K.kv_pages_copy(L, None, P, 1), lambda: K.kv_pages_copy(L, P, P + 2, 1), lambda: K.kv_pages_copy(L, P, P, 0),
            lambda: K.kv_pages_copy(L, P, P, (1 << 24) + 1), lambda: K.kv_pages_copy(most, P, P, 1),
            lambda: K.kv_pages_free(t, 0), lambda: K.kv_pages_free(t, 4), lambda: K.kv_pages_free(t, 65536, seqs=P),
            lambda: K.kv_pages_free(t, 1, keep=-1), lambda: K.kv_pages_free(t, 1, end=P, behind=-1),
            lambda: K.kv_pages_free(t, 1, end=P + 1), lambda: K.kv_pages_free(t, 1, seqs=P + 2),
            lambda: K.kv_pages_reserve(t, 1, None, 1, P), lambda: K.kv_pages_reserve(t, 1, P, 0, P),
            lambda: K.kv_pages_reserve(t, 4, P, 1, P), lambda: K.kv_pages_reserve(t, 1, P, 1, P + 2),
            lambda: K.kv_pages_reserve(tables(max_pages=1 << 12), 65535, P, 1 << 30, P, seqs=P),
            lambda: K.kv_pages_fork(L, t, 1, None, P, P, P, P, 8), lambda: K.kv_pages_fork(L, t, 1, P, P, P, P, P, 7),
            lambda: K.kv_pages_fork(L, t, 1, P, P, P, P, P + 4, 8), lambda: K.kv_pages_fork(L, t, 1, P, P, P, P, None, 8),
            lambda: K.kv_pages_fork(L, t, 0, P, P, P, P, P, 8), lambda: K.kv_pages_fork(L, t, 1, P, P, P + 2, P, P, 8),
            lambda: K.kv_pages_compact(L, t, None, P, P, need), lambda: K.kv_pages_compact(L, t, P, None, P, need),
            lambda: K.kv_pages_compact(L, t, P, P, P, need - 1), lambda: K.kv_pages_compact(L, t, P, P, P + 8, need))
    lib, ref = K.lib, ctypes.byref
    assert lib.vte_kv_pages_copy(None, 1, P, P, 1, None) == -1 and lib.vte_kv_pages_copy(L, 0, P, P, 1, None) == -1
    assert lib.vte_kv_pages_free(None, 1, None, 0, None, 0, None) == -1
    assert lib.vte_qk_norm_rope(None, 1, 128, 1, P, P, P, 1, 0, None, None, 0, 0, None) == -1
    assert lib.vte_qk_norm_rope(ref(form()), 2, 128, 1, P, P, P, 1, 0, None, None, 0, 0, None) == -1


# ---------------------------------------------------------------------------- frequencies
def test_frequencies_without_scaling():
    f, a = rope_frequencies(8, 10000.0)
    assert a == 1.0 and np.allclose(f, [1, 0.1, 0.01, 0.001], rtol=1e-15, atol=0)


def test_scaled_frequencies():
    f, _ = rope_frequencies(64, 1e4)
    assert np.allclose(rope_frequencies(64, 1e4, "linear", 4)[0], f / 4, rtol=1e-15, atol=0)
    g, a = rope_frequencies(64, 1e4, "base", 4)
    assert a == 1 and g[0] == 1 and np.isclose(g[-1], f[-1] / 4, rtol=1e-12) and (np.diff(g) < 0).all()
    turns = 4096 * f / (2 * np.pi)
    for kind in ("turns", "yarn"):
        g, a = rope_frequencies(64, 1e4, kind, 8, 4096)
        assert np.allclose(g[turns > 40], f[turns > 40], rtol=1e-15, atol=0) and (g <= f).all() and (g >= f / 8 * (1 - 1e-15)).all()
        assert np.allclose(g[turns < 0.8], f[turns < 0.8] / 8, rtol=1e-12, atol=0)
        assert np.isclose(a, 1.0 if kind == "turns" else 0.1 * np.log(8) + 1)
        assert rope_frequencies(64, 1e4, kind, 8, 4096, amplitude=2.5)[1] == 2.5
    assert np.array_equal(rope_frequencies(64, 1e4, "yarn", 1, 4096)[0], f)


@pytest.mark.parametrize("bad", [(0, 1e4), (7, 1e4), (8, 0.0), (8, 1e4, "linear", 0.0), (8, 1e4, "other"), (2, 1e4, "base", 2.0),
                                 (8, 1e4, "yarn", 2.0), (8, 1e4, "turns", 2.0, 4096, 1.0, 2.0), (8, 0.5, "yarn", 2.0, 4096)], ids=str)
def test_bad_frequencies_are_refused(bad):
    with pytest.raises(ValueError):
        rope_frequencies(*bad)


# ---------------------------------------------------------------------------- the oracles
def test_head_form_closed_form():
    x = np.array([[[3.0, 0.0, 4.0, 0.0]]])
    y, _ = olc.head_form(x, [1], weight=[1, 1, 2, 1], eps=1e-30)
    assert np.allclose(y, [[[1.2, 0, 3.2, 0]]])
    y, _ = olc.head_form(x, [1], freq=[np.pi / 2, 0.0], amplitude=2)     # (3, 4) -> (-4, 3), (0, 0)
    assert np.allclose(y, [[[-8, 0, 6, 0]]])
    y, _ = olc.head_form(x, [1], freq=[np.pi / 2, np.pi], interleaved=True)
    assert np.allclose(y, [[[0, 3, -4, 0]]])
    y, _ = olc.head_form(x, [1], freq=[np.pi], rotary_dim=2)
    assert np.allclose(y, [[[-3, 0, 4, 0]]])


@pytest.mark.parametrize("pos,window,sinks,want", [(5, 1, 0, [5]), (5, 2, 1, [0, 4, 5]), (0, 3, 4, [0]), (2, 3, 0, [0, 1, 2]),
                                                   (9, 2, 9, [*range(8)]), (6, 10, 0, [*range(7)])])
def test_what_a_row_sees(pos, window, sinks, want):
    assert np.nonzero(olc.sees(pos, 8, window, sinks))[0].tolist() == want


def test_pool_oracle_counts_users():
    p = olc.Pool([[2, 0, -1], [-1, -1, -1], [-1, -1, -1]], [1, 0, 1, 0, 0], 16, "abcde")
    assert p.fork([0, 0], [1, 2], [20, 16]) == 0
    assert p.table.tolist() == [[2, 0, -1], [2, 1, -1], [2, -1, -1]] and p.refs.tolist() == [1, 1, 3, 0, 0]
    assert p.content == list("aacde")
    assert p.reserve([0, 1, 2], [30, 30, 16], 20) == 2
    assert p.table.tolist() == [[2, 0, 3], [2, 1, 4], [2, -1, -1]] and p.refs.tolist() == [1, 1, 3, 1, 1]
    p.free([0], keep=1, end=[40], behind=0)
    assert p.table[0].tolist() == [2, -1, 3] and p.refs.tolist() == [0, 1, 3, 1, 1]
    p.free([1])
    where, used = p.compact()
    assert used == 2 and where.tolist() == [-1, -1, 0, 1, -1] and p.table.tolist() == [[0, -1, 1], [-1] * 3, [0, -1, -1]]
    assert p.content[:2] == ["c", "d"] and p.refs.tolist() == [2, 1, 0, 0, 0]


def test_pool_oracle_leaves_begun_entries():
    p = olc.Pool([[-1, 0, -1], [-1, -1, -1]], [1, 0, 0, 0], 16, "abcd")
    assert p.reserve([0, 1, 1], [20, 7, 16], 20, follow=True) == 1
    assert p.table.tolist() == [[-1, 0, 1], [-1, 2, 3]] and p.refs.tolist() == [1, 1, 1, 1]
    assert p.reserve([1], [15], 1, follow=True) == 1 and p.reserve([0], [0], 16, follow=True) == 1


# ---------------------------------------------------------------------------- room for tokens that follow others
@pytest.mark.parametrize("bad", BAD_TABLES, ids=str)
def test_extend_refuses_bad_tables(bad):
    refused(lambda: kernels().kv_pages_extend(tables(**bad), 1, P, 1, P))


def test_extend_refusals():
    K, t = kernels(), tables()
    refused(lambda: K.kv_pages_extend(t, 1, None, 1, P), lambda: K.kv_pages_extend(t, 1, P, 0, P),
            lambda: K.kv_pages_extend(t, 4, P, 1, P), lambda: K.kv_pages_extend(t, 0, P, 1, P),
            lambda: K.kv_pages_extend(t, 1, P, 1, P + 2), lambda: K.kv_pages_extend(t, 1, P + 1, 1, P),
            lambda: K.kv_pages_extend(t, 1, P, 1, P, seqs=P + 2), lambda: K.kv_pages_extend(t, 1, P, 1, P, stop=P + 3),
            lambda: K.kv_pages_extend(tables(max_pages=1 << 12), 65535, P, 1 << 30, P, seqs=P))
    assert K.lib.vte_kv_pages_extend(None, 1, None, P, None, 1, P, None) == -1
