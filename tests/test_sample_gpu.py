"""The device draw against the sorted row in extended precision: the same token, always."""
import numpy as np
import pytest

from oracle import sampling as osm
from tests._dev import down, empty, up

pytestmark = pytest.mark.gpu


def draw(hip, K, logits, temperature=None, top_k=None, top_p=None, min_p=None, u=None):
    R, V = logits.shape
    f = lambda x, t: None if x is None else up(hip, np.broadcast_to(np.asarray(x, t), (R,)))
    tok = up(hip, np.full(R, -7, np.int32))
    need = K.sample_scratch_bytes(R)
    scratch = up(hip, np.full(need, 0xFF, np.uint8))  # nothing relies on what scratch held
    K.sample(up(hip, np.asarray(logits, np.float32)), R, V, tok, scratch, temperature=f(temperature, np.float32),
             top_k=f(top_k, np.int32), top_p=f(top_p, np.float32), min_p=f(min_p, np.float32), u=f(u, np.float64),
             stream=hip.stream)
    return down(tok)


def check(hip, K, logits, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.5):
    """Every row's token; one whose u (or border) lies within 2^-44 * vocab of another token could be either."""
    R, V = logits.shape
    got = draw(hip, K, logits, temperature, top_k, top_p, min_p, u)
    row = lambda x, t: np.broadcast_to(np.asarray(x, t), (R,))
    s = [row(temperature, np.float32), row(top_k, np.int32), row(top_p, np.float32), row(min_p, np.float32),
         row(u, np.float64)]
    sure = 0
    for r in range(R):
        want, near = osm.sample(logits[r], float(s[0][r]), int(s[1][r]), float(s[2][r]), float(s[3][r]), float(s[4][r]))
        assert got[r] == want or near < V * 2.0 ** -44, (r, got[r], want, near, [x[r] for x in s])
        sure += near >= V * 2.0 ** -44
    return sure


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 1000, 4096, 4097, 32003, 151936, 262144])
def test_settings(hip, K, vocab):
    """Rows of one call with all settings apart: greedy, top-k below and above the vocabulary, top-p, min-p."""
    rng = np.random.default_rng(vocab)
    R = 24 if vocab < 50000 else 8
    x = (2.5 * rng.standard_normal((R, vocab))).astype(np.float32)
    x[::2, rng.integers(0, vocab, 5)] += 12
    for _ in range(3):
        sure = check(hip, K, x, rng.choice([0.0, 0.3, 0.7, 1.0, 1.5, -1.0], R), rng.choice([0, 1, 2, 40, 500, 10 ** 6, -3], R),
                     rng.choice([0.0, 0.1, 0.5, 0.9, 0.95, 1.0, 2.0], R), rng.choice([0.0, 0.02, 0.1, 1.0, 1.5], R),
                     rng.random(R))
        assert sure >= R - 1


@pytest.mark.parametrize("sigma", [0.0, 0.01, 1.0, 4.0, 30.0])
@pytest.mark.parametrize("top_k,top_p", [(0, 1.0), (0, 0.95), (40, 0.9), (5000, 0.99), (0, 0.999999)])
def test_spreads(hip, K, sigma, top_k, top_p):
    """From equal logits (every entry tied) to one that stands alone."""
    rng = np.random.default_rng(int(sigma * 100) + top_k)
    x = (sigma * rng.standard_normal((5, 20011))).astype(np.float32)
    check(hip, K, x, 1.0, top_k, top_p, 0.0, [0.0, 0.25, 0.5, 0.9, 1 - 2.0 ** -53])


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 128, 129, 512, 513, 1024, 1025, 8191, 8193, 20000])
@pytest.mark.parametrize("spread", [0.0, 0.02, 0.3])
def test_entries_in_question(hip, K, n, spread):
    """The filters and the draw end among n entries of one bin or a few, the rest of the row far below."""
    rng = np.random.default_rng(n)
    x = (-25 - rng.random((6, 40000))).astype(np.float32)
    for row in x:
        row[rng.permutation(40000)[:n]] = 3 + spread * rng.random(n)
    check(hip, K, x, top_k=np.array([0, n // 2 + 1, n, 0, 0, n // 3 + 1]), top_p=np.array([0.5, 1.0, 0.9, 0.3, 1.0, 0.7]),
          min_p=np.array([0, 0, 0, 0.9, 0.8, 0.995]), u=rng.random(6))


def test_more_rows_than_compute_units(hip, K):
    rng = np.random.default_rng(22)
    check(hip, K, (2 * rng.standard_normal((700, 301))).astype(np.float32), rng.choice([0.0, 0.5, 1.0, 2.0], 700),
          rng.choice([0, 5, 100], 700), rng.choice([0.5, 0.95, 1.0], 700), rng.choice([0.0, 0.05], 700), rng.random(700))


def test_ties_go_to_the_lowest_index(hip, K):
    """Levels of equal logits: the order inside a level is the index's, at top-k and top-p borders too."""
    rng = np.random.default_rng(3)
    x = rng.integers(-3, 4, (12, 3001)).astype(np.float32)
    for top_k, top_p in ((0, 1.0), (7, 1.0), (700, 1.0), (0, 0.3), (1000, 0.7)):
        check(hip, K, x, 1.0, top_k, top_p, 0.0, (np.arange(12) + 0.37) / 12)
    z = np.zeros((1, 1000), np.float32)
    z[0, ::2] = -0.0  # equal to 0
    assert draw(hip, K, z, 1.0, 10, u=0.999)[0] == 9 and draw(hip, K, z, 0.0, u=0.5)[0] == 0


def test_not_finite_logits(hip, K):
    inf, nan = np.inf, np.nan
    x = np.full((6, 300), -1.0, np.float32)
    x[0, 5], x[0, 6] = nan, 3
    x[1] = -inf
    x[2] = nan
    x[3, [7, 9]] = inf
    x[4] = -inf
    x[4, 250] = -1e30
    x[5, :299] = nan
    got = draw(hip, K, x, 1.0, u=[0.9, 0.5, 0.5, 0.6, 0.99, 0.99])
    assert list(got[1:]) == [-1, -1, 9, 250, 299]
    assert got[0] == osm.sample(x[0], u=0.9)[0]
    assert list(draw(hip, K, x, 0.0, u=0.5)) == [6, -1, -1, 7, 250, 299]
    assert list(draw(hip, K, x, np.nan, u=0.5)) == [6, -1, -1, 7, 250, 299]


def test_uniforms_at_and_outside_the_ends(hip, K):
    """u <= 0 and NaN: the first of the kept; u >= 1: the last one with weight."""
    x = np.log(np.array([[2, 4, 1, 1, 0]] * 6, np.float32) + 1e-38)
    got = draw(hip, K, x, 1.0, top_k=3, u=[0.0, -1.0, np.nan, 1.0, 7.0, np.inf])
    assert list(got) == [1, 1, 1, 2, 2, 2]


@pytest.mark.parametrize("temperature", [1e-30, 1e-3, 50.0, 1e30, np.inf])
def test_extreme_temperatures(hip, K, temperature):
    rng = np.random.default_rng(11)
    x = (3 * rng.standard_normal((8, 5000))).astype(np.float32)
    x[:, 77] = -np.inf
    check(hip, K, x, temperature, [0, 0, 3, 40, 0, 0, 5, 0], [1, 0.5, 1, 0.9, 0.99, 1, 0.5, 1], 0.0, rng.random(8))


def halfway(T, count):
    """Values x > 0 whose 32 x / T (the factor rounded to fp64) rounds to N + 1/2 in fp64, N even, and lies above it."""
    from fractions import Fraction
    T = np.float32(T)
    s = np.float64(32.0) / np.float64(T)
    x = np.random.default_rng(0).uniform(1, 40, 400000).astype(np.float32)
    y = x.astype(np.float64) * s
    tie = x[(y - np.floor(y) == 0.5) & (np.floor(y) % 2 == 0)]
    return [v for v in tie if Fraction(float(v)) * Fraction(float(s)) > Fraction(float(np.float64(v) * s))][:count]


@pytest.mark.parametrize("T", [1e-8, 1e-9, 3e-10])
@pytest.mark.parametrize("rows,vocab", [(8, 300), (172, 20000), (172, 100003)])
def test_largest_entry_halfway_between_two_bins(hip, K, T, rows, vocab):
    """The largest entry is in the first bin of its scale however its place there is rounded: it alone has weight, or
    shares it with its equals, early and late in the row."""
    values = halfway(T, 8)
    assert values
    rng = np.random.default_rng(int(1 / T))
    x = rng.uniform(-5, 0.9, (rows, vocab)).astype(np.float32)
    at = rng.integers(0, vocab, (rows, 2))
    for r in range(rows):
        x[r, at[r]] = values[r % len(values)]
    u = rng.random(rows)
    got = draw(hip, K, x, np.float32(T), top_p=0.9, min_p=np.where(np.arange(rows) % 2, 0.5, 0.0), u=u)
    # (top-p keeps both: the mass before the second, 1/2, is below 0.9)
    assert list(got) == [int(np.sort(at[r])[int(u[r] * 2)]) for r in range(rows)]


def test_no_settings_is_the_plain_draw(hip, K):
    rng = np.random.default_rng(12)
    x = rng.standard_normal((4, 999)).astype(np.float32)
    u = rng.random(4)
    got = draw(hip, K, x, u=u)
    assert [osm.sample(x[r], u=u[r])[0] for r in range(4)] == list(got)


def test_frequencies(hip, K):
    """4096 evenly spread uniforms fall on the tokens in their proportions, one apart at most."""
    p = np.array([0.4, 0.3, 0.2, 0.1])
    x = np.broadcast_to(np.log(p).astype(np.float32), (4096, 4))
    got = draw(hip, K, np.ascontiguousarray(x), u=(np.arange(4096) + 0.5) / 4096)
    assert (np.abs(np.bincount(got, minlength=4) - 4096 * p) <= 1).all()


@pytest.mark.parametrize("vocab", [100003, 100004])
def test_long_parts_of_many_rows(hip, K, vocab):
    """172 rows: two parts each, longer than what stays in registers; a much larger entry late in a part, parts of
    nothing but -Inf, an infinite temperature."""
    rng = np.random.default_rng(vocab)
    x = (2 * rng.standard_normal((172, vocab))).astype(np.float32)
    x[1, 49000] = x[2, 99999] = 60
    x[3, :50000] = x[4, 49000:] = -np.inf
    x[5, 40000:] += 200
    x[6, 48000:49000] = np.nan
    x[7, 49999] = np.inf
    T = rng.choice([0.2, 0.7, 1.0, 1.5], 172)
    T[8], T[9] = np.inf, 0
    check(hip, K, x, T, rng.choice([0, 0, 40, 3000], 172), rng.choice([1.0, 0.95, 0.5], 172),
          rng.choice([0.0, 0.0, 0.05], 172), rng.random(172))


@pytest.mark.parametrize("most,rows", [(33, 32), (52, 51), (129, 128), (86, 85), (256, 1)])
def test_scratch_of_a_larger_batch(hip, K, most, rows):
    """Draws of fewer rows in memory sized for more: what lies behind it stays as it was.  (The rows' scratch is what the
    largest vocabulary takes; guards are 2 MiB.)"""
    rng = np.random.default_rng(most)
    V, need, guard = 262144, K.sample_scratch_bytes(most), 2 << 20
    scratch = up(hip, np.full(need + guard, 0xA5, np.uint8))
    x = (2 * rng.standard_normal((rows, V))).astype(np.float32)
    tok, u = empty(hip, rows, np.int32), rng.random(rows)
    K.sample(up(hip, x), rows, V, tok, scratch, top_k=up(hip, np.full(rows, 40, np.int32)), u=up(hip, u), stream=hip.stream,
             scratch_bytes=need)
    got = down(tok)
    assert (down(scratch)[need:] == 0xA5).all()
    for r in range(0, rows, 9):
        want, near = osm.sample(x[r], 1.0, 40, u=u[r])
        assert got[r] == want or near < V * 2.0 ** -44


# ---------------------------------------------------------------------------- in the decode step
@pytest.fixture(scope="module")
def tiny():
    from vte_amd.core.model_config import TINY
    from vte_amd.core.weights import SyntheticQwen2
    return SyntheticQwen2(TINY, seed=3)


@pytest.mark.parametrize("B", [1, 3])
def test_generate_sampled_matches_host_loop(hip, K, tiny, B):
    """The draws of the captured loop are those of a loop that reads each step's logits, for the settings of each
    sequence; a second call with other settings replays the same graph; temperature 0 is generate_greedy."""
    from vte_amd.core.hip_graph_executor import HIPGraphExecutor
    ex = HIPGraphExecutor(hip, tiny, batch_size=B, max_seq=256, top_k=40)
    rng = np.random.default_rng(B)
    try:
        toks0, pos0 = [5 + 7 * b for b in range(B)], [60 + 17 * b for b in range(B)]
        for n, T, k, p, m in ((12, [0.7, 1.5, 0.0][:B], 0, 0.95, 0.0), (7, 1.0, [40, 0, 5][:B], 1.0, [0.0, 0.1, 0.0][:B])):
            u = rng.random((n, B))
            ex.fill_kv_prefix(seed=12)
            host, toks, pos = [], list(toks0), list(pos0)
            row = lambda v, b: v[b] if isinstance(v, list) else v
            for i in range(n):
                ex.execute_decode_batch(toks, pos)
                x = ex.read_logits()
                toks = [osm.sample(x[b], float(np.float32(row(T, b))), row(k, b), float(np.float32(row(p, b))),
                                   float(np.float32(row(m, b))), u[i, b])[0] for b in range(B)]
                pos = [q + 1 for q in pos]
                host.append(toks)
            ex.fill_kv_prefix(seed=12)
            assert np.array_equal(ex.generate_sampled(toks0, pos0, n, u, T, k, p, m), np.array(host))
        ex.fill_kv_prefix(seed=12)
        greedy = ex.generate_greedy(toks0, pos0, 6)
        ex.fill_kv_prefix(seed=12)
        assert np.array_equal(ex.generate_sampled(toks0, pos0, 6, np.zeros((6, B)), temperature=0.0), greedy)
        from vte_amd.bridge.hip_runtime import HIPSafetyError
        for bad in (lambda: ex.generate_sampled(toks0, pos0, 0, np.zeros((0, B))),
                    lambda: ex.generate_sampled(toks0, [255] * B, 2, np.zeros((2, B))),
                    lambda: ex.generate_sampled(toks0, pos0, 2, np.zeros((3, B))),
                    lambda: ex.generate_sampled(toks0, pos0, 2, np.ones((2, B))),
                    lambda: ex.generate_sampled(toks0, pos0, 2, np.full((2, B), np.nan))):
            with pytest.raises(HIPSafetyError):
                bad()
    finally:
        ex.close()


def test_advance_keeps_a_row_without_a_draw_inside_the_vocabulary(hip, K):
    tok, off, hist, step = (up(hip, np.array(a, np.int32)) for a in ([4, 4], [7, 9], [0] * 4, [0]))
    K.greedy_advance(up(hip, np.array([-1, 12], np.int32)), 1, 2, tok, off, 9, hist, 2, step, stream=hip.stream)
    assert list(down(tok)) == [0, 12] and list(down(off)) == [8, 9] and list(down(hist)) == [-1, 12, 0, 0]


def test_captured_draws(hip, K):
    """Replays of a captured draw see the logits, settings and uniforms staged before each, with eager draws of another
    size (and scratch of their own) in between."""
    rng = np.random.default_rng(21)
    R, V = 5, 50001
    need = K.sample_scratch_bytes(R)
    x, u = empty(hip, (R, V), np.float32), empty(hip, R, np.float64)
    T, k, tok, scratch = empty(hip, R, np.float32), empty(hip, R, np.int32), empty(hip, R, np.int32), empty(hip, need, np.uint8)
    hip.stream_synchronize()
    hip.stream_begin_capture()
    K.sample(x, R, V, tok, scratch, temperature=T, top_k=k, u=u, stream=hip.stream)
    g = hip.stream_end_capture()
    ge = hip.graph_instantiate(g)
    try:
        for i in range(5):
            logits = (rng.choice([0.5, 2.5]) * rng.standard_normal((R, V))).astype(np.float32)
            st = rng.choice([0.0, 0.8, 1.2], R).astype(np.float32), rng.choice([0, 3, 400], R).astype(np.int32), rng.random(R)
            x.upload(logits), T.upload(st[0]), k.upload(st[1]), u.upload(st[2])
            hip.graph_launch(ge)
            hip.synchronize()
            want = [osm.sample(logits[r], float(st[0][r]), int(st[1][r]), u=float(st[2][r])) for r in range(R)]
            assert all(a == b or near < V * 2.0 ** -44 for a, (b, near) in zip(down(tok), want))
            check(hip, K, (3 * rng.standard_normal((2, 777))).astype(np.float32), 1.0, 0, 0.9, 0.0, rng.random(2))
    finally:
        hip.graph_exec_destroy(ge)
        hip.graph_destroy(g)
