"""Attention over the paged cache, the cache's write with rotary positions, rotary positions and the norms around a block, against
their formulas in 64 bits (attention_ref.py, which derives the tolerances)."""
import ctypes

import numpy as np
import pytest

from attention_ref import EPS, Pool, attention, bf16_bits, bf16_value, norm_residual, turned

pytestmark = pytest.mark.gpu


def _attend(hip, pool, q, heads, causal=True, window=0, scale=None, max_new=None, max_length=None):
    cache, batch = pool.on(hip, max_new, max_length)
    O = hip.full((len(q), q.shape[1]), -7.0)
    hip.paged_attention(hip.array(q), O, cache, batch, scale=scale, causal=causal, window=window)
    return O.numpy()


def _near(got, want, tol, what=""):
    off = np.abs(got - want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    worst = np.nanmax(np.where(tol > 0, off / np.where(tol > 0, tol, 1), off * 1e30), initial=0.0)
    assert worst <= 1.0, (what, worst)


def _check(hip, rng, news, lengths, heads, kv_heads, dim, page, dtype, causal, window, **more):
    pool = Pool(rng, news, lengths, kv_heads, dim, page, dtype)
    q = rng.standard_normal((pool.rows, heads * dim), dtype=np.float32)
    want, tol = attention(q, pool, heads, dim ** -0.5, causal, window)
    got = _attend(hip, pool, q, heads, causal, window, **more)
    _near(got, want, tol)
    # as exact as the same formula in fp32 arithmetic, over all outputs
    plain, _ = attention(q, pool, heads, dim ** -0.5, causal, window, np.float32)
    norm = np.linalg.norm(want)
    if norm > 0:
        assert np.linalg.norm(got - want) <= 4 * np.linalg.norm(plain - want) + 8 * EPS * norm
    return pool, q, got


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 96, 128, 192, 256])
def test_attention_of_ragged_sequences(hip, dtype, dim):
    """Single tokens, chunks, a sequence with no new token, one of length 1, pages that end inside a step."""
    rng = np.random.default_rng(dim)
    _check(hip, rng, [1, 5, 0, 1, 33, 2], [70, 5, 40, 1, 100, 17], 4, 2, dim, 16, dtype, True, 0)
    _check(hip, rng, [3, 17], [64, 33], 3, 3, dim, 32, dtype, False, 0)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (2, 1), (8, 1), (6, 2), (40, 8), (33, 1), (64, 1)])
def test_attention_heads(hip, dtype, heads, kv_heads):
    rng = np.random.default_rng(heads)
    _check(hip, rng, [1, 4, 9], [50, 4, 31], heads, kv_heads, 64, 16, dtype, True, 0)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("page", [16, 64, 128, 1024])
@pytest.mark.parametrize("length", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257])
def test_attention_lengths(hip, dtype, page, length):
    rng = np.random.default_rng(length)
    for new in sorted({1, min(length, 7), length}):
        _check(hip, rng, [new], [length], 2, 1, 64, page, dtype, True, 0)
        _check(hip, rng, [new], [length], 2, 1, 64, page, dtype, False, 0)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 64, 100, 5000])
def test_attention_windows(hip, dtype, causal, window):
    rng = np.random.default_rng(window)
    _check(hip, rng, [1, 40, 70], [300, 200, 70], 4, 2, 64, 32, dtype, causal, window)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_divided_lengths(hip, dtype, dim):
    """Few rows over long sequences: the length is divided and joined; short ones in the same call."""
    rng = np.random.default_rng(3)
    _check(hip, rng, [1, 1, 2], [5000, 3, 2077], 4, 1, dim, 64, dtype, True, 0)
    _check(hip, rng, [1], [3001], 8, 8, dim, 128, dtype, True, 1000)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim, heads, kv_heads", [(64, 4, 4), (128, 8, 2), (80, 3, 1), (256, 2, 1)])
def test_attention_of_long_chunks(hip, dtype, dim, heads, kv_heads):
    """Many rows of a sequence: 150 new tokens behind 300 others, and a whole sequence at once."""
    rng = np.random.default_rng(dim)
    _check(hip, rng, [150, 130], [450, 130], heads, kv_heads, dim, 32, dtype, True, 0)
    _check(hip, rng, [131], [300], heads, kv_heads, dim, 64, dtype, False, 0)
    _check(hip, rng, [200], [333], heads, kv_heads, dim, 64, dtype, True, 50)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_in_many_parts(hip, dtype, dim):
    """One key head and one sequence of 40000 tokens: more parts than the last workgroup joins; and chunks in parts over it."""
    rng = np.random.default_rng(dim)
    _check(hip, rng, [1], [40000], 3, 1, dim, 256, dtype, True, 0)
    _check(hip, rng, [40], [3000], 1, 1, dim, 64, dtype, True, 0)
    _check(hip, rng, [20, 3], [3000, 700], 2, 1, dim, 64, dtype, False, 0)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_attention_of_chunks_of_all_lengths(hip, dtype):
    """Long and short chunks, and sequences without new tokens, in one call: tiles that are not there."""
    rng = np.random.default_rng(23)
    _check(hip, rng, [200, 3, 0, 5, 60, 1, 129], [210, 300, 40, 5, 333, 1, 200], 4, 2, 64, 32, dtype, True, 0)
    _check(hip, rng, [1, 140, 2], [90, 200, 400], 2, 2, 96, 32, dtype, False, 70)


def test_attention_beyond_the_bounds(hip):
    """max_new and max_length too small size the launch too small, never the result."""
    rng = np.random.default_rng(0)
    for dtype in ("float32", "bfloat16"):
        _check(hip, rng, [200, 3], [250, 300], 4, 2, 64, 32, dtype, True, 0, max_new=1, max_length=1)
        _check(hip, rng, [3, 4], [250, 30], 4, 2, 64, 32, dtype, True, 0, max_new=900, max_length=100000)
        # tiles of many rows beyond those that the launch has, undivided beside divided ones
        _check(hip, rng, [300, 10], [1500, 700], 4, 2, 64, 32, dtype, True, 0, max_new=150)
        _check(hip, rng, [300, 300], [900, 300], 2, 2, 80, 32, dtype, False, 100, max_new=40)
        # the same of few rows, in parts that the last workgroup or a launch joins
        _check(hip, rng, [50, 1], [1100, 600], 2, 2, 64, 32, dtype, True, 0, max_new=2)
        _check(hip, rng, [20], [41000], 1, 1, 64, 256, dtype, True, 0, max_new=1)


def test_attention_large_scores(hip):
    """Scores of hundreds: one token takes nearly all the weight, the others' exponentials are zeros."""
    rng = np.random.default_rng(1)
    pool = Pool(rng, [9], [90], 2, 64, 16, "float32")
    q = 40.0 * rng.standard_normal((9, 4 * 64), dtype=np.float32)
    want, tol = attention(q, pool, 4, 0.5, True, 0)
    _near(_attend(hip, pool, q, 4, scale=0.5), want, tol)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new", [2, 130])
def test_attention_values_and_keys_of_all_sizes(hip, dtype, new):
    """Values and keys of 1e-30 and 1e30, and blocks of tokens whose values differ by a factor of 1e25: the largest values carry the result,
    the sums of the weights are those of all tokens."""
    rng = np.random.default_rng(21)
    length = new + 150
    for size in (1e-30, 1e-10, 1.0, 1e30):
        for what in ("k", "v", "both"):
            pool = Pool(rng, [new], [length], 1, 64, 16, dtype)
            j = np.arange(length)
            for name in ("k", "v"):
                if what in (name, "both"):
                    pool.put(0, j, name, pool.get(0, j, name) * np.float32(size))
            q = rng.standard_normal((new, 2 * 64), dtype=np.float32)
            scale = 0.125 / (size if what != "v" and size > 1 else 1.0)
            want, tol = attention(q, pool, 2, scale, True, 0)
            got = _attend(hip, pool, q, 2, scale=scale)
            _near(got, want, tol, (size, what))
            assert np.linalg.norm((got - want) / size ** (what != "k")) <= 32 * EPS * np.linalg.norm(want / size ** (what != "k"))
    for order in ((1e-15, 1e10), (1e10, 1e-15), (1e-15, 1.0, 0.0, 1e10, 1e-5)):
        pool = Pool(rng, [new], [length], 1, 64, 16, dtype)
        for n, size in enumerate(order):
            j = np.arange(length * n // len(order), length * (n + 1) // len(order))
            pool.put(0, j, "v", pool.get(0, j, "v") * np.float32(size))
        q = rng.standard_normal((new, 2 * 64), dtype=np.float32)
        want, tol = attention(q, pool, 2, 0.125, False, 0)
        _near(_attend(hip, pool, q, 2, causal=False), want, tol, order)
        # the first tokens alone: with a window of the last rows' neighbours none of the large values counts
        want, tol = attention(q, pool, 2, 0.125, True, 20)
        _near(_attend(hip, pool, q, 2, causal=True, window=20), want, tol + 2.0 ** -38 * np.abs(want).max(), order)


def test_attention_negative_and_zero_scale(hip):
    rng = np.random.default_rng(22)
    for dtype in ("float32", "bfloat16"):
        for new in (2, 60):
            pool = Pool(rng, [new], [new + 40], 1, 64, 16, dtype)
            q = rng.standard_normal((new, 2 * 64), dtype=np.float32)
            for scale in (-0.3, 0.0):
                want, _ = attention(q, pool, 2, scale, True, 0)
                tol = attention(q, pool, 2, 0.3, True, 0)[1]
                _near(_attend(hip, pool, q, 2, scale=scale), want, tol)


def test_attention_rows_that_see_nothing_are_zero(hip):
    """Rows before place 0 (a sequence with more rows than tokens) and sequences of no tokens see nothing."""
    rng = np.random.default_rng(2)
    for dtype in ("float32", "bfloat16"):
        for new, length in ((5, 3), (40, 3), (4, 0), (1, 0), (200, 100)):
            for window in (0, 2):
                _, _, got = _check(hip, rng, [new, 1], [length, 50], 4, 2, 64, 16, dtype, True, window)
                assert np.all(got[:max(0, new - length)] == 0.0)
        _, _, got = _check(hip, rng, [3], [0], 4, 2, 64, 16, dtype, False, 0)
        assert np.all(got == 0.0)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new", [7, 150])
def test_attention_nonfinite_numbers_in_hidden_places(hip, dtype, new):
    """Infinities and NaN in keys and values that a row does not see leave it as it is; rows that see them come out as the formula."""
    rng = np.random.default_rng(4)
    length = new + 90
    pool = Pool(rng, [new], [length], 2, 64, 32, dtype)
    q = rng.standard_normal((new, 4 * 64), dtype=np.float32)
    clean, tol = attention(q, pool, 4, 0.125, True, 60)
    places = [3, length - new + 3, length - 2]  # before every window; seen from row 3 on; seen by the last two rows
    pool.put(0, places[:1], "v", np.full((1, 2, 64), np.nan, np.float32))
    pool.put(0, places[:1], "k", np.full((1, 2, 64), np.inf, np.float32))
    x = pool.get(0, places[1:2], "v")
    x[0, 1, 5] = np.inf
    pool.put(0, places[1:2], "v", x)
    x = pool.get(0, places[2:], "k")
    x[0, 0, 3] = np.nan
    pool.put(0, places[2:], "k", x)
    want, _ = attention(q, pool, 4, 0.125, True, 60)
    got = _attend(hip, pool, q, 4, True, 60)
    fine = np.isfinite(want)
    assert fine[:3].all() and not fine[-1, :128].any() and np.isposinf(want[4, 2 * 64 + 5])
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
    assert np.all(np.abs(got[fine] - want[fine]) <= tol[fine])
    assert np.all(clean[:3] == want[:3])


def test_attention_infinite_scores(hip):
    """A key of -inf scores gets no weight; a row whose only scores are -inf, and one with a score of +inf, are NaN, as in the formula."""
    rng = np.random.default_rng(5)
    for dtype in ("float32", "bfloat16"):
        for length, news in ((40, 3), (3000, 1)):
            pool = Pool(rng, [news], [length], 1, 64, 16, dtype)
            q = np.abs(rng.standard_normal((news, 64), dtype=np.float32)) + 0.1
            pool.put(0, [5], "k", np.full((1, 1, 64), -np.inf, np.float32))
            want, tol = attention(q, pool, 1, 0.125, True, 0)
            assert np.isfinite(want).all()
            _near(_attend(hip, pool, q, 1), want, tol)
            pool.put(0, [5], "k", np.full((1, 1, 64), np.inf, np.float32))
            assert np.isnan(_attend(hip, pool, q, 1)).all()
            pool.put(0, np.arange(length), "k", np.full((length, 1, 64), -np.inf, np.float32))
            assert np.isnan(_attend(hip, pool, q, 1)).all()


def test_attention_rows_behind_and_before_the_batch_are_left(hip):
    rng = np.random.default_rng(6)
    for dtype in ("float32", "bfloat16"):
        for length in (20, 4000):
            pool = Pool(rng, [2, 3], [length, 9], 2, 64, 16, dtype)
            q = rng.standard_normal((pool.rows, 2 * 64), dtype=np.float32)
            want, tol = attention(q, pool, 2, 0.125, True, 0)
            pool.offsets = pool.offsets + 4
            wide = np.full((pool.rows + 9, 2 * 64), np.nan, np.float32)
            wide[4:9] = q
            got = _attend(hip, pool, wide, 2)
            assert np.all(got[:4] == -7.0) and np.all(got[9:] == -7.0)
            _near(got[4:9], want, tol)


def test_attention_rows_of_other_distances_and_alignments(hip):
    """Queries as columns of a wider tensor, aligned and not."""
    rng = np.random.default_rng(7)
    pool = Pool(rng, [5, 70], [60, 75], 2, 48, 16, "float32")
    q = rng.standard_normal((pool.rows, 4 * 48), dtype=np.float32)
    want, tol = attention(q, pool, 4, 48 ** -0.5, True, 0)
    cache, batch = pool.on(hip)
    for width, at, o_width, o_at in ((400, 64, 300, 8), (333, 3, 257, 1), (192, 0, 195, 2)):
        wide, out = np.full((pool.rows, width), np.nan, np.float32), hip.full((pool.rows, o_width), -7.0)
        wide[:, at:at + 192] = q
        hip.paged_attention(hip.array(wide).columns(at, at + 192), out.columns(o_at, o_at + 192), cache, batch)
        got = out.numpy()
        _near(got[:, o_at:o_at + 192], want, tol)
        got[:, o_at:o_at + 192] = -7.0
        assert np.all(got == -7.0)


def test_attention_pages_outside_the_pool_make_their_rows_nan(hip):
    """A page number out of range, and a length beyond the table's row, read nothing outside the buffers and leave the other sequences right."""
    rng = np.random.default_rng(8)
    for dtype in ("float32", "bfloat16"):
        for new in (1, 5, 140):
            for wrong in (-1, 10 ** 6):
                pool = Pool(rng, [new, 2, 1], [170, 50, 9], 1, 64, 16, dtype)
                q = rng.standard_normal((pool.rows, 2 * 64), dtype=np.float32)
                want, tol = attention(q, pool, 2, 0.125, False, 0)
                pool.table[0, 4] = wrong
                got = _attend(hip, pool, q, 2, causal=False)
                assert np.isnan(got[:new]).all()
                _near(got[new:], want[new:], tol[new:])
                pool.lengths[1] = 16 * pool.width + 1
                got = _attend(hip, pool, q, 2, causal=False)
                assert np.isnan(got[:new + 2]).all()
                _near(got[new + 2:], want[new + 2:], tol[new + 2:])
                pool.lengths[1] = -3
                assert np.isnan(_attend(hip, pool, q, 2, causal=False)[new:new + 2]).all()


def test_attention_shared_pages(hip):
    """Sequences with a common beginning read the same pages."""
    rng = np.random.default_rng(9)
    pool = Pool(rng, [1, 1, 1], [100, 90, 80], 2, 64, 16, "bfloat16", shared=3)
    for s in range(3):  # (the shared pages hold what the last sequence put there; nothing is NaN)
        for name in ("k", "v"):
            assert np.isfinite(pool.get(s, np.arange(pool.lengths[s]), name)).all()
    q = rng.standard_normal((3, 4 * 64), dtype=np.float32)
    want, tol = attention(q, pool, 4, 0.125, True, 0)
    _near(_attend(hip, pool, q, 4), want, tol)


def test_attention_twice_gives_the_same_bits(hip):
    rng = np.random.default_rng(10)
    pool = Pool(rng, [1, 60], [3000, 100], 2, 128, 64, "bfloat16")
    q = rng.standard_normal((61, 4 * 128), dtype=np.float32)
    a, b = _attend(hip, pool, q, 4), _attend(hip, pool, q, 4)
    assert np.array_equal(a.view(np.uint32), b.view(np.uint32))


def test_attention_pages_past_4_gib_elements(hip):
    """Offsets into a large pool pass 32 bits: a bf16 pool of 2.5 G numbers, the sequence on its last pages."""
    from eddl_amd.attention import PagedBatch, PagedCache
    rng = np.random.default_rng(11)
    page, kv, dim, pages = 256, 8, 128, 9600
    pool = Pool(rng, [3], [300], kv, dim, page, "bfloat16", spare=0, fill=0.0)
    cache = PagedCache(hip, pages, page, kv, dim, "bfloat16")
    assert cache.keys.size > 2 ** 31
    per = page * kv * dim
    table = np.array([[pages - 1, pages - 2]], np.int32)
    for i, p in enumerate(pool.table[0]):
        for t, x in ((cache.keys, pool.k), (cache.values, pool.v)):
            bits = np.ascontiguousarray(bf16_bits(x[p * per:(p + 1) * per]))
            hip._check(hip.lib.eddlhip_memcpy_h2d(hip.dev, t.address + 2 * per * int(table[0, i]), bits.ctypes.data, bits.nbytes))
    q = rng.standard_normal((3, kv * dim), dtype=np.float32)
    want, tol = attention(q, pool, kv, dim ** -0.5, True, 0)
    batch = PagedBatch(hip.array(table, "int32"), hip.array(pool.offsets, "int32"), hip.array(np.array([300]), "int32"), 3, 300)
    O = hip.empty(q.shape)
    hip.paged_attention(hip.array(q), O, cache, batch)
    _near(O.numpy(), want, tol)


# ------------------------------------------------------------------------------------------------- rotary positions
def _plan(dim, rot, axes, pairing, rng):
    from eddl_amd.attention import RotaryPlan
    return RotaryPlan(dim, rng.integers(0, axes, rot // 2), 10000.0 ** -rng.uniform(0, 1, rot // 2), pairing, axes)


@pytest.mark.parametrize("pairing", ["halves", "adjacent"])
@pytest.mark.parametrize("dim, rot, heads", [(8, 8, 1), (64, 64, 3), (64, 32, 5), (80, 40, 2), (128, 128, 16), (256, 256, 2), (256, 8, 1), (64, 0, 2), (328, 248, 2)])
def test_rotary(hip, pairing, dim, rot, heads):
    """One product rounding each, one of their sum, the sine's (4 EPS) and that of its fp32 argument (half a step of a fraction of a turn: 2 pi 2^-26): 8 EPS of |x|."""
    rng = np.random.default_rng(dim + rot)
    for rows, axes in ((1, 1), (37, 2), (5000, 3)):
        plan = _plan(dim, rot, axes, pairing, rng)
        x = rng.standard_normal((rows, heads * dim), dtype=np.float32)
        pos = np.floor(rng.uniform(-1e6, 1e6, (rows, axes))).astype(np.float32)
        if rows == 37:
            pos = rng.uniform(-50, 50, (rows, axes)).astype(np.float32)  # (positions between pixels)
        want = turned(x, pos, heads, dim, plan.axis, plan.freq, pairing == "adjacent")
        X, P = hip.array(x), hip.array(pos)
        Y = hip.empty(x.shape)
        hip.rotary_axes(X, Y, plan, P)
        got = Y.numpy()
        # angles up to 1e6: the fraction of a turn is off by 2^-53 of 1.6e5 turns, 2e-11, nothing beside fp32
        size = np.sqrt(2) * np.abs(x).max()
        assert np.abs(got - want).max() <= 8 * EPS * size
        if rot < dim:
            assert np.array_equal(got.reshape(rows, heads, dim)[:, :, rot:], x.reshape(rows, heads, dim)[:, :, rot:])
        hip.rotary_axes(X, X, plan, P)
        assert np.array_equal(X.numpy(), got)


def test_rotary_of_columns(hip):
    rng = np.random.default_rng(1)
    plan = _plan(16, 16, 2, "halves", rng)
    pos = rng.integers(0, 99, (11, 2)).astype(np.float32)
    for width, at, to in ((100, 32, 4), (99, 33, 5)):
        x = rng.standard_normal((11, width), dtype=np.float32)
        Y = hip.full((11, 90), -7.0)
        hip.rotary_axes(hip.array(x).columns(at, at + 48), Y.columns(to, to + 48), plan, hip.array(pos))
        got = Y.numpy()
        assert np.abs(got[:, to:to + 48] - turned(x[:, at:at + 48], pos, 3, 16, plan.axis, plan.freq, False)).max() <= 8 * EPS * 1.5 * np.abs(x).max()
        got[:, to:to + 48] = -7.0
        assert np.all(got == -7.0)


def test_rotary_back(hip):
    """Negative frequencies undo it, and a rotation is the gradient of its inverse: difference quotients of a weighted sum."""
    from eddl_amd.attention import RotaryPlan
    rng = np.random.default_rng(2)
    plan = _plan(32, 24, 3, "adjacent", rng)
    back = RotaryPlan(32, plan.axis, -plan.freq, "adjacent", 3)
    x, g = rng.standard_normal((7, 64), dtype=np.float32), rng.standard_normal((7, 64), dtype=np.float32)
    pos = hip.array(rng.integers(0, 1000, (7, 3)))
    Y, Z, G = hip.empty((7, 64)), hip.empty((7, 64)), hip.empty((7, 64))
    hip.rotary_axes(hip.array(x), Y, plan, pos)
    hip.rotary_axes(Y, Z, back, pos)
    assert np.abs(Z.numpy() - x).max() <= 16 * EPS * 2 * np.abs(x).max()
    hip.rotary_axes(hip.array(g), G, back, pos)
    base = (Y.numpy().astype(np.float64) * g).sum()
    for i, j in ((0, 0), (3, 33), (6, 31), (2, 23)):
        moved = x.copy()
        moved[i, j] += 1.0
        hip.rotary_axes(hip.array(moved), Y, plan, pos)
        assert abs((Y.numpy().astype(np.float64) * g).sum() - base - G.numpy()[i, j]) <= 448 * 8 * EPS * 4 * 4


# ------------------------------------------------------------------------------------------------- the cache's write
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("dim, rot, heads, kv", [(64, 64, 4, 2), (80, 40, 3, 1), (16, 16, 2, 2), (256, 256, 2, 1), (64, 0, 2, 2)])
@pytest.mark.parametrize("pairing", ["halves", "adjacent"])
def test_append(hip, dtype, page, dim, rot, heads, kv, pairing):
    rng = np.random.default_rng(dim + rot + page)
    news, lengths = [1, 37, 0, 16, 3, 5], [18, 50, 20, 16, 129, 5]
    pool = Pool(rng, news, lengths, kv, dim, page, dtype)
    plan = _plan(dim, rot, 2, pairing, rng) if rot else None
    rows = pool.rows + 3
    qkv = rng.standard_normal((rows, (heads + 2 * kv) * dim), dtype=np.float32)
    pos = rng.integers(0, 5000, (rows, 2)).astype(np.float32)
    cache, batch = pool.on(hip)
    QKV, P = hip.array(qkv), hip.array(pos)
    a, b = heads * dim, (heads + kv) * dim
    Q = hip.full((rows, a), -7.0)
    hip.paged_append(QKV.columns(0, a), QKV.columns(a, b), QKV.columns(b, b + kv * dim), Q, cache, batch, plan, P if rot else None)
    axis, freq = (plan.axis, plan.freq) if rot else (np.zeros(0, int), np.zeros(0))
    want = turned(qkv[:, :b], pos, heads + kv, dim, axis, freq, pairing == "adjacent")
    got = Q.numpy()
    tol = 8 * EPS * 1.5 * np.abs(qkv).max()
    assert np.abs(got[:pool.rows] - want[:pool.rows, :a]).max() <= tol and np.all(got[pool.rows:] == -7.0)
    k, v = pool.read(cache)
    k0, v0 = pool.k.copy(), pool.v.copy()
    step = 0.0 if dtype == "float32" else 2.0 ** -8  # (half a step of bf16, relative)
    for s in range(len(news)):
        rows_s, places = np.arange(pool.offsets[s], pool.offsets[s + 1]), np.arange(lengths[s] - news[s], lengths[s])
        at = pool.index(s, places, "k")
        x = want[rows_s, a:].reshape(-1, kv, dim)
        assert np.all(np.abs(k[at] - x) <= tol + step * (np.abs(x) + tol))
        k0[at] = k[at]
        at = pool.index(s, places, "v")
        x = qkv[rows_s, b:].reshape(-1, kv, dim)
        assert np.array_equal(v[at], x if dtype == "float32" else bf16_value(bf16_bits(x)))
        v0[at] = v[at]
    assert np.array_equal(k, k0, equal_nan=True) and np.array_equal(v, v0, equal_nan=True)  # nothing else was written


def test_append_without_queries_in_place_and_beyond_the_bounds(hip):
    rng = np.random.default_rng(12)
    pool = Pool(rng, [100, 2], [130, 40], 2, 32, 16, "float32")
    k, v, q = (rng.standard_normal((102, 64), dtype=np.float32) for _ in range(3))
    plan, pos = _plan(32, 32, 1, "halves", rng), rng.integers(0, 99, (102, 1)).astype(np.float32)
    cache, batch = pool.on(hip, max_new=1)
    hip.paged_append(None, hip.array(k), hip.array(v), None, cache, batch, plan, hip.array(pos))
    first = pool.read(cache)
    cache2, batch2 = pool.on(hip)
    Q = hip.array(q)
    hip.paged_append(Q, hip.array(k), hip.array(v), Q, cache2, batch2, plan, hip.array(pos))
    second = pool.read(cache2)
    assert all(np.array_equal(x, y, equal_nan=True) for x, y in zip(first, second))
    assert np.abs(Q.numpy() - turned(q, pos, 2, 32, plan.axis, plan.freq, False)).max() <= 8 * EPS * 1.5 * np.abs(q).max()


def test_append_tokens_without_a_place_are_not_written(hip):
    rng = np.random.default_rng(13)
    for dtype in ("float32", "bfloat16"):
        pool = Pool(rng, [20, 5, 3, 2], [12, 70, 30, 16], 1, 32, 16, dtype, fill=-3.0)
        pool.table[1, 4] = 10 ** 6
        pool.lengths[3] = 16 * pool.width + 2
        cache, batch = pool.on(hip)
        x = rng.standard_normal((30, 32), dtype=np.float32)
        hip.paged_append(None, hip.array(x), hip.array(x), None, cache, batch)
        x = x if dtype == "float32" else bf16_value(bf16_bits(x))
        k0, v0 = pool.k.copy(), pool.v.copy()
        for s, rows, places in ((0, np.arange(8, 20), np.arange(12)), (2, np.arange(25, 28), np.arange(27, 30))):
            k0[pool.index(s, places, "k")] = v0[pool.index(s, places, "v")] = x[rows].reshape(-1, 1, 32)
        k, v = pool.read(cache)
        assert np.array_equal(k, k0) and np.array_equal(v, v0)


# ------------------------------------------------------------------------------------------------- norms
@pytest.mark.parametrize("cols", [1, 2, 3, 7, 64, 100, 255, 256, 257, 512, 1000, 1024, 1025, 2048, 4097, 8192, 9000, 16384, 30000, 32768])
@pytest.mark.parametrize("post, pre", [(None, "layer"), ("rms", "rms"), ("layer", None), ("layer", "layer"), (None, None)])
def test_norm_residual(hip, cols, post, pre):
    """Sums of squares are formed in a tree over at most 32 values a thread and ten levels, their relative error stays below 140 EPS, half of it
    in the root; mean, difference, division, weight, bias, gate and sum round once or twice each: 160 EPS.  (Layer norm: the mean's
    error, 140 EPS of the largest value, moves every difference.)"""
    rng = np.random.default_rng(cols)
    for rows, group_rows, mode in ((1, 1, 0), (13, 5, 1), (70, 70, 2)):
        n = lambda *s: rng.standard_normal(s, dtype=np.float32)
        x, r, groups = n(rows, cols) + 0.3, n(rows, cols), -(-rows // group_rows)
        po = (post, 1 + 0.1 * n(cols), 0.1 * n(cols), 1e-5) if post else (None, None, None, 0.0)
        pr = (pre, 1 + 0.1 * n(cols), None if mode else 0.1 * n(cols), 1e-3) if pre else (None, None, None, 0.0)
        gate = (None, n(groups, cols), n(1, cols))[mode]
        mod, shift = (0.2 * n(groups, cols), 0.2 * n(groups, cols)) if mode == 1 else (None, None)
        res = r if mode < 2 else None
        want_s, want_h = norm_residual(x, res, po, pr, gate, 0.7, mod, shift, group_rows)
        d = lambda t: None if t is None else hip.array(t)
        S, H = hip.empty((rows, cols)), hip.empty((rows, cols))
        args = dict(post=(po[0], d(po[1]), d(po[2]), po[3]), pre=(pr[0], d(pr[1]), d(pr[2]), pr[3]), gate=d(gate), residual_scale=0.7, mod=d(mod), shift=d(shift),
                    group_rows=group_rows)
        hip.norm_residual(d(x), d(res), S, H, **args)
        s, h = S.numpy(), H.numpy()
        e = 160 * EPS
        # the sum: a normed value is off by e of its size and e of the mean's share; its gate multiplies that
        top = np.abs(x).max(1, keepdims=True)
        size = np.abs(want_s) + (np.abs(r) if res is not None else 0)
        if post:
            sd = np.sqrt(((x - (x.mean(1, keepdims=True) if post == "layer" else 0)) ** 2).mean(1, keepdims=True, dtype=np.float64) + 1e-5)
            size = size + 2 * (top / sd) * 1.6 * (np.abs(gate).max() if gate is not None else 1)
        tol_s = e * size + 1e-30
        assert np.all(np.abs(s - want_s) <= tol_s)
        # the norm of it, against the norm of the sum that came out
        given = s.astype(np.float64)
        ref_h = norm_residual(s, None, (None, None, None, 0.0), pr, None, 1.0, mod, shift, group_rows)[1]
        size = np.abs(ref_h) + 1.0
        if pre:
            sd = np.sqrt(((given - (given.mean(1, keepdims=True) if pre == "layer" else 0)) ** 2).mean(1, keepdims=True) + 1e-3)
            size = size + 2 * np.abs(given).max(1, keepdims=True) / sd * 3
        assert np.all(np.abs(h - ref_h) <= e * size)
        # the same numbers in place, and with one output only
        X, R = d(x), d(res)
        hip.norm_residual(X, R, R if R is not None else X, H, **args)
        assert np.array_equal((R if R is not None else X).numpy(), s) and np.array_equal(H.numpy(), h)
        X = d(x)
        hip.norm_residual(X, d(res), None, X, **args)
        assert np.array_equal(X.numpy(), h)
        if pre is None and mod is None:
            hip.norm_residual(d(x), d(res), S, None, **dict(args, pre=(None, None, None, 0.0)))
            assert np.array_equal(S.numpy(), s)


def test_norm_of_columns(hip):
    rng = np.random.default_rng(1)
    for width, at, cols in ((200, 64, 100), (99, 33, 50)):
        x = rng.standard_normal((9, width), dtype=np.float32)
        H = hip.full((9, width), -7.0)
        hip.norm_residual(hip.array(x).columns(at, at + cols), None, None, H.columns(4, 4 + cols), pre=("rms", None, None, 1e-6))
        got = H.numpy()
        want = norm_residual(x[:, at:at + cols], None, (None, None, None, 0.0), ("rms", None, None, 1e-6), None, 1.0, None, None, 9)[1]
        assert np.all(np.abs(got[:, 4:4 + cols] - want) <= 160 * EPS * (np.abs(want) + 1))
        got[:, 4:4 + cols] = -7.0
        assert np.all(got == -7.0)


# ------------------------------------------------------------------------------------------------- graphs, streams, a block as it is used
def test_recorded_steps_follow_the_batch(hip):
    """A recorded append and attention, replayed while the lengths grow: every replay equals the eager calls on the same state."""
    from eddl_amd.attention import PagedBatch
    rng = np.random.default_rng(14)
    heads, kv, dim, steps = 4, 2, 64, 6
    for start in (20, 2500):
        pool = Pool(rng, [1, 1], [start + steps, 40 + steps], kv, dim, 16, "bfloat16", fill=0.0)
        (cache, batch), (other, _) = pool.on(hip), pool.on(hip)
        lengths = hip.array(np.array([start, 40]), "int32")
        batch = PagedBatch(batch.table, batch.offsets, lengths, 1, start + steps)
        plan = _plan(dim, dim, 1, "halves", rng)
        QKV, P, T = hip.empty((2, (heads + 2 * kv) * dim)), hip.empty((2, 1)), hip.empty((2, heads * dim))
        O = [hip.empty((2, heads * dim)) for _ in range(2)]

        def step(c, out):
            a, b = heads * dim, (heads + kv) * dim
            hip.paged_append(QKV.columns(0, a), QKV.columns(a, b), QKV.columns(b, b + kv * dim), T, c, batch, plan, P)
            hip.paged_attention(T, out, c, batch)

        QKV.copy_from(np.zeros(QKV.shape))
        P.copy_from(np.zeros((2, 1)))
        for c in (cache, other):  # (the workspace has its size; both caches take the same zeros)
            step(c, O[1])
        graph = hip.record(lambda: step(cache, O[0]))
        for i in range(steps):
            lengths.copy_from(np.array([start + 1 + i, 41 + i]))
            QKV.copy_from(rng.standard_normal(QKV.shape))
            P.copy_from(np.array([[start + i], [40 + i]]))
            graph.launch()
            step(other, O[1])
            hip.synchronize()
            same = np.array_equal(O[0].numpy(), O[1].numpy())
            assert same, i
            assert all(np.array_equal(x.numpy(), y.numpy()) for x, y in ((cache.keys, other.keys), (cache.values, other.values)))
        del graph


def test_graphs_that_share_the_workspace(hip):
    """Two recorded calls whose parts lie in the same workspace, replayed in turn with an eager third between them, several times."""
    rng = np.random.default_rng(24)
    calls = []
    for news, lengths, heads, kv, dim, dtype in (([1, 1], [3000, 700], 4, 2, 128, "bfloat16"), ([1], [40000], 3, 1, 64, "bfloat16"), ([40], [2500], 2, 1, 64, "float32")):
        pool = Pool(rng, news, lengths, kv, dim, 64, dtype)
        cache, batch = pool.on(hip)
        Q = hip.array(rng.standard_normal((pool.rows, heads * dim)))
        O = hip.empty(Q.shape)
        run = lambda Q=Q, O=O, cache=cache, batch=batch: hip.paged_attention(Q, O, cache, batch)
        run()
        calls.append((run, O, O.numpy()))
    for run, _, _ in calls:  # (the workspace has its size)
        run()
    graphs = [hip.record(run) for run, _, _ in calls[:2]]
    for _ in range(4):
        for _, O, _ in calls:
            hip.fill_(O, -7.0)
        graphs[0].launch()
        calls[2][0]()
        graphs[1].launch()
        graphs[0].launch()
        for _, O, want in calls:
            same = np.array_equal(O.numpy(), want)
            assert same
    del graphs


def test_on_a_stream_of_the_callers(hip):
    rng = np.random.default_rng(15)
    pool = Pool(rng, [1], [3000], 1, 64, 64, "float32")
    q = rng.standard_normal((1, 4 * 64), dtype=np.float32)
    want, tol = attention(q, pool, 4, 0.125, True, 0)
    cache, batch = pool.on(hip)
    Q, O = hip.array(q), hip.full(q.shape, 0.0)
    stream = ctypes.c_void_p()
    assert hip.lib.hipStreamCreateWithFlags(ctypes.byref(stream), 1) == 0  # (of the runtime that the library runs on; non-blocking)
    hip.synchronize()
    hip._check(hip.lib.eddlhip_set_stream(hip.dev, stream))
    try:
        hip.paged_attention(Q, O, cache, batch)
        hip.norm_residual(O, None, None, O, pre=("rms", None, None, 1e-6))
        got = O.numpy()
    finally:
        hip._check(hip.lib.eddlhip_set_stream(hip.dev, None))
        hip.lib.hipStreamDestroy(stream)
    ref = want / np.sqrt((want * want).mean() + 1e-6)
    assert np.abs(got - ref).max() <= 8 * tol.max() / np.sqrt((want * want).mean()) + 160 * EPS * np.abs(ref).max()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_block_of_video_frames(hip, dtype):
    """An attention block over frames that arrive one by one: norm, dense layer, rotary positions of time, row and column into the cache,
    attention over all frames so far, dense layer, gate, residual sum and norm - against the whole in 64 bits."""
    from eddl_amd.attention import PagedBatch, PagedCache, RotaryPlan
    rng = np.random.default_rng(16)
    side, frames, videos, heads, kv, dim = 5, 4, 2, 4, 2, 32
    tokens, cols = side * side, heads * dim
    n = lambda *s: rng.standard_normal(s, dtype=np.float32)
    Wqkv, Wo, w1, w2 = n(cols, (heads + 2 * kv) * dim) / np.float32(np.sqrt(cols)), n(cols, cols) / np.float32(np.sqrt(cols)), 1 + 0.1 * n(cols), 1 + 0.1 * n(cols)
    gate = n(videos, cols)
    xs = [n(videos * tokens, cols) for _ in range(frames)]
    plan = RotaryPlan.sections(dim, (4, 6, 6), interleaved=True)
    assert [list(plan.axis).count(a) for a in range(3)] == [4, 6, 6]
    width = -(-frames * tokens // 16)
    cache = PagedCache(hip, videos * width, 16, kv, dim, dtype)
    table = rng.permutation(videos * width).reshape(videos, width)
    offsets, lengths = hip.array(np.arange(videos + 1) * tokens, "int32"), hip.empty((videos,), "int32")
    batch = PagedBatch(hip.array(table, "int32"), offsets, lengths, tokens, frames * tokens)
    d = lambda t: hip.array(t)
    dW, dWo, dw1, dw2, dgate = d(Wqkv), d(Wo), d(w1), d(w2), d(gate)
    H, QKV, Q, A, B = hip.empty((videos * tokens, cols)), hip.empty((videos * tokens, Wqkv.shape[1])), *(hip.empty((videos * tokens, cols)) for _ in range(3))
    past_k, past_v = [], []
    a, b = cols, cols + kv * dim
    for f, x in enumerate(xs):
        yy, xx = np.divmod(np.tile(np.arange(tokens), videos), side)
        pos = np.stack([np.full(videos * tokens, f), yy, xx], 1).astype(np.float32)
        X = d(x)
        lengths.copy_from(np.full(videos, (f + 1) * tokens))
        hip.norm_residual(X, None, None, H, pre=("rms", dw1, None, 1e-6))
        hip.dense(H, dW, None, QKV)
        hip.paged_append(QKV.columns(0, a), QKV.columns(a, b), QKV.columns(b, b + kv * dim), Q, cache, batch, plan, d(pos))
        hip.paged_attention(Q, A, cache, batch, causal=False)
        hip.dense(A, dWo, None, B)
        hip.norm_residual(B, X, X, H, post=("rms", dw2, None, 1e-6), pre=("layer", None, None, 1e-6), gate=dgate, group_rows=tokens)
        # in 64 bits
        h = norm_residual(x, None, (None,) * 3 + (0.0,), ("rms", w1, None, 1e-6), None, 1.0, None, None, 1)[1]
        qkv = h @ Wqkv.astype(np.float64)
        qk = turned(qkv[:, :b], pos, heads + kv, dim, plan.axis, plan.freq, False)
        round_ = (lambda t: t) if dtype == "float32" else (lambda t: bf16_value(bf16_bits(t.astype(np.float32))).astype(np.float64))
        past_k.append(round_(qk[:, a:]).reshape(videos, tokens, kv, dim))
        past_v.append(round_(qkv[:, b:]).reshape(videos, tokens, kv, dim))
        K, V = np.concatenate(past_k, 1), np.concatenate(past_v, 1)
        q = qk[:, :a].reshape(videos, tokens, heads, dim)
        out = np.zeros((videos, tokens, heads, dim))
        for s in range(videos):
            for hd in range(heads):
                sc = q[s, :, hd] @ K[s, :, hd * kv // heads].T * dim ** -0.5
                w = np.exp(sc - sc.max(1, keepdims=True))
                out[s, :, hd] = (w / w.sum(1, keepdims=True)) @ V[s, :, hd * kv // heads]
        y = out.reshape(-1, cols) @ Wo.astype(np.float64)
        want_s, want_h = norm_residual(y, x.astype(np.float64), ("rms", w2, None, 1e-6), ("layer", None, None, 1e-6), gate, 1.0, None, None, tokens)
        # every stage is off by about 1e-6 of its values (some tens of EPS), a bf16 cache may round a number next to a border the other way
        # (2^-8 of one of 25 to 100 tokens' values, a few of them): 2e-5 and 2e-3 of the largest value
        tol = (2e-5 if dtype == "float32" else 2e-3)
        assert np.abs(X.numpy() - want_s).max() <= tol * np.abs(want_s).max()
        assert np.abs(H.numpy() - want_h).max() <= tol * np.abs(want_h).max()


def test_net_of_attention_blocks(hip):
    """Layers: norm, dense, paged attention, dense, norm, Add, norm, dense, ReLU, dense, Add, norm.  The fused plan, the layer walk and a captured
    plan give the same bits, frame after frame, and the network in 64 bits within 2e-5 of its largest output (some tens of EPS a stage)."""
    from eddl_amd import net as L
    from eddl_amd.attention import PagedBatch, PagedCache, RotaryPlan
    rng = np.random.default_rng(17)
    videos, tokens, heads, kv, dim, frames = 2, 9, 4, 2, 16, 3
    cols, width = heads * dim, -(-frames * tokens // 16)
    plan = RotaryPlan.sections(dim, (2, 3, 3))
    table = rng.permutation(videos * width).reshape(videos, width)

    def build(fuse):
        cache = PagedCache(hip, videos * width, 16, kv, dim)
        batch = PagedBatch(hip.array(table, "int32"), hip.array(np.arange(videos + 1) * tokens, "int32"), hip.empty((videos,), "int32"), tokens, frames * tokens)
        pos = hip.empty((videos * tokens, 3))
        x = L.Input([tokens, cols], videos)
        a = L.PagedAttention(L.Dense(L.RMSNormalization(x), (heads + 2 * kv) * dim, use_bias=False), heads, cache, batch, plan, pos, causal=False)
        s = L.Add(x, L.RMSNormalization(L.Dense(a, cols)))
        h = L.Dense(L.ReLu(L.Dense(L.LayerNormalization(s), 2 * cols)), cols)
        n = L.Net([x], [L.LayerNormalization(L.Add(s, h), affine=False)])
        r = np.random.default_rng(18)
        for l in n.layers:
            for k, v in l.params.items():
                scale = 1 / np.sqrt(v.shape[0]) if k == "W" else 0.1
                l.params[k] = ((1.0 if k == "w" else 0.0) + scale * r.standard_normal(v.shape)).astype(np.float32)
        return n.build(hip, fuse=fuse), batch, pos

    (fused, b0, p0), (walk, b1, p1) = build(True), build(False)
    assert sorted(op.kind for op in fused.ops) == ["attention"] + ["dense"] * 4 + ["norm"] * 3
    assert sum(op.kind in ("norm", "sum") for op in walk.ops) == 6
    graph, want_k, want_v = None, [], []
    P = {(l.kind, i): {k: v.astype(np.float64) for k, v in l.params.items()} for i, l in enumerate(fused.layers)}
    norms, denses = ([P[k] for k in P if k[0] == kind] for kind in ("norm", "dense"))
    for f in range(frames):
        x = rng.standard_normal((videos, tokens, cols), dtype=np.float32)
        yy, xx = np.divmod(np.tile(np.arange(tokens), videos), 3)
        pos = np.stack([np.full(videos * tokens, f), yy, xx], 1).astype(np.float32)
        for b, p in ((b0, p0), (b1, p1)):
            b.lengths.copy_from(np.full(videos, (f + 1) * tokens))
            p.copy_from(pos)
        got = fused.predict(x)[0]
        assert np.array_equal(walk.predict(x)[0], got)
        if graph is None:
            graph = fused.capture()
        fused.input_tensor().copy_from(x)
        fused.run_graph()
        assert np.array_equal(fused.output_of(fused.lout[0]).numpy(), got)
        # in 64 bits
        rows = x.reshape(-1, cols).astype(np.float64)
        rms = lambda t, w: t / np.sqrt((t * t).mean(1, keepdims=True) + 1e-6) * w
        lay = lambda t: (t - t.mean(1, keepdims=True)) / np.sqrt(((t - t.mean(1, keepdims=True)) ** 2).mean(1, keepdims=True) + 1e-5)
        qkv = rms(rows, norms[0]["w"]) @ denses[0]["W"]
        qk = turned(qkv[:, :cols + kv * dim], pos, heads + kv, dim, plan.axis, plan.freq, False)
        want_k.append(qk[:, cols:].reshape(videos, tokens, kv, dim))
        want_v.append(qkv[:, cols + kv * dim:].reshape(videos, tokens, kv, dim))
        K, V, q = np.concatenate(want_k, 1), np.concatenate(want_v, 1), qk[:, :cols].reshape(videos, tokens, heads, dim)
        att = np.zeros((videos, tokens, heads, dim))
        for s in range(videos):
            for hd in range(heads):
                w = np.exp(q[s, :, hd] @ K[s, :, hd * kv // heads].T * dim ** -0.5)
                att[s, :, hd] = w / w.sum(1, keepdims=True) @ V[s, :, hd * kv // heads]
        s = rows + rms(att.reshape(-1, cols) @ denses[1]["W"] + denses[1]["bias"], norms[1]["w"])
        h = np.maximum((lay(s) * norms[2]["w"] + norms[2]["b"]) @ denses[2]["W"] + denses[2]["bias"], 0) @ denses[3]["W"] + denses[3]["bias"]
        want = lay(s + h)
        assert np.abs(got.reshape(-1, cols) - want).max() <= 2e-5 * np.abs(want).max()


@pytest.mark.parametrize("fuse", [True, False])
def test_norms_in_nets_keep_what_others_read(hip, fuse):
    """A sum that a norm and another layer read, a norm that two layers read, and a norm of a network's input as output."""
    from eddl_amd import net as L
    rng = np.random.default_rng(19)
    x, y = L.Input([5, 24], 2), L.Input([5, 24], 2)
    s = L.Add(x, y)
    n1, r = L.LayerNormalization(s), L.ReLu(s)
    n2 = L.RMSNormalization(n1)
    net = L.Net([x, y], [L.Add(n1, r), n2, L.RMSNormalization(x, affine=False)]).build(hip, fuse=fuse)
    a, b = (rng.standard_normal((2, 5, 24), dtype=np.float32) for _ in range(2))
    got = net.predict([a, b])
    t = (a.astype(np.float64) + b).reshape(10, 24)
    n = (t - t.mean(1, keepdims=True)) / np.sqrt(t.var(1, keepdims=True) + 1e-5)
    rms = lambda v: v / np.sqrt((v * v).mean(1, keepdims=True) + 1e-6)
    for g, w in zip(got, (n + np.maximum(t, 0), rms(n), rms(a.reshape(10, 24).astype(np.float64)))):
        assert np.abs(g.reshape(10, 24) - w).max() <= 160 * EPS * 2 * np.abs(w).max()
