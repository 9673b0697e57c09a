"""Attention over keys and values of very different sizes: every row against its own bound (attention_bound.py)."""
import ctypes

import numpy as np
import pytest

from attention_bound import check_rows
from attention_ref import EPS, Pool

pytestmark = pytest.mark.gpu


def _attend(hip, pool, q, heads, causal=True, window=0, scale=None):
    cache, batch = pool.on(hip)
    O = hip.full((len(q), q.shape[1]), -7.0)
    hip.paged_attention(hip.array(q), O, cache, batch, scale=scale, causal=causal, window=window)
    return O.numpy()


def _scaled(pool, s, places, name, factor):
    pool.put(s, places, name, pool.get(s, places, name) * np.asarray(factor, np.float32))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("size", [1e-8, 1e-6, 1e-4, 1e-2, 1.0])
def test_small_values_at_all_lengths(hip, dtype, size):
    """Every number of tokens behind the last whole step of 32, in one call: 16 places and more behind the last token hold nothing."""
    rng = np.random.default_rng(1)
    for base in (0, 192):
        lengths = [base + r for r in range(1, 33)]
        pool = Pool(rng, [33] + [1] * 31, [base + 33] + lengths[1:], 1, 64, 32, dtype)
        for s in range(32):
            _scaled(pool, s, np.arange(pool.lengths[s]), "v", size)
        q = rng.standard_normal((pool.rows, 64), dtype=np.float32)
        check_rows(_attend(hip, pool, q, 1, causal=False), q, pool, 1, 0.125, False, 0, (base, size))
        check_rows(_attend(hip, pool, q, 1), q, pool, 1, 0.125, True, 0, (base, size))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("zero", [(0, 16), (0, 32), (96, 112), (100, 150), (288, 304), (304, 320), (0, 320)])
def test_values_that_are_zero(hip, dtype, zero):
    """Tokens whose values are zeros, in front, between and behind others that are small: padding, fresh pages."""
    rng = np.random.default_rng(2)
    for size in (1e-8, 1e-4, 1.0):
        pool = Pool(rng, [40, 2], [320, 320], 2, 64, 64, dtype)
        for s in range(2):
            _scaled(pool, s, np.arange(320), "v", size)
            _scaled(pool, s, np.arange(*zero), "v", 0.0)
        q = rng.standard_normal((42, 4 * 64), dtype=np.float32)
        check_rows(_attend(hip, pool, q, 4, causal=False), q, pool, 4, 0.125, False, 0, (zero, size))
        check_rows(_attend(hip, pool, q, 4), q, pool, 4, 0.125, True, 0, (zero, size))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_keys_that_are_zero(hip, dtype):
    rng = np.random.default_rng(3)
    for size in (1e-8, 1.0):
        pool = Pool(rng, [40], [170], 1, 64, 32, dtype)
        _scaled(pool, 0, np.arange(170), "k", size)
        _scaled(pool, 0, np.arange(64, 80), "k", 0.0)
        q = rng.standard_normal((40, 2 * 64), dtype=np.float32)
        check_rows(_attend(hip, pool, q, 2, scale=0.125 / size), q, pool, 2, 0.125 / size, True, 0, size)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["v", "k", "both"])
@pytest.mark.parametrize("factor", [1e4, 1e6, 1e8, 1e12, 1e25])
def test_large_numbers_in_hidden_places(hip, dtype, name, factor):
    """Finite keys and values that a row does not see - later tokens, tokens before its window - beside small ones that it sees."""
    rng = np.random.default_rng(4)
    for new, length, window in ((150, 240, 0), (150, 240, 40), (7, 240, 40), (40, 200, 0)):
        pool = Pool(rng, [new], [length], 2, 64, 32, dtype)
        places = np.array([3, length - new + 5, length - new // 2, length - 2])
        for n in ("k", "v"):
            if name in (n, "both"):
                _scaled(pool, 0, places, n, factor)
        q = rng.standard_normal((new, 4 * 64), dtype=np.float32)
        check_rows(_attend(hip, pool, q, 4, True, window), q, pool, 4, 0.125, True, window, (name, factor, new, window))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 96, 112, 128, 192, 240, 256])
@pytest.mark.parametrize("new", [2, 40, 130])
def test_tokens_of_very_different_sizes(hip, dtype, dim, new):
    """Tokens in stretches whose values differ by up to 1e25, seen by some rows, by all, or through a window; every row against its own size."""
    rng = np.random.default_rng(5)
    length = new + 150
    for order in ((1e-15, 1e10), (1e10, 1e-15), (1e-15, 1.0, 0.0, 1e10, 1e-5), (1.0, 1e6), (1e7, 1.0, 1e7)):
        pool = Pool(rng, [new], [length], 1, dim, 16, dtype)
        for n, size in enumerate(order):
            _scaled(pool, 0, np.arange(length * n // len(order), length * (n + 1) // len(order)), "v", size)
        q = rng.standard_normal((new, 2 * dim), dtype=np.float32)
        for causal, window in ((False, 0), (True, 0), (True, 20)):
            check_rows(_attend(hip, pool, q, 2, causal, window), q, pool, 2, dim ** -0.5, causal, window, (order, causal, window))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("large", [1e6, 1e9, 1e15])
def test_visible_tokens_without_weight(hip, dtype, large):
    """Large values whose scores are so low that they have no weight, and large keys among small ones that carry the result."""
    rng = np.random.default_rng(6)
    for new in (2, 60, 200):
        length = new + 90
        pool = Pool(rng, [new], [length], 1, 64, 32, dtype)
        q = np.abs(rng.standard_normal((new, 2 * 64), dtype=np.float32)) + np.float32(0.5)
        heavy = np.arange(0, length, 23)
        pool.put(0, heavy, "k", np.full((len(heavy), 1, 64), -300.0, np.float32))
        _scaled(pool, 0, heavy, "v", large)
        check_rows(_attend(hip, pool, q, 2, causal=False), q, pool, 2, 0.125, False, 0, (new, "values"))
        pool.put(0, heavy, "k", np.full((len(heavy), 1, 64), -large, np.float32))
        check_rows(_attend(hip, pool, q, 2, causal=False), q, pool, 2, 0.125, False, 0, (new, "keys"))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_tokens_of_very_different_sizes_in_parts(hip, dtype):
    """The same where a length is divided over workgroups, and beyond the bounds that sized the launch."""
    rng = np.random.default_rng(7)
    for new, length, dim in ((40, 2500, 64), (130, 3000, 128), (300, 1500, 96)):
        pool = Pool(rng, [new, 1], [length, 33], 1, dim, 64, dtype)
        _scaled(pool, 0, np.arange(length), "v", np.where(np.arange(length) % 700 < 350, 1e9, 1.0)[:, None, None])
        q = rng.standard_normal((new + 1, dim), dtype=np.float32)
        for causal, window in ((True, 0), (True, 200)):
            check_rows(_attend(hip, pool, q, 1, causal, window), q, pool, 1, dim ** -0.5, causal, window, (new, causal, window))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_offsets_that_are_no_offsets(hip, dtype):
    """Offsets out of order or at the ends of an int: sequences without rows, and no access outside the buffers (sequence_rows.h, which
    test_sequence_rows_cpu.py checks over all of them)."""
    from eddl_amd.attention import PagedBatch
    rng = np.random.default_rng(8)
    low, high = -2 ** 31, 2 ** 31 - 1
    for new in (5, 100):
        pool = Pool(rng, [new, 3], [new + 20, 40], 1, 64, 16, dtype, fill=0.0)
        cache, batch = pool.on(hip)
        q = rng.standard_normal((new + 3, 2 * 64), dtype=np.float32)
        Q, KV = hip.array(q), hip.array(rng.standard_normal((new + 3, 64)))
        # a row ends before it begins, far before it begins, begins behind the batch, begins before it (those rows are the sequence's first new + 3)
        for offsets, filled in (((4, low, low), 0), ((4, -1, 2), 2), ((high, high, low), 0), ((new + 3, low, 0), 0), ((low, 0, new + 3), new + 3), ((0, high, high), new + 3)):
            b = PagedBatch(batch.table, hip.array(np.array(offsets, np.int64), "int32"), batch.lengths, new, new + 20)
            O, T = hip.full(q.shape, -7.0), hip.full(q.shape, -7.0)
            hip.paged_attention(Q, O, cache, b)
            written = np.any(O.numpy() != -7.0, axis=1)
            assert written[:filled].all() and not written[filled:].any(), offsets
            keys = cache.keys.numpy()
            hip.paged_append(Q, KV, KV, T, cache, b)
            written = np.any(T.numpy() != -7.0, axis=1)
            assert written[:filled].all() and not written[filled:].any(), offsets
            assert filled or np.array_equal(cache.keys.numpy(), keys), offsets
        lengths = hip.array(np.array([low, high]), "int32")
        b = PagedBatch(batch.table, batch.offsets, lengths, new, new + 20)
        hip.paged_append(Q, KV, KV, T, cache, b)
        assert np.array_equal(T.numpy(), q)
        hip.paged_attention(Q, O, cache, b)
        assert np.isnan(O.numpy()).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("page", [16, 32, 64])
def test_released_pages_before_the_windows(hip, dtype, page):
    """Pages before the windows of all rows, released by the program: the same bits as with the pages in place, for windows that begin at
    every place of a page, rows of one and of many tokens and divided lengths."""
    rng = np.random.default_rng(9)
    for new, length, heads, dim in ((1, 300, 2, 64), (20, 300, 1, 80), (100, 300, 1, 64), (1, 3000, 4, 128), (40, 2600, 1, 64), (140, 700, 1, 96)):
        pool = Pool(rng, [new], [length], 1, dim, page, dtype)
        q = rng.standard_normal((new, heads * dim), dtype=np.float32)
        for window in (range(50, 83) if length == 300 else (700, 715, 716, 717)):
            pool_table = pool.table.copy()
            first = max(0, length - new - window + 1)
            want = _attend(hip, pool, q, heads, True, window)
            pool.table[0, :first // page] = -1
            got = _attend(hip, pool, q, heads, True, window)
            pool.table[:] = pool_table
            assert np.array_equal(got, want), (new, length, window)
        check_rows(want, q, pool, heads, dim ** -0.5, True, window, (new, length, window))


# ------------------------------------------------------------------------------------------------- streams
def _streams(hip, n):
    streams = [ctypes.c_void_p() for _ in range(n)]
    for s in streams:
        assert hip.lib.hipStreamCreateWithFlags(ctypes.byref(s), 1) == 0  # (non-blocking: nothing but eddlhip_set_stream orders them)
    return streams


def test_calls_on_changing_streams_come_one_after_another(hip):
    """Calls on two streams in turn, without a synchronization between them, each reading what the one before wrote, divided lengths among
    them, whose counts and parts lie in memory that all calls share; a stream that is destroyed before the next one is set."""
    rng = np.random.default_rng(10)
    calls = []
    for new, length, dim in ((1, 30000, 64), (2, 2000, 64), (1, 7000, 64)):  # (different numbers of parts)
        pool = Pool(rng, [new], [length], 1, dim, 64, "float32")
        cache, batch = pool.on(hip)
        Q = hip.array(rng.standard_normal((new, 4 * dim)))
        O = hip.empty(Q.shape)
        hip.paged_attention(Q, O, cache, batch)
        calls.append((Q, O, O.numpy(), cache, batch))
    a, b = hip.array(rng.standard_normal((20000, 512))), hip.empty((20000, 512))
    hip.norm_residual(a, None, None, b, pre=("rms", None, None, 1e-6))
    once = b.numpy()
    hip.norm_residual(b, None, None, b, pre=("layer", None, None, 1e-6))
    twice = b.numpy()
    streams = _streams(hip, 2)
    try:
        for turn in range(12):
            for _, O, _, _, _ in calls:
                hip.fill_(O, -7.0)
            hip._check(hip.lib.eddlhip_set_stream(hip.dev, streams[0]))
            hip.norm_residual(a, None, None, b, pre=("rms", None, None, 1e-6))
            for n, (Q, O, _, cache, batch) in enumerate(calls):
                hip._check(hip.lib.eddlhip_set_stream(hip.dev, streams[n % 2]))
                hip.paged_attention(Q, O, cache, batch)
            hip._check(hip.lib.eddlhip_set_stream(hip.dev, streams[1]))
            hip.norm_residual(b, None, None, b, pre=("layer", None, None, 1e-6))
            hip._check(hip.lib.eddlhip_set_stream(hip.dev, None))
            for _, O, want, _, _ in calls:
                assert np.array_equal(O.numpy(), want), turn
            assert np.array_equal(b.numpy(), twice), turn
        hip._check(hip.lib.eddlhip_set_stream(hip.dev, streams[0]))
        hip.norm_residual(a, None, None, b, pre=("rms", None, None, 1e-6))
        hip.synchronize()
        assert hip.lib.hipStreamDestroy(streams.pop(0)) == 0
    finally:
        hip._check(hip.lib.eddlhip_set_stream(hip.dev, None))
        for s in streams:
            hip.lib.hipStreamDestroy(s)
    assert np.array_equal(b.numpy(), once)


def test_a_stream_that_the_program_captures(hip):
    """A program's own graph of the library's calls: setting its stream, and the next one, waits for nothing and leaves the capture whole."""
    lib, stream = hip.lib, _streams(hip, 1)[0]
    rng = np.random.default_rng(13)
    x = rng.standard_normal((300, 256), dtype=np.float32)
    X, H, other = hip.array(x), hip.full((300, 256), -7.0), hip.empty((300, 256))
    norm = lambda X, H: hip.norm_residual(X, None, None, H, pre=("rms", None, None, 1e-6))
    norm(X, other)
    want = other.numpy()
    hip.fill_(other, 0.0)
    graph, program = ctypes.c_void_p(), ctypes.c_void_p()
    assert lib.hipStreamBeginCapture(stream, 1) == 0  # (thread-local)
    first = lib.eddlhip_set_stream(hip.dev, stream)
    norm(X, H)
    second = lib.eddlhip_set_stream(hip.dev, None)
    assert lib.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0 and (first, second) == (0, 0)
    assert np.all(H.numpy() == -7.0)
    assert lib.hipGraphInstantiate(ctypes.byref(program), graph, None, None, ctypes.c_size_t(0)) == 0
    for turn in range(3):
        hip.fill_(H, float(turn))
        X.copy_from(x * np.float32(2.0 ** turn))
        assert lib.hipGraphLaunch(program, None) == 0
        norm(X, other)
        hip.synchronize()
        assert np.array_equal(H.numpy(), other.numpy())
    assert np.abs(other.numpy() - want).max() <= 1e-5 * np.abs(want).max()
    lib.hipGraphExecDestroy(program)
    lib.hipGraphDestroy(graph)
    lib.hipStreamDestroy(stream)


def test_setting_a_stream_while_a_graph_is_recorded_is_refused(hip):
    stream, t = _streams(hip, 1)[0], hip.empty((64,))
    hip._check(hip.lib.eddlhip_graph_begin(hip.dev))
    hip.fill_(t, 1.0)
    refused = hip.lib.eddlhip_set_stream(hip.dev, stream)
    graph = ctypes.c_void_p()
    hip._check(hip.lib.eddlhip_graph_end(hip.dev, ctypes.byref(graph)))
    hip._check(hip.lib.eddlhip_graph_destroy(hip.dev, graph))
    assert refused == -1
    hip.lib.hipStreamDestroy(stream)


# ------------------------------------------------------------------------------------------------- sizes at the end of an int
def test_rotary_of_as_many_rows_as_an_int_counts(hip):
    """2^31 - 1 rows of one head of 8, in place: the loops' steps and the launch's size stay in range, and the last rows are turned."""
    from eddl_amd.attention import RotaryPlan
    rows = 2 ** 31 - 1
    X, P = hip.empty((rows, 8)), hip.empty((rows, 1))
    hip.fill_(X, 1.0)
    hip.fill_(P, 0.5)
    hip.rotary_axes(X, X, RotaryPlan(8, [0] * 4, [1.0, 2.0, 3.0, 4.0]), P)
    angle = 0.5 * np.array([1.0, 2.0, 3.0, 4.0])
    want = np.concatenate([np.cos(angle) - np.sin(angle), np.cos(angle) + np.sin(angle)])
    got = np.empty((64, 8), np.float32)
    for row in (0, 2 ** 22 - 32, 2 ** 22 * 100, 2 ** 30, 2 ** 31 - 2 ** 22 - 64, rows - 64):
        hip._check(hip.lib.eddlhip_memcpy_d2h(hip.dev, got.ctypes.data, X.ptr + 32 * row, got.nbytes))
        assert np.abs(got - want).max() <= 8 * EPS * np.sqrt(2), row


def test_the_device_of_a_pointer(hip):
    t, device = hip.empty((64, 64)), ctypes.c_int(7)
    for ptr, want in ((t.ptr, hip.dev), (t.ptr + 100, hip.dev), (np.zeros(64).ctypes.data, -1), (None, -1)):
        assert hip.lib.eddlhip_pointer_device(ptr, ctypes.byref(device)) == 0 and device.value == want
    assert hip.lib.eddlhip_pointer_device(t.ptr, None) == -1
    hip.fill_(t, 1.0)  # (the question about other memory leaves no error behind)


# ------------------------------------------------------------------------------------------------- rotary positions' accuracy
def _turned_in_fp32(x, angle):
    """Halves [rows, 2, pairs] turned with correctly rounded sines, products and sums rounded to fp32."""
    c, s = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    return np.concatenate([x[:, 0] * c - x[:, 1] * s, x[:, 1] * c + x[:, 0] * s], 1)


def test_turned_pairs_are_as_exact_as_with_rounded_sines(hip):
    """The argument of the sine is rounded by 2^-29 of a turn in the mean square (0.26 of the error that correctly rounded sines and the products
    leave, 4.2e-8 of the pair), and a sine of one step's error where half a step is the least adds 0.5 of it: 1.15 times that error together."""
    from eddl_amd.attention import RotaryPlan
    rng = np.random.default_rng(11)
    rows, pairs = 4000, 64
    freq = 10000.0 ** -rng.uniform(0, 1, pairs)
    x = rng.standard_normal((rows, 2, pairs), dtype=np.float32)
    for positions in (np.floor(rng.uniform(0, 1e5, (rows, 1))), np.floor(rng.uniform(-1e6, 1e6, (rows, 1))), rng.uniform(-30, 30, (rows, 1))):
        positions = positions.astype(np.float32)
        Y = hip.empty((rows, 2 * pairs))
        hip.rotary_axes(hip.array(x.reshape(rows, -1)), Y, RotaryPlan(2 * pairs, [0] * pairs, freq), hip.array(positions))
        angle = positions.astype(np.longdouble) * freq
        c, s, z = np.cos(angle), np.sin(angle), x.astype(np.longdouble)
        want = np.concatenate([z[:, 0] * c - z[:, 1] * s, z[:, 1] * c + z[:, 0] * s], 1)
        off, least = np.linalg.norm((Y.numpy() - want).astype(float)), np.linalg.norm((_turned_in_fp32(x, angle) - want).astype(float))
        assert off <= 1.15 * least, (off, least)


def test_quarters_of_a_turn(hip):
    """Angles on and beside whole quarters, both ways round: the right quarter's signs, and on them the 0 and 1 of the angle in 64 bits (9 / 4 of a
    turn, rounded three times, 2^-53 each: 7.5e-16 of a turn, 5e-15)."""
    from eddl_amd.attention import RotaryPlan
    quarters = np.arange(-9, 10)
    turns = (quarters[:, None] / 4 + np.array([-0.125, -1e-3, 0.0, 1e-3, 0.125])[None, :]).reshape(-1, 1)
    positions = turns.astype(np.float32)
    x = np.tile(np.array([[1.0, 0, 0, 0, 0, 0, 0, 0]], np.float32), (len(turns), 1))  # (the first pair's first number; y = cos, sin)
    Y = hip.empty(x.shape)
    hip.rotary_axes(hip.array(x), Y, RotaryPlan(8, [0] * 4, [2 * np.pi] * 4), hip.array(positions))
    got = Y.numpy()[:, [0, 4]]
    angle = 2 * np.pi * positions[:, 0].astype(np.float64)
    want = np.stack([np.cos(angle), np.sin(angle)], 1)
    assert np.abs(got - want).max() <= 4 * EPS
    whole = got.reshape(len(quarters), 5, 2)[:, 2]
    assert np.abs(whole - np.array([[[1, 0], [0, 1], [-1, 0], [0, -1]][q % 4] for q in quarters])).max() <= 5e-15


# ------------------------------------------------------------------------------------------------- memory
@pytest.mark.parametrize("new, length", [(1, 40000), (2, 3000), (40, 3000)])
def test_parts_of_a_padded_batch_take_the_room_of_its_rows(hip, new, length):
    """Tensors of 120000 rows of which the batch has a few: the parts of a divided length do not take room for all of them in every part (30 GB
    for 150 parts), and the result is right, at the front, in the middle and at the end of the tensors."""
    from eddl_amd.attention import PagedBatch
    rng = np.random.default_rng(12)
    pool = Pool(rng, [new], [length], 1, 64, 64, "float32")
    q = rng.standard_normal((new, 8 * 64), dtype=np.float32)
    cache, batch = pool.on(hip)
    rows = 120000
    Q, O = hip.empty((rows, 8 * 64)), hip.empty((rows, 8 * 64))
    hip.workspace_trim()
    for at in (0, 70001, rows - new):
        hip.fill_(O, -7.0)
        hip._check(hip.lib.eddlhip_memcpy_h2d(hip.dev, Q.ptr + 4 * 8 * 64 * at, q.ctypes.data, q.nbytes))
        b = PagedBatch(batch.table, hip.array([at, at + new], "int32"), batch.lengths, new, length)
        hip.paged_attention(Q, O, cache, b)
        got = O.numpy()
        check_rows(got[at:at + new], q, pool, 8, 0.125, True, 0, (new, at))
        assert np.all(got[:at] == -7.0) and np.all(got[at + new:] == -7.0)
        assert hip.workspace_bytes() <= 2 ** 30 + 2 ** 20
