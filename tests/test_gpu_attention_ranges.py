"""Attention over keys and values of very different sizes: every row against its own bound (attention_bound.py)."""
import numpy as np
import pytest

from attention_bound import check_rows
from attention_ref import Pool

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
