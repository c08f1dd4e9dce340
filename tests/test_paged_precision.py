"""The bound on FP32 rows' mean error (tests/paged_precision.py) holds for the parts that the
kernels take, and not for fewer, on inputs like those of the GPU's tests."""
import numpy as np
import pytest

from tests import paged_precision as R


def rows(seed, dim, lens, cache, q_parts, w_parts):
    g = np.random.default_rng(seed)
    off, expected = [], []
    for n in lens:
        k, v = g.standard_normal((n, dim)), g.standard_normal((n, dim))
        k[:, ::16] *= 4
        k, v = (R.rounded(x.astype(np.float32), cache).astype(np.float64) for x in (k, v))
        for _ in range(4):
            q = g.standard_normal(dim).astype(np.float32).astype(np.float64)
            o, e = R.row(q, k, v, dim ** -0.5, cache)
            off.append(R.simulated(q, k, v, dim ** -0.5, cache, q_parts, w_parts) - o)
            expected.append(e)
    return R.ratio(np.array(off), np.array(expected))


@pytest.mark.parametrize("cache", ("F16", "BF16"))
@pytest.mark.parametrize("dim", (64, 128, 256))
@pytest.mark.parametrize("lens", ([31, 65, 130, 257], [9001, 700, 5003]), ids=("short", "long"))
def test_bound_sees_a_missing_part(cache, dim, lens):
    full = R.PARTS[cache]
    assert rows(dim, dim, lens, cache, full, full) <= 0.8
    assert rows(dim, dim, lens, cache, full - 1, full - 1) > 1.1
