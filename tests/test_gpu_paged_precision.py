"""FP32 rows' mean error on the GPU against the bound of tests/paged_precision.py, which a kernel
with fewer parts of q and of the weights would not keep (tests/test_paged_precision.py)."""
import numpy as np
import pytest

from tests import paged_precision as R
from tests.test_gpu_paged import attention_case, f64, run_attention

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", ("F16", "BF16"))
@pytest.mark.parametrize("dim", (64, 128, 256))
@pytest.mark.parametrize("lens,new", [([31, 65, 130, 257], [1, 1, 1, 1]), ([40, 130, 260], [40, 64, 30]),
                                      ([9001, 700, 5003], [1, 1, 1]), ([9001, 700], [20, 34])],
                         ids=("single", "chunks", "long", "long_chunks"))
def test_mean_error(hip, cache, dim, lens, new):
    c = attention_case(dim + sum(new), lens, new, 4, 2, dim, "F32", cache, 16)
    got, q, k, v = (f64(x) for x in (run_attention(hip, c), c["q"], c["k"], c["v"]))
    off, expected = [], []
    for r, n in enumerate(lens):
        i = np.arange(n)
        at = c["table"][r, i // 16].astype(np.int64), i % 16
        for j in range(new[r]):
            t, p = int(c["start"][r]) + j, n - new[r] + j + 1
            for h in range(4):
                o, e = R.row(q[t, h], k[at[0][:p], at[1][:p], h // 2], v[at[0][:p], at[1][:p], h // 2], dim ** -0.5, cache)
                off.append(got[t, h] - o)
                expected.append(e)
    ratio = R.ratio(np.array(off), np.array(expected))
    print(f"{ratio:.3f}")
    assert ratio <= 1.0
