"""Infinities and NaN in the paged attention, against plain 64-bit numpy: what masked positions
hold does not matter."""
import numpy as np
import pytest

from tests import paged as P
from tests.test_gpu_paged import attention_case, f64, run_attention

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def slot(c, r, i):
    """Page and slot of request r's position i."""
    return int(c["table"][r, i // c["page"]]), i % c["page"]


def clean(c):
    """The same call with its NaN and infinities gone."""
    return {**c, "k": c["k"].nan_to_num(0, 0, 0), "v": c["v"].nan_to_num(0, 0, 0)}


def close(c, got, rows, window=0, sinks=0, columns=slice(None)):
    """The rows' columns are those of the call without NaN and infinities, within its bound."""
    ref = clean(c)
    want, bound = P.attention(f64(ref["q"]), f64(ref["k"]), f64(ref["v"]), c["table"], c["start"], c["lens"], c["page"],
                              c["dim"] ** -0.5, window, sinks)
    tol = P.attention_tolerance(np.nan_to_num(want), bound, c["dim"], c["gtype"], c["cache"])
    got = f64(got)[rows][..., columns]
    assert np.all(np.isfinite(got))
    assert np.all(np.abs(got - want[rows][..., columns]) <= tol[rows][..., columns])


# ---- masked values --------------------------------------------------------------------

@pytest.mark.parametrize("gtype,cache", [("F32", "F16"), ("BF16", "BF16")])
@pytest.mark.parametrize("bad", (NAN, INF))
def test_later_token_beside_rows_of_one_position(hip, gtype, cache, bad):
    """32 rows of a tile at one position, the tile's others at later ones."""
    c = attention_case(70, [100], [4], 32, 1, 64, gtype, cache, 16)
    c["v"][slot(c, 0, 99)] = bad
    close(c, run_attention(hip, c), [0, 1, 2])


@pytest.mark.parametrize("gtype,cache", [("F32", "F16"), ("BF16", "BF16")])
@pytest.mark.parametrize("heads,kvh,new", [(2, 2, 33), (2, 1, 17), (4, 1, 17)])
@pytest.mark.parametrize("bad", (NAN, INF))
def test_hidden_by_a_window_beside_rows_of_one_position(hip, gtype, cache, heads, kvh, new, bad):
    """A tile whose last few rows stand at one position: the window hides from them what the
    tile's first rows see."""
    c = attention_case(71, [100 + new], [new], heads, kvh, 64, gtype, cache, 16)
    last = 100 + new - 1
    i = last - 50  # the first position that the last row does not see
    c["v"][slot(c, 0, i)] = bad
    got = run_attention(hip, c, window=50)
    close(c, got, [new - 1], window=50)
    assert not torch.isfinite(got[0].float()).any()  # and the first row does see it
