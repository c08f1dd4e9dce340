"""Infinities and NaN in the paged attention, against plain 64-bit numpy: what masked positions
hold does not matter."""
import numpy as np
import pytest

from tests import paged as P
from tests.test_gpu_paged import TYPES, attention_call, attention_case, f64, run_attention

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
    tol = np.broadcast_to(P.attention_tolerance(np.nan_to_num(want), bound, c["dim"], c["gtype"], c["cache"]), want.shape)
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


@pytest.mark.parametrize("gtype,cache", TYPES)
@pytest.mark.parametrize("new", (3, 40))
@pytest.mark.parametrize("bad", (NAN, INF))
def test_a_seen_nan_does_not_hide_a_masked_one(hip, gtype, cache, new, bad):
    """Rows that see a NaN in one column keep the masked values of a later token out of the
    others."""
    c = attention_case(72, [160], [new], 4, 2, 128, gtype, cache, 16)
    c["v"][slot(c, 0, 3)][0, 5] = NAN
    c["v"][slot(c, 0, 159)][:, 6] = bad
    got = run_attention(hip, c)
    rest = [i for i in range(128) if i != 5]
    rows = list(range(new - 1))
    close(c, got, rows, columns=rest)
    assert torch.isnan(got[:new, :2, 5]).all()
    assert torch.isfinite(got[rows, 2:, 5].float()).all()


# ---- what a NaN that rows see costs ---------------------------------------------------

def least_time(hip, c):
    """Of several calls, the shortest time between events around it, in ms."""
    out = torch.full_like(c["q"], 5.0)
    call, best = attention_call(c, out), INF
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(8):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record(stream)
        hip.paged_attention_async(call, stream.cuda_stream)
        b.record(stream)
        stream.synchronize()
        if i:
            best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("gtype,cache", [("BF16", "BF16"), ("F32", "F16")])
def test_seen_nan_does_not_do_rows_again(hip, gtype, cache):
    """Rows that see a NaN, in one column or all, are not done again by themselves: another look
    at their keys and values, no more."""
    c = attention_case(78, [4000], [4000], 8, 2, 128, gtype, cache, 16)
    plain = least_time(hip, c)
    for name, column in (("v", 5), ("k", 5), ("v", slice(None))):
        bad = {**c, name: c[name].clone()}
        bad[name][slot(c, 0, 64)][:, column] = NAN
        spent = least_time(hip, bad)
        print(f"{gtype} {name} {column}: {plain:.3f} -> {spent:.3f} ms")
        assert spent < 6 * plain
