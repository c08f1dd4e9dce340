"""Infinities, NaN and the ends of the types' ranges in the paged attention, against plain 64-bit
numpy: what masked positions hold does not matter, what visible ones hold counts as the
definition says."""
import numpy as np
import pytest

from tests import paged as P
from tests.test_gpu_paged import TYPES, attention_call, attention_case, check_attention, f64, run_attention

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


# ---- visible infinities ---------------------------------------------------------------

def visible(c, hidden, window=0):
    """attention_case's call in 64 bits, without the positions `hidden` of every request and
    with V's infinities as 0."""
    q, k, v = f64(c["q"]), f64(c["k"].nan_to_num(0, 0, 0)), f64(c["v"].nan_to_num(0, 0, 0))
    out, tol = np.zeros_like(q), np.zeros_like(q)
    for r, n in enumerate(c["lens"]):
        for j in range(c["new"][r]):
            t, p = int(c["start"][r]) + j, n - c["new"][r] + j
            i = np.array([x for x in range(max(0, p + 1 - window) if window else 0, p + 1) if x not in hidden])
            at = c["table"][r, i // c["page"]].astype(np.int64), i % c["page"]
            for h in range(c["heads"]):
                kk, vv = (x[at[0], at[1], h * c["kvh"] // c["heads"]] for x in (k, v))
                s = kk @ q[t, h] * c["dim"] ** -0.5
                w = np.exp(s - s.max())
                out[t, h] = w @ vv / w.sum()
                bound = np.array([np.abs(kk * q[t, h]).sum(-1).max() * c["dim"] ** -0.5, np.abs(vv).max(), len(i)])
                tol[t, h] = P.attention_tolerance(out[t, h], bound, c["dim"], c["gtype"], c["cache"])
    return out, tol


@pytest.mark.parametrize("gtype,cache", TYPES)
@pytest.mark.parametrize("dim", (64, 128, 256))
@pytest.mark.parametrize("new", ([1, 1], [3, 1], [70, 40]))
def test_visible_infinities(hip, gtype, cache, dim, new):
    """A key of -inf where q is positive has no weight; a value of +-inf makes its column so."""
    c = attention_case(73, [200, 90], new, 4, 2, dim, gtype, cache, 16)
    c["q"][..., 7] = c["q"][..., 7].abs() + 0.25
    for r in range(2):
        for i in (5, 15):
            c["k"][slot(c, r, i)][:, 7] = -INF
        c["v"][slot(c, r, 9)][:, 3] = INF
        c["v"][slot(c, r, 12)][:, 11] = -INF
    want, tol = visible(c, {5, 15})
    got = run_attention(hip, c)[:sum(new)].float()
    assert (got[..., 3] == INF).all() and (got[..., 11] == -INF).all()
    rest = [i for i in range(dim) if i not in (3, 11)]
    off = np.abs(got.cpu().numpy().astype(np.float64) - want[:sum(new)])[..., rest]
    assert np.all(np.isfinite(off)) and np.all(off <= tol[:sum(new)][..., rest])


@pytest.mark.parametrize("gtype,cache", TYPES)
@pytest.mark.parametrize("new", ([1], [40]))
def test_visible_infinities_in_long_contexts(hip, gtype, cache, new):
    """The same in one of a long row's parts, and in whole tiles and cut ones."""
    c = attention_case(74, [5000], new, 2, 1, 64, gtype, cache, 16)
    c["q"][..., 7] = c["q"][..., 7].abs() + 0.25
    keys = {100, 2047, 4950}
    for i in keys:
        c["k"][slot(c, 0, i)][:, 7] = -INF
    c["v"][slot(c, 0, 3001)][:, 3] = INF
    want, tol = visible(c, keys)
    got = run_attention(hip, c)[:sum(new)].float()
    assert (got[..., 3] == INF).all()
    rest = [i for i in range(64) if i != 3]
    off = np.abs(got.cpu().numpy().astype(np.float64) - want[:sum(new)])[..., rest]
    assert np.all(np.isfinite(off)) and np.all(off <= tol[:sum(new)][..., rest])


@pytest.mark.parametrize("gtype", ("F16", "F32"))
@pytest.mark.parametrize("new", ([1], [40]))
def test_infinity_of_a_small_weight(hip, gtype, new):
    """A weight that F16 cannot hold beside the row's largest still makes infinity of it."""
    c = attention_case(75, [90], new, 2, 1, 64, gtype, "F16", 16)
    c["q"][..., 7] = 8.0
    c["k"][slot(c, 0, 20)][:, 7] = -40.0  # 40 below the others: a weight of about 2^-57
    c["v"][slot(c, 0, 20)][:, 3] = INF
    got = run_attention(hip, c)[:sum(new)].float()
    assert (got[..., 3] == INF).all() and torch.isfinite(got[..., 4:]).all()


@pytest.mark.parametrize("gtype,cache", TYPES)
def test_no_score_above_minus_infinity(hip, gtype, cache):
    """A row all of whose scores are -inf is 0, its neighbours that see more are not."""
    c = attention_case(79, [3, 5], [3, 1], 4, 2, 64, gtype, cache, 16)
    c["q"][..., 7] = c["q"][..., 7].abs() + 0.25
    for r, i in ((0, 0), (0, 1), (1, 0), (1, 1), (1, 2), (1, 3), (1, 4)):
        c["k"][slot(c, r, i)][:, 7] = -INF
    got = run_attention(hip, c)
    assert (got[[0, 1, 3]] == 0).all()
    v = c["v"][slot(c, 0, 2)].float().repeat_interleave(2, 0)
    # w v / w of one weight w: F32's parts hold 22 bits of it (four half steps of FP32), the sum
    # of their products, 1 / w and its product lose a half step each; 16-bit types end on v
    assert torch.all((got[2].float() - v).abs() <= 8 * 2.0 ** -24 * v.abs())


@pytest.mark.parametrize("gtype,cache", TYPES)
@pytest.mark.parametrize("new", ([1, 1], [40, 3]))
def test_infinite_queries(hip, gtype, cache, new):
    """An infinity in q that makes -inf of every score gives 0, one that makes +inf of any NaN."""
    c = attention_case(80, [90, 50], new, 4, 2, 64, gtype, cache, 16)
    c["k"][..., 7] = -c["k"][..., 7].abs() - 0.5
    c["k"][..., 9] = -c["k"][..., 9].abs() - 0.5
    c["k"][slot(c, 1, 5)][:, 9] = 1.0
    c["q"][:new[0], 1, 7] = INF
    c["q"][new[0]:, 2, 9] = INF
    got = run_attention(hip, c)
    assert (got[:new[0], 1] == 0).all() and torch.isnan(got[new[0]:sum(new), 2]).all()
    assert torch.isfinite(got[:new[0], [0, 2, 3]].float()).all()


def test_largest_query(hip):
    """The largest FP32 value, which as BF16 would be infinite, times the smallest K."""
    c = attention_case(81, [70, 40], [1, 40], 2, 1, 64, "F32", "BF16", 16)
    c["q"][..., 7] = torch.finfo(torch.float32).max
    c["k"][..., 7] = torch.where(c["k"][..., 7].float() > 0, 2.0 ** -126, 2.0 ** -127).bfloat16()
    check_attention(c, run_attention(hip, c))


# ---- the ends of the range ------------------------------------------------------------

@pytest.mark.parametrize("gtype", ("BF16", "F32"))
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("lens,new", [([300, 4000], [1, 1]), ([300, 4000], [70, 40])])
def test_largest_values(hip, gtype, dim, lens, new):
    """Values near the end of BF16's range: their mean is in it."""
    c = attention_case(76, lens, new, 4, 2, dim, gtype, "BF16", 16)
    v = c["v"]
    v[torch.isfinite(v)] = (2.0 ** 127 * (1.25 + 0.25 * torch.tanh(v[torch.isfinite(v)].float()))).bfloat16()
    check_attention(c, run_attention(hip, c))


@pytest.mark.parametrize("gtype", ("BF16", "F32"))
@pytest.mark.parametrize("new", ([1, 1], [70, 40]))
def test_small_values(hip, gtype, new):
    """Small values keep their bits: the same call with values 2^-70 times as large."""
    c = attention_case(77, [300, 4000], new, 4, 2, 64, gtype, "BF16", 16)
    small = {**c, "v": (c["v"].float() * 2.0 ** -70).bfloat16()}
    assert torch.equal(run_attention(hip, c)[:sum(new)], run_attention(hip, small)[:sum(new)] * 2.0 ** 70)


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
