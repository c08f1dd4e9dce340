"""The paged-cache operators on the GPU against plain 64-bit numpy (tests/paged.py)."""
import threading

import numpy as np
import pytest

from pokitlms_amd.backend import PagedAppend, PagedAttention, PagedKV, PagedPlan, rotary_axes
from tests import paged as P

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

GGUF = {"F32": 0, "F16": 1, "BF16": 30}
DT = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16}


def ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.uint32).view(np.int32)).cuda()


def words(t):
    return t.cpu().numpy().view(np.uint32)


def f64(t):
    return t.float().cpu().numpy().astype(np.float64)


class Plan:
    """A plan's buffers on the device."""

    def __init__(self, page, pages, rows, lens, new, table, stack, count, release=None, alias=False):
        n = len(lens)
        self.lens, self.new, self.table = ints(lens), ints(new), ints(table)
        self.stack, self.count = ints(stack), ints([count])
        self.release = None if release is None else ints(release)
        self.lens_out = self.lens if alias else ints([77] * n)
        self.count_out = self.count if alias else ints([77])
        self.start, self.status = ints([77] * (n + 1)), ints([77] * 4)
        self.positions, self.slots, self.owner = (ints([77] * rows) for _ in range(3))
        self.call = PagedPlan(n, pages, page, table.shape[1], rows, lens=self.lens.data_ptr(),
                              new_lens=self.new.data_ptr(), block_table=self.table.data_ptr(),
                              free_pages=self.stack.data_ptr(), free_count=self.count.data_ptr(),
                              lens_out=self.lens_out.data_ptr(), free_count_out=self.count_out.data_ptr(),
                              query_start=self.start.data_ptr(), positions=self.positions.data_ptr(),
                              slots=self.slots.data_ptr(), token_request=self.owner.data_ptr(),
                              status=self.status.data_ptr(),
                              release=0 if release is None else self.release.data_ptr())

    def outputs(self):
        return {"table": words(self.table), "stack": words(self.stack), "count": words(self.count_out)[0],
                "lens": words(self.lens_out), "start": words(self.start), "positions": words(self.positions),
                "slots": words(self.slots), "owner": words(self.owner), "status": words(self.status)}


def same_plan(got, want):
    for name in want:
        assert np.array_equal(np.asarray(got[name]), np.asarray(want[name], dtype=np.uint32)), name


def plan_inputs(seed, requests, page, width, spare, released=False, holes=False):
    g = np.random.default_rng(seed)
    lens = g.integers(0, width * page - 2, requests)
    lens[g.random(requests) < 0.2] = 0
    new = np.minimum(g.integers(0, 3 * page + 2, requests), width * page - lens)
    new[g.random(requests) < 0.3] = 0
    release = (g.random(requests) < 0.3).astype(int) if released else None
    used = -(-lens // page)
    pages = int(used.sum()) + spare
    order = g.permutation(pages)
    table = np.full((requests, width), P.NONE, np.uint32)
    at = 0
    for r in range(requests):
        table[r, :used[r]] = order[at:at + used[r]]
        at += used[r]
    stack = np.full(pages, 0xEEEE, np.uint32)
    count = pages - at
    stack[:count] = order[at:]
    if holes:  # pages that a window has left behind, and an entry that names none
        table[:, ::3] = np.where(table[:, ::3] != P.NONE, P.NONE, table[:, ::3])
        table[-1, -1] = pages
    return pages, lens, new, release, table, stack, count


@pytest.mark.parametrize("requests,page,width", [(1, 16, 4), (1, 1, 3), (7, 16, 5), (64, 8, 9), (65, 1024, 2),
                                                 (1024, 4, 6), (1025, 4, 6), (8192, 2, 3)])
@pytest.mark.parametrize("released,holes,alias", [(False, False, False), (True, False, True), (True, True, False)])
def test_plan(hip, requests, page, width, released, holes, alias):
    spare = requests * 4 * (3 if page < 8 else 2) + 3
    pages, lens, new, release, table, stack, count = plan_inputs(
        requests + page, requests, page, width, spare, released, holes)
    for rows in {max(1, int(new.sum())), int(new.sum()) + 5, int(new.sum()) + 4500}:
        bits, want = P.plan(page, pages, rows, lens, new, release, table, stack, count)
        assert bits == 0
        p = Plan(page, pages, rows, lens, new, table, stack, count, release, alias)
        hip.paged_plan_async(p.call)
        hip.sync()
        same_plan(p.outputs(), want)


def test_plan_many_tokens_in_one_request(hip):
    """More tokens than one workgroup writes, a start inside a page, an end inside one."""
    page, width, n = 32, 700, 20011
    table = np.full((3, width), P.NONE, np.uint32)
    table[1, 0] = 5
    pages = 1300
    stack = np.array([i for i in range(pages) if i != 5] + [0xEEEE], np.uint32)
    args = ([0, 9, 0], [40, n, 33], None, table, stack, pages - 1)
    _, want = P.plan(page, pages, n + 100, *args[:2], None, *args[3:])
    p = Plan(page, pages, n + 100, *args[:2], *args[3:])
    hip.paged_plan_async(p.call)
    hip.sync()
    same_plan(p.outputs(), want)


@pytest.mark.parametrize("rows", (64, 5000))
def test_plan_that_does_not_fit_changes_nothing(hip, rows):
    page, width = 16, 4
    base = dict(lens=[16, 5, 30], new=[3, 12, 2], release=None, count=4)
    table = np.full((3, width), P.NONE, np.uint32)
    table[0, 0], table[1, 0], table[2, :2] = 1, 2, (3, 4)
    stack = np.array([7, 0, 6, 5, 9, 9, 9, 9], np.uint32)
    cases = [(dict(count=1), 1), (dict(new=[60, 1, 1]), 2), (dict(new=[49, 70, 1], count=8), 2),
             (dict(new=[rows + 1, 1, 1]), 4), (dict(count=9), 8), (dict(lens=[65, 5, 30]), 8),
             (dict(release=[1, 1, 1], count=5), 8), (dict(new=[0xFFFFFFFF, 0xFFFFFFFF, 2]), 4)]
    for change, bit in cases:
        a = {**base, **change}
        for alias in (False, True):
            want_bits, want = P.plan(page, 8, rows, a["lens"], a["new"], a["release"], table, stack, a["count"])
            p = Plan(page, 8, rows, a["lens"], a["new"], table, stack, a["count"], a["release"], alias)
            hip.paged_plan_async(p.call)
            hip.sync()
            assert want_bits & bit and want_bits == want["status"][0]
            same_plan(p.outputs(), want)


# ---- append ---------------------------------------------------------------------------

def append_case(seed, tokens, heads, kvh, dim, gtype, cache, page, axes=1, rotary=None, norm=True, far=4096,
                layout="slots", pads=0):
    g = torch.Generator().manual_seed(seed)
    rotary = dim if rotary is None else rotary
    rows, qd, kd = tokens + pads, heads * dim, kvh * dim
    pages = -(-rows // page) + 2
    qkv = torch.randn(rows, qd + 2 * kd + 16, generator=g).to(DT[gtype]).cuda()
    shape = (pages, page, kvh, dim) if layout == "slots" else (pages, kvh, page, dim)
    kc, vc = (torch.randn(shape, generator=g).to(DT[cache]).cuda() for _ in range(2))
    slots = np.full(rows, P.NONE, np.uint32)
    slots[:tokens] = torch.randperm(pages * page, generator=g)[:tokens].numpy()
    if pads > 1:  # a slot behind the cache, in the middle
        slots[tokens // 2], slots[tokens] = pages * page, slots[tokens // 2]
    pos = torch.randint(0, far, (axes, rows), generator=g).numpy().astype(np.uint32)
    w = [(1 + 0.2 * torch.randn(dim, generator=g)).cuda() if norm else None for _ in range(2)]
    axis = [(5 * i) % axes for i in range(rotary // 2)]
    return dict(qkv=qkv, kc=kc, vc=vc, slots=slots, pos=pos, w=w, axis=axis, rows=rows, pages=pages,
                qd=qd, kd=kd, rotary=rotary, layout=layout, heads=heads, kvh=kvh, dim=dim, gtype=gtype,
                cache=cache, page=page, axes=axes)


def strides(c):
    if c["layout"] == "slots":
        return {}
    return dict(page_stride=c["kvh"] * c["page"] * c["dim"], slot_stride=c["dim"],
                head_stride=c["page"] * c["dim"])


def run_append(hip, c, in_place=False, stream=0):
    qkv = c["qkv"].clone()
    q, k, v = qkv[:, 8:8 + c["qd"]], qkv[:, 8 + c["qd"]:], qkv[:, 8 + c["qd"] + c["kd"]:]
    q_out = q if in_place else torch.full((c["rows"], c["qd"]), 3.0, dtype=DT[c["gtype"]], device="cuda")
    kc, vc, slots, pos = c["kc"].clone(), c["vc"].clone(), ints(c["slots"]), ints(c["pos"])
    hip.paged_append_async(PagedAppend(
        PagedKV(kc.data_ptr(), vc.data_ptr(), GGUF[c["cache"]], c["pages"], c["page"], c["kvh"], c["dim"],
                **strides(c)),
        GGUF[c["gtype"]], c["rows"], c["heads"], q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(),
        q_out=q_out.data_ptr(), slots=slots.data_ptr(), q_stride=qkv.stride(0), k_stride=qkv.stride(0),
        v_stride=qkv.stride(0), q_out_stride=qkv.stride(0) if in_place else 0,
        q_norm=0 if c["w"][0] is None else c["w"][0].data_ptr(),
        k_norm=0 if c["w"][1] is None else c["w"][1].data_ptr(), rms_eps=1e-6, rope_theta=1e6,
        rotary_dim=c["rotary"], positions=pos.data_ptr(), axes=c["axes"], pair_axis=c["axis"]), stream)
    torch.cuda.synchronize()
    return q_out, kc, vc, qkv


def check_append(c, q_out, kc, vc, before):
    """q, K and V of live tokens within their bound; everything else as it was.  Bound: an
    FP32 norm of dim values loses (dim + 8) half steps at most, a rotation of two products
    with cosine and sine of 2^-23 each 8 more, of the pair's size; then one rounding."""
    d, rows, qd, kd = c["dim"], c["rows"], c["qd"], c["kd"]
    x = f64(c["qkv"])
    q = x[:, 8:8 + qd].reshape(rows, -1, d)
    k = x[:, 8 + qd:8 + qd + kd].reshape(rows, -1, d)
    v = x[:, 8 + qd + kd:8 + qd + 2 * kd].reshape(rows, -1, d)
    w = [None if t is None else f64(t) for t in c["w"]]
    live = np.nonzero(c["slots"] < c["pages"] * c["page"])[0]
    order = (0, 1, 2, 3) if c["layout"] == "slots" else (0, 2, 1, 3)
    for what, got, rows_in, weight, rounding in (
            ("q", f64(q_out), q, w[0], P.EPS[c["gtype"]]), ("k", f64(kc), k, w[1], P.EPS[c["cache"]]),
            ("v", f64(vc), v, None, P.EPS[c["cache"]])):
        want = rows_in[live] if what == "v" else P.heads(
            rows_in[live], weight, 1e-6, c["pos"][:, live], c["axis"], 1e6, c["rotary"])
        size = np.abs(want)
        half = c["rotary"] // 2
        if what != "v" and half:
            pair = np.maximum(size[..., :half], size[..., half:2 * half])
            size[..., :half], size[..., half:2 * half] = pair, pair
        tol = size * (d + 16) * 2.0 ** -24 * (what != "v") + np.abs(want) * rounding / 2 + 2.0 ** -25
        if what == "q":
            full = before[0].reshape(rows, -1, d).copy()
            full_tol = np.zeros_like(full)
            full[live], full_tol[live] = want, tol
            got = got.reshape(rows, -1, d)
        else:
            full = before[1 if what == "k" else 2].transpose(order).reshape(-1, c["kvh"], d).copy()
            full_tol = np.zeros_like(full)
            full[c["slots"][live]], full_tol[c["slots"][live]] = want, tol
            got = got.transpose(order).reshape(-1, c["kvh"], d)
        over = np.abs(got - full) - full_tol
        assert np.max(over) <= 0.0, (what, np.unravel_index(np.argmax(over), over.shape), np.max(over))


@pytest.mark.parametrize("tokens,heads,kvh,dim", [(1, 32, 4, 128), (5, 8, 2, 64), (33, 6, 3, 256),
                                                  (1, 1, 1, 64), (1025, 4, 1, 128), (1030, 3, 3, 256)])
@pytest.mark.parametrize("gtype,cache", [("F32", "F16"), ("F16", "F16"), ("BF16", "BF16"), ("F32", "BF16"),
                                         ("F16", "BF16")])
def test_append(hip, tokens, heads, kvh, dim, gtype, cache):
    c = append_case(tokens + dim, tokens, heads, kvh, dim, gtype, cache, 16)
    before = np.full((c["rows"], c["qd"]), 3.0), f64(c["kc"]), f64(c["vc"])
    q, k, v, _ = run_append(hip, c)
    check_append(c, q, k, v, before)


@pytest.mark.parametrize("case", [
    dict(axes=3, rotary=128), dict(axes=4, rotary=64), dict(rotary=16), dict(rotary=0), dict(norm=False),
    dict(far=1 << 31, axes=2), dict(page=1), dict(page=1024), dict(layout="heads"), dict(pads=3),
    dict(layout="heads", pads=7, axes=3, rotary=96)], ids=str)
@pytest.mark.parametrize("tokens", (9, 1101))
def test_append_forms(hip, case, tokens):
    args = dict(page=8, axes=1)
    args.update(case)
    c = append_case(7, tokens, 5, 2, 128, "F32", "F16", **args)
    before = np.full((c["rows"], c["qd"]), 3.0), f64(c["kc"]), f64(c["vc"])
    q, k, v, _ = run_append(hip, c)
    check_append(c, q, k, v, before)


def test_append_in_place(hip):
    """q turned where it lies: its neighbours in the projections' rows stay."""
    c = append_case(3, 40, 8, 2, 128, "BF16", "BF16", 16, pads=2)
    before = f64(c["qkv"])[:, 8:8 + c["qd"]], f64(c["kc"]), f64(c["vc"])
    q, k, v, qkv = run_append(hip, c, in_place=True)
    check_append(c, q.contiguous(), k, v, before)
    a, b = c["qkv"].clone(), qkv.clone()
    a[:, 8:8 + c["qd"]], b[:, 8:8 + c["qd"]] = 0, 0
    assert torch.equal(a, b)


def test_append_without_q(hip):
    c = append_case(4, 11, 2, 2, 64, "F16", "F16", 16)
    kc, vc, slots, pos = c["kc"].clone(), c["vc"].clone(), ints(c["slots"]), ints(c["pos"])
    q, k, v, _ = run_append(hip, c)
    kk = c["qkv"][:, 8 + c["qd"]:]
    hip.paged_append_async(PagedAppend(
        PagedKV(kc.data_ptr(), vc.data_ptr(), 1, c["pages"], 16, 2, 64), 1, c["rows"], 0, k=kk.data_ptr(),
        v=kk[:, c["kd"]:].data_ptr(), slots=slots.data_ptr(), k_stride=kk.stride(0), v_stride=kk.stride(0),
        k_norm=c["w"][1].data_ptr(), rms_eps=1e-6, rope_theta=1e6, rotary_dim=64, positions=pos.data_ptr(),
        pair_axis=c["axis"]))
    torch.cuda.synchronize()
    assert torch.equal(k, kc) and torch.equal(v, vc)


# ---- attention ------------------------------------------------------------------------

def attention_case(seed, lens, new, heads, kvh, dim, gtype, cache, page, width_more=1, layout="slots", pads=1):
    g = torch.Generator().manual_seed(seed)
    used = [-(-n // page) for n in lens]
    pages, width = sum(used) + 2, max(used + [1]) + width_more
    order = torch.randperm(pages, generator=g).numpy()
    table = np.full((len(lens), width), P.NONE, np.uint32)
    at = 0
    for r, u in enumerate(used):
        table[r, :u] = order[at:at + u]
        at += u
    shape = (pages, page, kvh, dim) if layout == "slots" else (pages, kvh, page, dim)
    k = torch.randn(shape, generator=g)
    k[..., ::16] *= 4
    v = torch.randn(shape, generator=g)
    # what no position fills: poison
    free = torch.ones(pages, page, dtype=torch.bool)
    for r, n in enumerate(lens):
        i = np.arange(n)
        free[torch.from_numpy(table[r, i // page].astype(np.int64)), torch.from_numpy(i % page)] = False
    if layout == "slots":
        k[free], v[free] = float("nan"), float("inf")
    else:
        k.transpose(1, 2)[free], v.transpose(1, 2)[free] = float("nan"), float("inf")
    rows = sum(new) + pads
    return dict(k=k.to(DT[cache]).cuda(), v=v.to(DT[cache]).cuda(), table=table, lens=list(lens), new=list(new),
                q=torch.randn(rows, heads, dim, generator=g).to(DT[gtype]).cuda(), heads=heads, kvh=kvh, dim=dim,
                gtype=gtype, cache=cache, page=page, pages=pages, layout=layout, rows=rows,
                start=np.concatenate([[0], np.cumsum(new)]).astype(int))


def attention_call(c, out, window=0, sinks=0, scale=0.0, max_new=0, held=None):
    lens, start, table = ints(c["lens"]), ints(c["start"]), ints(c["table"])
    call = PagedAttention(
        PagedKV(c["k"].data_ptr(), c["v"].data_ptr(), GGUF[c["cache"]], c["pages"], c["page"], c["kvh"],
                c["dim"], **strides(c)),
        GGUF[c["gtype"]], c["heads"], len(c["lens"]), c["rows"], q=c["q"].data_ptr(), out=out.data_ptr(),
        query_start=start.data_ptr(), lens=lens.data_ptr(), block_table=table.data_ptr(),
        table_stride=c["table"].shape[1], window=window, sinks=sinks, scale=scale, max_new=max_new)
    call.held = lens, start, table
    return call


def run_attention(hip, c, **kw):
    out = torch.full_like(c["q"], 5.0)
    hip.paged_attention_async(attention_call(c, out, **kw))
    torch.cuda.synchronize()
    return out


def check_attention(c, got, window=0, sinks=0, scale=0.0):
    k, v = f64(c["k"]), f64(c["v"])
    if c["layout"] != "slots":
        k, v = k.transpose(0, 2, 1, 3), v.transpose(0, 2, 1, 3)
    want, bound = P.attention(f64(c["q"]), k, v, c["table"], c["start"], c["lens"], c["page"],
                              scale or c["dim"] ** -0.5, window, sinks)
    tol = P.attention_tolerance(np.nan_to_num(want), bound, c["dim"], c["gtype"], c["cache"])
    live = ~np.isnan(want[..., :1]).repeat(c["dim"], -1)
    got = f64(got)
    assert np.all(got[~live] == 5.0)
    off = np.where(live, np.abs(got - np.where(live, want, got)), 0.0)
    assert np.all(np.isfinite(got)) and np.all(off <= tol), (
        np.unravel_index(np.argmax(off - tol), off.shape), np.max(off - tol))


TYPES = [("F32", "F16"), ("F16", "F16"), ("BF16", "BF16"), ("F32", "BF16")]


@pytest.mark.parametrize("gtype,cache", TYPES)
@pytest.mark.parametrize("dim", (64, 128, 256))
@pytest.mark.parametrize("heads,kvh", [(8, 2), (3, 3), (16, 1), (7, 1)])
def test_attention_single_tokens(hip, gtype, cache, dim, heads, kvh):
    lens = [1, 2, 31, 32, 33, 64, 65, 130, 257]
    c = attention_case(dim + heads, lens, [1] * len(lens), heads, kvh, dim, gtype, cache, 16)
    check_attention(c, run_attention(hip, c, max_new=1))


@pytest.mark.parametrize("gtype,cache", TYPES)
@pytest.mark.parametrize("dim", (64, 128, 256))
@pytest.mark.parametrize("heads,kvh", [(8, 2), (2, 2), (5, 1)])
def test_attention_mixed(hip, gtype, cache, dim, heads, kvh):
    """Chunks of many lengths (from nothing, over a context), single tokens and idle requests."""
    lens = [40, 5, 77, 1, 130, 200, 0, 33, 64, 260]
    new = [40, 1, 17, 1, 64, 3, 0, 0, 63, 130]
    c = attention_case(dim + heads, lens, new, heads, kvh, dim, gtype, cache, 8)
    check_attention(c, run_attention(hip, c))


@pytest.mark.parametrize("page", (1, 2, 16, 64, 1024))
@pytest.mark.parametrize("layout", ("slots", "heads"))
def test_attention_pages(hip, page, layout):
    c = attention_case(page, [70, 129, 3], [1, 66, 3], 4, 2, 128, "F32", "F16", page, layout=layout)
    check_attention(c, run_attention(hip, c))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (33, 0), (64, 64), (65, 70), (100, 3),
                                          (1000, 4), (0xFFFFFFFF, 0), (20, 0xFFFFFFFF)])
@pytest.mark.parametrize("gtype,cache,dim", [("F32", "F16", 64), ("BF16", "BF16", 128)])
def test_attention_window(hip, window, sinks, gtype, cache, dim):
    c = attention_case(5, [300, 90, 150, 20], [1, 90, 70, 2], 4, 2, dim, gtype, cache, 16)
    check_attention(c, run_attention(hip, c, window=window, sinks=sinks), window, sinks)


def test_attention_pages_that_are_not_there(hip):
    """Entries that name no page, inside and at both ends; a row with none left gives zeros."""
    for new in ([1, 1, 1], [70, 30, 20]):
        c = attention_case(6, [150, 90, 40], new, 8, 2, 128, "F32", "F16", 16)
        c["table"][0, 0], c["table"][0, 4], c["table"][0, 9] = P.NONE, c["pages"], 0x80000000
        c["table"][2] = P.NONE
        got = run_attention(hip, c)
        check_attention(c, got)
        assert torch.all(got[c["start"][2]:c["start"][3]] == 0)


@pytest.mark.parametrize("gtype,cache", [("F32", "F16"), ("BF16", "BF16")])
def test_attention_masked_values_do_not_matter(hip, gtype, cache):
    """NaN and infinities of later tokens, and of positions a window hides, stay out of the
    rows that do not see them."""
    c = attention_case(8, [100, 140], [60, 2], 4, 2, 128, gtype, cache, 16)
    def at(r, i):
        return int(c["table"][r, i // 16]), i % 16
    c["v"][at(0, 70)], c["k"][at(0, 80)] = float("nan"), float("inf")
    c["v"][at(0, 90)] = float("-inf")
    c["v"][at(1, 3)], c["k"][at(1, 4)] = float("inf"), float("nan")
    got = run_attention(hip, c, window=50)
    clean = {**c, "k": c["k"].nan_to_num(0, 0, 0), "v": c["v"].nan_to_num(0, 0, 0)}
    rows = list(range(30)) + [60, 61]  # positions 40 .. 69 of request 0, all of request 1
    assert torch.isfinite(got[rows].float()).all() and torch.isnan(got[31].float()).all()
    k, v = f64(clean["k"]), f64(clean["v"])
    want, bound = P.attention(f64(c["q"]), k, v, c["table"], c["start"], c["lens"], 16, 128 ** -0.5, 50, 0)
    tol = P.attention_tolerance(np.nan_to_num(want), bound, 128, gtype, cache)
    assert np.all(np.abs(f64(got) - want)[rows] <= tol[rows])


def test_attention_nan_that_rows_see_costs_no_more(hip):
    """A NaN key, value or query makes NaN of the rows that see it, and of no others, in the time
    that any values take."""
    import time
    c = attention_case(62, [4000, 4000], [4000, 1], 8, 2, 128, "BF16", "BF16", 16)
    run_attention(hip, c)
    def timed(case):
        run_attention(hip, case)
        t = time.perf_counter()
        out = run_attention(hip, case)
        return out, time.perf_counter() - t
    clean, plain = timed(c)
    def at(r, i):
        return int(c["table"][r, i // 16]), i % 16
    for name in ("k", "v"):
        bad = {**c, name: c[name].clone()}
        bad[name][at(0, 100)][0, 5] = float("nan")
        bad[name][at(1, 100)][1, 5] = float("nan")
        got, spent = timed(bad)
        nan = torch.isnan(got)
        seen = nan[100:4000, :4] if name == "k" else nan[100:4000, :4, 5]
        assert seen.all() and nan[4000, 4:, 5].all()
        nan[100:4000, :4] = False
        nan[4000, 4:] = False
        assert not nan.any() and torch.equal(got[:64], clean[:64]) and torch.equal(got[:100, 4:], clean[:100, 4:])
        # rows of the tile that holds the NaN without seeing it are done again by themselves, with
        # unrounded weights: half a step of BF16 of max |v| (2^-12 more for FP32's sums), and
        # each side's own rounding
        off = (got[64:100, :4].float() - clean[64:100, :4].float()).abs()
        vmax = c["v"][torch.isfinite(c["v"])].abs().max().float()
        assert torch.all(off <= vmax * (2.0 ** -8 + 2.0 ** -12) + clean[64:100, :4].float().abs() * 2.0 ** -7)
        assert spent < 20 * plain + 0.05
    bad = {**c, "q": c["q"].clone()}
    bad["q"][77, 3, 9] = float("nan")
    got, spent = timed(bad)
    nan = torch.isnan(got)
    assert nan[77, 3].all() and nan.sum() == 128 and spent < 20 * plain + 0.05


@pytest.mark.parametrize("scale", (0.3, 1e-8))
def test_attention_scale_and_large_scores(hip, scale):
    c = attention_case(9, [90, 33], [30, 1], 4, 2, 64, "F32", "F16", 16)
    c["q"] *= 30
    check_attention(c, run_attention(hip, c, scale=scale), scale=scale)


def test_attention_lowest_scores(hip):
    """Scores near -1e4 everywhere: the maximum comes off before the exponential."""
    c = attention_case(10, [70], [3], 2, 1, 64, "F32", "F16", 16)
    k = c["k"]
    k[torch.isfinite(k)] = k[torch.isfinite(k)].abs() + 20
    c["q"] = -c["q"].abs() * 30 - 20
    check_attention(c, run_attention(hip, c))


def test_attention_leaves_requests_over_the_bound(hip):
    c = attention_case(11, [50, 40, 9], [1, 4, 2], 8, 2, 128, "F32", "F16", 16)
    got = run_attention(hip, c, max_new=3)
    assert torch.all(got[1:5] == 5.0)
    alone = run_attention(hip, c)
    assert torch.equal(got[5:7], alone[5:7]) and torch.equal(got[:1], alone[:1])


def test_attention_strided_rows(hip):
    """q and out inside wider rows."""
    c = attention_case(12, [60, 20], [20, 1], 4, 2, 64, "F16", "F16", 16)
    wide = torch.randn(c["rows"], 4 * 64 + 24, device="cuda").to(torch.float16)
    out = torch.full((c["rows"], 4 * 64 + 40), 5.0, dtype=torch.float16, device="cuda")
    wide[:, 8:8 + 256] = c["q"].view(c["rows"], 256)
    call = attention_call(c, out)
    call.desc.q, call.desc.q_stride = wide[:, 8:].data_ptr(), wide.stride(0)
    call.desc.out, call.desc.out_stride = out[:, 16:].data_ptr(), out.stride(0)
    hip.paged_attention_async(call)
    torch.cuda.synchronize()
    check_attention(c, out[:, 16:16 + 256].reshape(c["rows"], 4, 64))
    assert torch.all(out[:, :16] == 5.0) and torch.all(out[:, 16 + 256:] == 5.0)


@pytest.mark.parametrize("seed", range(6))
def test_attention_drawn(hip, seed):
    g = np.random.default_rng(seed)
    lens, new = P.ragged(g, int(g.integers(1, 12)), 300, [1, 4, 40][seed % 3])
    gtype, cache = TYPES[seed % 4]
    kvh = int(g.integers(1, 4))
    c = attention_case(seed, lens, new, kvh * int(g.integers(1, 10)), kvh, [64, 128, 256][seed % 3], gtype, cache,
                       [4, 16, 32][seed % 3])
    window, sinks = [(0, 0), (40, 2)][seed % 2]
    check_attention(c, run_attention(hip, c, window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("gtype,cache,dim", [("F32", "F16", 64), ("F16", "F16", 128), ("F32", "BF16", 128),
                                             ("BF16", "BF16", 256)])
@pytest.mark.parametrize("new", ([1, 1, 1], [40, 1, 3], [90, 130, 20]))
@pytest.mark.parametrize("window,sinks", [(0, 0), (3000, 5), (100, 2500)])
def test_attention_long_contexts(hip, gtype, cache, dim, new, window, sinks):
    """Rows whose keys are spread over several workgroups and joined."""
    c = attention_case(dim + sum(new), [9001, 700, 5003], new, 4, 2, dim, gtype, cache, 16, width_more=900)
    check_attention(c, run_attention(hip, c, window=window, sinks=sinks), window, sinks)


def test_attention_masked_values_in_long_contexts(hip):
    """A later token's NaN and infinity, in the part of the keys that holds the rows themselves."""
    for new in ([4, 1], [60, 1]):
        c = attention_case(31, [6000, 100], new, 8, 2, 128, "F32", "F16", 16)
        page = int(c["table"][0, 5999 // 16])
        c["v"][page, 5999 % 16], c["v"][page, 5998 % 16, 0, 3] = float("nan"), float("inf")
        got = run_attention(hip, c)
        clean = {**c, "v": c["v"].nan_to_num(0, 0, 0)}
        ref = run_attention(hip, clean)
        n = new[0]
        want, bound = P.attention(f64(c["q"]), f64(clean["k"]), f64(clean["v"]), c["table"], c["start"], c["lens"],
                                  16, 128 ** -0.5, 0, 0)
        tol = P.attention_tolerance(np.nan_to_num(want), bound, 128, "F32", "F16")
        rows = list(range(n - 2)) + [n]
        assert np.all(np.abs(f64(got) - want)[rows] <= tol[rows])
        assert torch.isnan(got[n - 1]).all() and torch.all(got[n - 2, :4, 3] == float("inf"))
        assert torch.equal(got[n - 2, 4:], ref[n - 2, 4:]) or np.all(
            np.abs(f64(got) - want)[n - 2, 4:] <= tol[n - 2, 4:])


@pytest.mark.parametrize("requests", (65, 200, 1030))
def test_attention_many_requests(hip, requests):
    g = np.random.default_rng(requests)
    lens, new = P.ragged(g, requests, 90, 2)
    lens[7], new[7] = 400, 70
    c = attention_case(requests, lens, new, 2, 1, 64, "F16", "F16", 8)
    check_attention(c, run_attention(hip, c))


@pytest.mark.parametrize("requests", (64, 192, 193, 256, 1030, 4096, 4097, 8192))
def test_attention_requests_beyond_a_wave(hip, requests):
    """Where every wave finds its piece by itself and where a launch before leaves the sums:
    rows long enough to be cut, requests without a row in between."""
    g = np.random.default_rng(requests)
    lens, new = P.ragged(g, requests, 90 if requests < 2000 else 12, 2)
    lens[7], new[7] = 400, 70
    lens[-1], new[-1], lens[-3], new[-3] = 6000, 1, 3000, 33
    new[10:40] = [0] * 30
    c = attention_case(requests, lens, new, 2, 1, 64, "F16", "F16", 8)
    check_attention(c, run_attention(hip, c))


@pytest.mark.parametrize("requests", (6, 300))
def test_attention_starts_that_decrease(hip, requests):
    """A query_start that decreases: more rows than max_tokens, so that not all of the work
    has a workgroup.  What the rows get is not said; nothing beyond max_tokens is written,
    and the next call is right."""
    c = attention_case(20, [6000] * requests if requests < 10 else [700] * requests, [6] * requests, 4, 2, 64, "F16",
                       "F16", 64)
    rows = 30
    assert rows < c["q"].shape[0]
    for start in ([0] + [rows, 3] * (requests // 2), [0, 25] * (requests // 2) + [7],
                  [rows - 1, rows] * (requests // 2) + [2]):
        out = torch.full_like(c["q"], 5.0)
        hip.paged_attention_async(attention_call(dict(c, start=np.array(start), rows=rows), out))
        torch.cuda.synchronize()
        assert torch.all(out[rows:] == 5.0)
    check_attention(c, run_attention(hip, c))


@pytest.mark.parametrize("gtype,cache", TYPES)
def test_attention_smallest_scale(hip, gtype, cache):
    """The smallest positive scale: all scores are alike, masked ones still have no weight."""
    c = attention_case(21, [5, 70, 300], [5, 40, 1], 4, 2, 64, gtype, cache, 16)
    check_attention(c, run_attention(hip, c, scale=1e-45), scale=1e-45)


def test_attention_order_does_not_change_bits(hip):
    c = attention_case(13, [3000, 700], [1, 1], 8, 2, 128, "F32", "F16", 16)
    first = run_attention(hip, c)
    for _ in range(3):
        assert torch.equal(first, run_attention(hip, c))


# ---- together -------------------------------------------------------------------------

def test_steps_together_in_a_graph(hip):
    """Plan, append and attention of one layer over several steps, requests ending and
    others taking their rows, as one captured graph: each step against numpy."""
    g = np.random.default_rng(3)
    heads, kvh, dim, page, pages, requests, rows, width = 4, 2, 64, 8, 24, 3, 24, 12
    table = np.full((requests, width), P.NONE, np.uint32)
    order = g.permutation(pages)
    stack, count, lens = order.astype(np.uint32).copy(), pages, [0] * requests
    p = Plan(page, pages, rows, lens, [0] * requests, table, stack, count, [0] * requests, alias=True)
    kc, vc = (torch.zeros(pages, page, kvh, dim, dtype=torch.float16, device="cuda") for _ in range(2))
    qkv = torch.zeros(rows, (heads + 2 * kvh) * dim, device="cuda")
    turned, out = (torch.zeros(rows, heads * dim, device="cuda") for _ in range(2))
    w = (1 + 0.1 * torch.randn(dim)).cuda()
    kv = PagedKV(kc.data_ptr(), vc.data_ptr(), 1, pages, page, kvh, dim)
    append = PagedAppend(kv, 0, rows, heads, q=qkv.data_ptr(), k=qkv[:, heads * dim:].data_ptr(),
                         v=qkv[:, (heads + kvh) * dim:].data_ptr(), q_out=turned.data_ptr(),
                         slots=p.slots.data_ptr(), q_stride=qkv.stride(0), k_stride=qkv.stride(0),
                         v_stride=qkv.stride(0), q_norm=w.data_ptr(), k_norm=w.data_ptr(), rms_eps=1e-6,
                         rope_theta=1e4, rotary_dim=dim, positions=p.positions.data_ptr())
    attend = PagedAttention(kv, 0, heads, requests, rows, q=turned.data_ptr(), out=out.data_ptr(),
                            query_start=p.start.data_ptr(), lens=p.lens_out.data_ptr(),
                            block_table=p.table.data_ptr(), table_stride=width)
    stream = torch.cuda.Stream()

    def enqueue(s):
        hip.paged_plan_async(p.call, s)
        hip.paged_append_async(append, s)
        hip.paged_attention_async(attend, s)
    torch.cuda.synchronize()
    enqueue(stream.cuda_stream)  # no tokens: sizes the scratch
    hip.sync(stream.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        enqueue(torch.cuda.current_stream().cuda_stream)
    history = [[] for _ in range(requests)]  # float16 K and V rows per request
    steps = [([9, 5, 0], [0, 0, 0]), ([1, 1, 13], [0, 0, 0]), ([1, 7, 1], [0, 1, 0]), ([0, 1, 1], [0, 0, 0]),
             ([12, 1, 0], [1, 0, 1])]
    for new, release in steps:
        x = torch.randn(rows, qkv.shape[1])
        qkv.copy_(x)
        p.new.copy_(ints(new))
        p.release.copy_(ints(release))
        out.fill_(5.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        bits, want = P.plan(page, pages, rows, lens, new, release, table, stack, count)
        assert bits == 0
        same_plan(p.outputs(), want)
        lens, table, stack, count = want["lens"], want["table"], want["stack"], want["count"]
        x = x.numpy().astype(np.float64)
        t = 0
        for r in range(requests):
            if release[r]:
                history[r] = []
            for j in range(new[r]):
                pos = np.array([[len(history[r])]])
                row = x[t].reshape(-1, dim)[None]
                turn = P.heads(row[:, :heads + kvh], f64(w), 1e-6, pos, [0] * (dim // 2), 1e4, dim)[0]
                history[r].append((turn[heads:], row[0, heads + kvh:]))
                keys = np.array([h[0] for h in history[r]])
                values = np.array([h[1] for h in history[r]])
                for h in range(heads):
                    s = keys[:, h // 2] @ turn[h] * dim ** -0.5
                    e = np.exp(s - s.max())
                    o = (e / e.sum()) @ values[:, h // 2]
                    # K and V are held in F16: half a step of K's values moves a score by at
                    # most 2^-11 scale sum |q k|, and V's the result by 2^-11 max |v|
                    move = np.max(np.abs(keys[:, h // 2] * turn[h]).sum(-1)) * dim ** -0.5 * 2.0 ** -11
                    tol = np.abs(values[:, h // 2]).max() * (2 * move + 2.0 ** -11 + 2.0 ** -12)
                    got = f64(out[t].view(heads, dim)[h])
                    assert np.max(np.abs(got - o)) <= tol, (r, j, h)
                t += 1
        assert torch.all(out[t:] == 5.0)


def test_attention_replayed_with_other_lengths(hip):
    """A captured call of long contexts, replayed with other lengths, values and eager calls of
    other shapes in between: each replay against a fresh eager call."""
    cases = [attention_case(40 + i, lens, new, 8, 2, 128, "F32", "F16", 16, width_more=700 - max(lens) // 16)
             for i, (lens, new) in enumerate((([9000, 40, 700], [1, 30, 2]), ([33, 10900, 1], [33, 1, 1]),
                                              ([1, 64, 8000], [0, 1, 34]), ([9000, 5000, 7000], [1, 1, 1])))]
    pages, rows = max(c["pages"] for c in cases), max(c["rows"] for c in cases)
    width = max(c["table"].shape[1] for c in cases)
    one = {**cases[0], "pages": pages, "rows": rows, "table": np.full((3, width), P.NONE, np.uint32),
           "k": torch.zeros(pages, 16, 2, 128, dtype=torch.float16, device="cuda"),
           "v": torch.zeros(pages, 16, 2, 128, dtype=torch.float16, device="cuda"),
           "q": torch.zeros(rows, 8, 128, device="cuda")}
    out = torch.zeros_like(one["q"])
    call = attention_call(one, out)
    lens, start, table = call.held
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    hip.paged_attention_async(call, stream.cuda_stream)  # sizes the scratch
    hip.sync(stream.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        hip.paged_attention_async(call, torch.cuda.current_stream().cuda_stream)
    other = attention_case(50, [5000, 6000], [1, 60], 4, 1, 64, "F16", "F16", 8)
    for c in cases + cases[:2]:
        one["k"][:c["pages"]], one["v"][:c["pages"]], one["q"][:c["rows"]] = c["k"], c["v"], c["q"]
        lens.copy_(ints(c["lens"]))
        start.copy_(ints(c["start"]))
        full = np.full((3, width), P.NONE, np.uint32)
        full[:, :c["table"].shape[1]] = c["table"]
        table.copy_(ints(full))
        out.fill_(5.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check_attention(c, out[:c["rows"]].contiguous())
        assert torch.all(out[c["rows"]:] == 5.0)
        run_attention(hip, other)


def test_capture_refuses_scratch_growth(hip):
    """A fresh context's first call under capture would need scratch: refused, and the context
    still works."""
    from pokitlms_amd.backend import HipBackend
    c = attention_case(60, [9000, 300], [1, 2], 4, 2, 64, "F16", "F16", 16)
    want = run_attention(hip, c)
    with HipBackend(0) as fresh:
        out = torch.full_like(c["q"], 5.0)
        call = attention_call(c, out)
        stream, refused = torch.cuda.Stream(), None
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            try:
                fresh.paged_attention_async(call, torch.cuda.current_stream().cuda_stream)
            except ValueError as e:
                refused = str(e)
        assert refused is not None and "outside stream capture" in refused
        fresh.paged_attention_async(call, stream.cuda_stream)
        fresh.sync(stream.cuda_stream)
        assert torch.equal(out, want)


def test_offsets_beyond_32_bits(hip):
    """A cache of 9 GB whose pages lie 128 KB apart, K and V of a page side by side."""
    pages, stride, page, kvh, dim = 70000, 1 << 16, 16, 2, 128
    pool = torch.empty(pages * stride, dtype=torch.float16, device="cuda")
    assert pages * stride > 1 << 32
    g = np.random.default_rng(1)
    table = np.full((2, 8), P.NONE, np.uint32)
    table[0, :6], table[1, :2] = [69999, 3, 66000, 65537, 69990, 32769], [68001, 1]
    lens, new = [90, 20], [25, 1]
    for rows in (new, [1, 20]):
        tokens = sum(rows)
        qkv = torch.randn(sum(lens), 2 * kvh * dim, device="cuda", dtype=torch.float16)
        slots = np.concatenate([table[r, np.arange(n) // page].astype(np.int64) * page + np.arange(n) % page
                                for r, n in enumerate(lens)])
        kv = PagedKV(pool.data_ptr(), pool.data_ptr() + stride, 1, pages, page, kvh, dim, stride, kvh * dim, dim)
        at = ints(slots)
        hip.paged_append_async(PagedAppend(kv, 1, len(slots), 0, k=qkv.data_ptr(), v=qkv[:, kvh * dim:].data_ptr(),
                                           k_stride=2 * kvh * dim, v_stride=2 * kvh * dim, slots=at.data_ptr()))
        q = torch.randn(tokens, 4, dim, device="cuda", dtype=torch.float16)
        out = torch.full_like(q, 5.0)
        ln, st, tb = ints(lens), ints(np.concatenate([[0], np.cumsum(rows)])), ints(table)
        hip.paged_attention_async(PagedAttention(kv, 1, 4, 2, tokens, q=q.data_ptr(), out=out.data_ptr(),
                                                 query_start=st.data_ptr(), lens=ln.data_ptr(),
                                                 block_table=tb.data_ptr(), table_stride=8))
        torch.cuda.synchronize()
        small = {int(p): i for i, p in enumerate(np.unique(table[table != P.NONE]))}
        k, v = np.zeros((len(small), page, kvh, dim)), np.zeros((len(small), page, kvh, dim))
        x = f64(qkv)
        for i, s in enumerate(slots):
            k[small[int(s) // page], s % page] = x[i, :kvh * dim].reshape(kvh, dim)
            v[small[int(s) // page], s % page] = x[i, kvh * dim:].reshape(kvh, dim)
        near = np.vectorize(lambda p: small.get(int(p), P.NONE))(table).astype(np.uint32)
        want, bound = P.attention(f64(q), k, v, near, np.concatenate([[0], np.cumsum(rows)]), lens, page,
                                  dim ** -0.5, 0, 0)
        tol = P.attention_tolerance(want, bound, dim, "F16", "F16")
        assert np.all(np.abs(f64(out) - want) <= tol)


def test_lengths_past_the_table_count_as_its_end(hip):
    c = attention_case(61, [64, 30], [5, 1], 4, 2, 64, "F16", "F16", 16, width_more=0)
    want = run_attention(hip, c)
    got = run_attention(hip, {**c, "lens": [0xFFFFFFFF, 30]})
    assert torch.equal(got, want)


def test_two_contexts_on_two_streams(hip):
    """The same work in flight on two contexts' streams at once."""
    from pokitlms_amd.backend import HipBackend
    cases = [attention_case(20 + i, [2500, 90, 1300], [1, 30, 2], 8, 2, 128, "F32", "F16", 16) for i in range(2)]
    want = [run_attention(hip, c) for c in cases]
    with HipBackend(0) as other:
        streams = [torch.cuda.Stream() for _ in range(2)]
        outs = [torch.full_like(c["q"], 5.0) for c in cases]
        calls = [attention_call(c, o) for c, o in zip(cases, outs)]
        torch.cuda.synchronize()
        for _ in range(8):
            for backend, call, s in zip((hip, other), calls, streams):
                backend.paged_attention_async(call, s.cuda_stream)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_calls_are_counted_and_timed(hip):
    c = attention_case(30, [20], [1], 4, 2, 64, "F32", "F16", 16)
    before = hip.stats()
    hip.set_kernel_timing(True)
    try:
        run_attention(hip, c)
    finally:
        hip.set_kernel_timing(False)
    after = hip.stats()
    assert after["paged_attention_calls"] == before["paged_attention_calls"] + 1
    assert after["paged_attention_ns"] > before["paged_attention_ns"]


def test_refusals_of_two_threads_keep_their_texts(hip):
    """Calls of two threads at once: each raises its own refusal."""
    kv = PagedKV(1 << 20, 1 << 20, 1, 4, 16, 1, 64)
    calls = {"out may not be q": PagedAttention(kv, 1, 1, 1, 1, q=4096, out=4096, query_start=64, lens=64,
                                                block_table=64, table_stride=1),
             "requests must be between": PagedAttention(kv, 1, 1, 0, 1, q=4096, out=8192, query_start=64, lens=64,
                                                        block_table=64, table_stride=1)}
    wrong = []

    def run(text):
        for _ in range(2000):
            try:
                hip.paged_attention_async(calls[text])
                wrong.append("no refusal")
            except ValueError as e:
                if text not in str(e):
                    wrong.append(str(e))
    threads = [threading.Thread(target=run, args=(text,)) for text in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
