"""The paged-cache operators: what is measured, and each in its plain form.

Several requests share one pool of pages per layer.  Three operators, in the
order in which a step takes them:

* ``plan``: from each request's cached and new lengths, the pages that its new
  tokens need (popped from a free stack, after finished requests' pages went
  back on it), and per new token its position, slot and request;
* ``append``: per new token the q and k head norms, rotary positions with one or
  several axes, and K and V into the pages at the token's slot;
* ``attention``: the new tokens' attention over their requests' pages, causal,
  optionally with a sliding window and first tokens that stay visible.

With ``own`` false they run as elementary torch operations in 32 bits (angles in
64), else through ``HipBackend``.  A case's lengths come from the case alone
("ragged" seeds them), so that its work is known; values and page order come
from the seed.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16}
GGUF = {"F32": 0, "F16": 1, "BF16": 30}
SIZE = {"F32": 4, "F16": 2, "BF16": 2}
EPS, THETA = 1e-6, 1e6
NONE = -1  # no page, no slot, no request (0xffffffff on the C side)


# ---- the cases ------------------------------------------------------------------------

def listed():
    return [
        # a decode step of eight requests in the model's 512-position window: latency alone
        {"name": "plan_decode", "kind": "plan", "requests": 8, "page": 16, "context": 512,
         "new": 1, "chunks": 0, "finished": 0, "ragged": 1},
        # a serving step: most requests decode, some bring a chunk of their prompt, some end
        {"name": "plan_mixed", "kind": "plan", "requests": 96, "page": 32, "context": 8192,
         "new": 512, "chunks": 12, "finished": 5, "ragged": 2},
        # an offline batch's prompts all at once
        {"name": "plan_prompts", "kind": "plan", "requests": 1024, "page": 16, "context": 2048,
         "new": 128, "chunks": 1024, "finished": 0, "ragged": 3},
        # the model's own shape and types, one token for each of eight requests
        {"name": "append_decode", "kind": "append", "type": "F32", "cache": "F16", "heads": 32,
         "kv_heads": 4, "dim": 128, "rotary": 128, "axes": 1, "norm": True, "tokens": 8, "rows": 8,
         "page": 16, "far": 512},
        # an image's tokens among text: time, height and width; two rows of padding
        {"name": "append_axes", "kind": "append", "type": "F16", "cache": "F16", "heads": 32,
         "kv_heads": 4, "dim": 128, "rotary": 128, "axes": 3, "norm": True, "tokens": 1021,
         "rows": 1023, "page": 32, "far": 32768},
        # long prompts, 64 of 256 dimensions rotated, no norms
        {"name": "append_prompts", "kind": "append", "type": "BF16", "cache": "BF16", "heads": 16,
         "kv_heads": 2, "dim": 256, "rotary": 64, "axes": 1, "norm": False, "tokens": 16384,
         "rows": 16384, "page": 64, "far": 262144},
        # one decode step of eight requests within the model's 512-position window
        {"name": "attend_decode", "kind": "attention", "type": "F32", "cache": "F16", "heads": 32,
         "kv_heads": 4, "dim": 128, "requests": 8, "page": 16, "context": 512, "new": 1,
         "chunks": 0, "window": 0, "sinks": 0, "ragged": 4},
        # a full server's decode step, contexts from a few hundred positions to 8192
        {"name": "attend_batch", "kind": "attention", "type": "BF16", "cache": "BF16", "heads": 32,
         "kv_heads": 4, "dim": 128, "requests": 64, "page": 16, "context": 8192, "new": 1,
         "chunks": 0, "window": 0, "sinks": 0, "ragged": 5},
        # one request far into a long document
        {"name": "attend_long", "kind": "attention", "type": "F16", "cache": "F16", "heads": 32,
         "kv_heads": 4, "dim": 128, "requests": 1, "page": 64, "context": 131072, "new": 1,
         "chunks": 0, "window": 0, "sinks": 0, "ragged": 6},
        # decoding requests and chunks of prompts in one call
        {"name": "attend_mixed", "kind": "attention", "type": "BF16", "cache": "BF16", "heads": 32,
         "kv_heads": 4, "dim": 128, "requests": 24, "page": 32, "context": 8192, "new": 512,
         "chunks": 6, "window": 0, "sinks": 0, "ragged": 7},
        # a window of 1024 with four first tokens; pages behind the window are gone
        {"name": "attend_window", "kind": "attention", "type": "F32", "cache": "F16", "heads": 8,
         "kv_heads": 2, "dim": 64, "requests": 16, "page": 16, "context": 16384, "new": 256,
         "chunks": 8, "window": 1024, "sinks": 4, "ragged": 8},
        # a prompt of 8192 tokens from nothing
        {"name": "attend_prompt", "kind": "attention", "type": "BF16", "cache": "BF16", "heads": 32,
         "kv_heads": 4, "dim": 128, "requests": 1, "page": 64, "context": 8192, "new": 8192,
         "chunks": 1, "window": 0, "sinks": 0, "ragged": 9},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(32, 4), (32, 4), (16, 2), (8, 2), (4, 4), (6, 2), (16, 1), (8, 8), (28, 4), (12, 1)]
PAIRS = [("F32", "F16"), ("F16", "F16"), ("BF16", "BF16"), ("F32", "BF16")]


def draw(rng):
    kind = rng.choice(["plan", "append", "attention", "attention"])
    page = rng.choice([8, 16, 16, 32, 64, 128, 256])
    if kind == "plan":
        requests = _log_int(rng, 1, 1024)
        return {"kind": kind, "requests": requests, "page": page,
                "context": _log_int(rng, 16, 16384 if requests < 256 else 2048),
                "new": _log_int(rng, 1, 128), "chunks": rng.randint(0, requests),
                "finished": rng.randint(0, requests // 4), "ragged": rng.randrange(1 << 20)}
    heads, kv_heads = rng.choice(HEADS)
    dim = rng.choice([64, 128, 128, 256])
    gtype, cache = rng.choice(PAIRS)
    if kind == "append":
        tokens = _log_int(rng, 1, 6000)
        return {"kind": kind, "type": gtype, "cache": cache, "heads": heads, "kv_heads": kv_heads,
                "dim": dim, "rotary": rng.choice([dim, dim, dim // 2, dim // 4, 0]),
                "axes": rng.choice([1, 1, 3]), "norm": rng.random() < 0.7, "tokens": tokens,
                "rows": tokens + rng.choice([0, 0, 1, 7]), "page": page,
                "far": _log_int(rng, 64, 1 << 20)}
    requests = _log_int(rng, 1, 64)
    context = _log_int(rng, 1, min(65536, 262144 // requests))
    chunks = rng.choice([0, 0, rng.randint(1, requests)])
    # requests times rows times keys: far below the largest listed case's
    most = max(1, min(context, 1 << 12, (1 << 25) // (context * requests * max(1, heads // 16))))
    return {"kind": kind, "type": gtype, "cache": cache, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "requests": requests, "page": page, "context": context,
            "new": _log_int(rng, 1, most) if chunks else rng.choice([1, 1, 1, min(2, context)]),
            "chunks": chunks, "window": rng.choice([0, 0, 0, _log_int(rng, 1, 4096)]),
            "sinks": rng.choice([0, 4, rng.randint(1, 80)]), "ragged": rng.randrange(1 << 20)}


# ---- lengths: of the case alone -------------------------------------------------------

def _lengths(case):
    """Per request the positions after the step and the new ones among them: the first
    reaches the case's context, the others spread over its logarithm; `chunks` requests
    bring up to `new` tokens, the others decode one (up to `new`, without chunks)."""
    g = np.random.RandomState(case["ragged"])
    n, context = case["requests"], case["context"]
    lens = np.exp(g.uniform(math.log(max(1, context // 32)), math.log(context + 1), n)).astype(np.int64)
    lens = np.clip(lens, 1, context)
    lens[0] = context
    new = np.full(n, min(case["new"], context) if not case["chunks"] else 1, np.int64)
    if case["chunks"]:
        who = g.permutation(n)[:case["chunks"]]
        new[who] = np.maximum(1, (case["new"] * g.uniform(0.5, 1.0, len(who))).astype(np.int64))
        new[who[0]] = case["new"]
    return lens, np.minimum(new, lens)


def _pages(n, page):
    return -(-n // page)


def _window(case, lens, new):
    """Per request the first position its new rows see behind the sinks."""
    if not case["window"]:
        return np.zeros_like(lens)
    return np.maximum(0, lens - new + 1 - case["window"])


def work(case):
    if case["kind"] == "plan":
        lens, new, finished = _plan_lengths(case)
        need = _pages(lens + new, case["page"]) - _pages(lens, case["page"])
        old = int(np.sum((lens % case["page"] > 0) & (new > 0)))
        gone = int(_pages(finished, case["page"]).sum())
        return {"bytes": 4.0 * (4 * len(lens) + 2 * int(need.sum()) + old + 3 * int(new.sum()) + 2 * gone),
                "flops": 0.0}
    size, csize, dim = SIZE[case["type"]], SIZE[case["cache"]], case["dim"]
    if case["kind"] == "append":
        t, q, kv = case["tokens"], case["heads"] * dim, case["kv_heads"] * dim
        per = (2 * q + 2 * kv) * size + 2 * kv * csize + 4 * case["axes"] + 4
        return {"bytes": float(t * per), "flops": float(t * (q + kv) * 10)}
    lens, new = _lengths(case)
    first = _window(case, lens, new)
    seen = lens - first + np.minimum(first, case["sinks"])
    rows = int(new.sum())
    keys = 0
    for n, m in zip(lens.tolist(), new.tolist()):
        p = np.arange(n - m, n)
        lo = np.maximum(0, p + 1 - case["window"]) if case["window"] else np.zeros_like(p)
        keys += int(np.sum(p + 1 - lo + np.minimum(lo, case["sinks"])))
    table = int(_pages(seen, case["page"]).sum()) * 4
    return {"bytes": float(int(seen.sum()) * case["kv_heads"] * dim * 2 * csize +
                           2 * rows * case["heads"] * dim * size + table),
            "flops": 4.0 * keys * case["heads"] * dim}


# ---- inputs ---------------------------------------------------------------------------

class _State:
    def __init__(self, **kw):
        self.call = None
        self.__dict__.update(kw)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _plan_lengths(case):
    """Cached lengths (0 for finished requests), new ones, and the finished ones' lengths."""
    after, new = _lengths(case)
    lens, done = after - new, np.zeros_like(after)
    if case["finished"]:
        who = np.random.RandomState(case["ragged"] + 1).permutation(len(after))[:case["finished"]]
        done[who] = lens[who]
        lens[who] = 0
        new[who] = 0
    return lens, new, done


def _prepare_plan(case, seed):
    g, page, n = _gen(seed), case["page"], case["requests"]
    lens, new, done = _plan_lengths(case)
    held, width = lens + done, int(_pages(case["context"], page)) + 1
    used = _pages(held, page)
    need = int((_pages(lens + new, page) - _pages(lens, page)).sum())
    free = need + 3 + need // 8
    pages = int(used.sum()) + free
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    col = torch.arange(width, device="cuda")
    use, at = torch.from_numpy(used).cuda(), torch.from_numpy(np.cumsum(used) - used).cuda()
    table = torch.where(col < use[:, None], order[(at[:, None] + col).clamp(max=pages - 1)], NONE)
    stack = torch.full((pages,), NONE, dtype=torch.int32, device="cuda")
    stack[:free] = order[int(used.sum()):]
    rows = int(new.sum()) + 5  # a step's buffers are seldom full
    def empty(*shape):
        return torch.zeros(shape, dtype=torch.int32, device="cuda")
    return _State(case=case, pages=pages, page=page, rows=rows, lens=_ints(held), new=_ints(new),
                  release=_ints(done > 0) if case["finished"] else None, table=table.to(torch.int32).contiguous(),
                  stack=stack, count=_ints([free]), lens_out=empty(n), count_out=empty(1),
                  start=empty(n + 1), positions=empty(rows), slots=empty(rows), owner=empty(rows),
                  status=empty(4))


def _normal(g, shape, dtype):
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def _axis_map(case):
    """Per pair its axis: a quarter of the pairs time, the rest height and width by turns."""
    pairs = case["rotary"] // 2
    if case["axes"] == 1:
        return [0] * pairs
    return [0 if i < pairs // 4 else 1 + (i - pairs // 4) % 2 for i in range(pairs)]


def _prepare_append(case, seed):
    g = _gen(seed)
    t, rows, dim, page = case["tokens"], case["rows"], case["dim"], case["page"]
    dtype, cache = TYPES[case["type"]], TYPES[case["cache"]]
    qd, kd = case["heads"] * dim, case["kv_heads"] * dim
    # projections' rows lie side by side, as one product gives them
    qkv = _normal(g, (rows, qd + 2 * kd), dtype)
    qkv[:, qd:qd + kd] *= 3
    pages = _pages(rows, page) + 2
    slots = torch.full((rows,), NONE, dtype=torch.int32, device="cuda")
    slots[:t] = torch.randperm(pages * page, device="cuda", generator=g)[:t].to(torch.int32)
    return _State(case=case, q=qkv[:, :qd], k=qkv[:, qd:qd + kd], v=qkv[:, qd + kd:], pages=pages,
                  q_out=_normal(g, (rows, qd), dtype), slots=slots,
                  q_norm=1 + 0.1 * torch.randn(dim, device="cuda", generator=g) if case["norm"] else None,
                  k_norm=1 + 0.1 * torch.randn(dim, device="cuda", generator=g) if case["norm"] else None,
                  positions=torch.randint(0, case["far"], (case["axes"], rows), device="cuda",
                                          generator=g).to(torch.int32), axis_map=_axis_map(case),
                  kcache=_normal(g, (pages, page, case["kv_heads"], dim), cache),
                  vcache=_normal(g, (pages, page, case["kv_heads"], dim), cache))


def _prepare_attention(case, seed):
    g, page, dim, kvh = _gen(seed), case["page"], case["dim"], case["kv_heads"]
    dtype, cache = TYPES[case["type"]], TYPES[case["cache"]]
    lens, new = _lengths(case)
    n, used, width = len(lens), _pages(lens, page), int(_pages(case["context"], page)) + 1
    pages = int(used.sum()) + 1
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    col = torch.arange(width, device="cuda")
    use, at = torch.from_numpy(used).cuda(), torch.from_numpy(np.cumsum(used) - used).cuda()
    there = col < use[:, None]
    if case["window"]:  # what neither the window nor the sinks see has been given back
        first = torch.from_numpy(_window(case, lens, new)).cuda()[:, None]
        there &= (col * page + page > first) | (col * page < case["sinks"])
    table = torch.where(there, order[(at[:, None] + col).clamp(max=pages - 1)], NONE).to(torch.int32)
    rows = int(new.sum()) + 1
    start = np.concatenate([[0], np.cumsum(new)])
    # keys with a few wide channels, as rotated and normed keys have them
    k = torch.randn(pages, page, kvh, dim, device="cuda", generator=g)
    k[..., :: dim // 4] *= 4
    return _State(case=case, pages=pages, rows=rows, width=width, k=k.to(cache),
                  v=_normal(g, (pages, page, kvh, dim), cache), table=table.contiguous(),
                  lens=_ints(lens), start=_ints(start), most=int(new.max()), longest=int(lens.max()),
                  q=_normal(g, (rows, case["heads"], dim), dtype),
                  out=(0.01 * torch.randn(rows, case["heads"], dim, device="cuda", generator=g)).to(dtype))


_stream = None


def prepare(case, seed):
    global _stream
    if own:  # a program's torch work and the framework's calls share a stream of the program's:
        # torch's default one has handle 0, which names the framework's own
        if _stream is None:
            _stream = torch.cuda.Stream()
        torch.cuda.set_stream(_stream)
    return {"plan": _prepare_plan, "append": _prepare_append,
            "attention": _prepare_attention}[case["kind"]](case, seed)


# ---- the plain forms ------------------------------------------------------------------

def _plan_plain(s):
    page, stack = s.page, s.stack
    width, n = s.table.shape[1], len(s.lens)
    held, new, top = s.lens.long(), s.new.long(), s.count.long()
    release = s.release.bool() if s.release is not None else torch.zeros_like(held, dtype=torch.bool)
    col = torch.arange(width, device="cuda")
    # finished requests' pages go on the stack in request and table order
    back = release[:, None] & (col < ((held + page - 1) // page)[:, None]) & (s.table != NONE)
    order = torch.cumsum(back.reshape(-1), 0)
    place = torch.where(back.reshape(-1), top + order - 1, len(stack))
    stack = torch.cat([stack, stack[:1]]).scatter(0, place, s.table.reshape(-1))[:-1]
    top, lens = top + order[-1:], torch.where(release, 0, held)
    # pages for the new tokens, from the top down
    have, after = (lens + page - 1) // page, (lens + new + page - 1) // page
    need = after - have
    first = torch.cumsum(need, 0) - need
    fresh = (col >= have[:, None]) & (col < after[:, None])
    take = (top - 1 - (first[:, None] + col - have[:, None])).clamp(0, len(stack) - 1)
    table = torch.where(fresh, stack[take], s.table)
    # tokens
    start = torch.cat([torch.zeros_like(top), torch.cumsum(new, 0)])
    t = torch.arange(s.rows, device="cuda")
    live = t < start[-1]
    owner = torch.searchsorted(start, t, right=True).clamp(max=n) - 1
    position = lens[owner] + t - start[owner]
    slots = table[owner, (position // page).clamp(max=width - 1)].long() * page + position % page
    def kept(x, other):
        return torch.where(live, x, other).int()
    status = torch.cat([torch.zeros_like(top), start[-1:], need.sum().view(1), order[-1:]])
    return {"table": table, "stack": stack, "count": (top - need.sum()).int(), "lens": (lens + new).int(),
            "start": start.int(), "positions": kept(position, 0), "slots": kept(slots, NONE),
            "owner": kept(owner, NONE), "status": status.int()}


def _rotated(x, weight, cos, sin, rotary):
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    a, b, rest = x[..., :rotary // 2], x[..., rotary // 2:rotary], x[..., rotary:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _append_plain(s):
    c = s.case
    t, dim, rotary = c["rows"], c["dim"], c["rotary"]
    pair = torch.arange(rotary // 2, device="cuda", dtype=torch.float64)
    axis = torch.tensor(s.axis_map, dtype=torch.long, device="cuda")
    angle = s.positions[axis].T.double() * THETA ** (-2 * pair / max(1, rotary))
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    live = s.slots >= 0
    q = _rotated(s.q.reshape(t, -1, dim).float(), s.q_norm, cos, sin, rotary).reshape(t, -1)
    k = _rotated(s.k.reshape(t, -1, dim).float(), s.k_norm, cos, sin, rotary)
    s.q_out.copy_(torch.where(live[:, None], q.to(s.q_out.dtype), s.q_out))
    at = s.slots[live].long()
    s.kcache.view(-1, c["kv_heads"], dim)[at] = k[live].to(s.kcache.dtype)
    s.vcache.view(-1, c["kv_heads"], dim)[at] = s.v.reshape(t, -1, dim)[live].float().to(s.vcache.dtype)
    return {"q": s.q_out, "k": s.kcache, "v": s.vcache}


def _attention_plain(s):
    c = s.case
    page, dim, kvh = c["page"], c["dim"], c["kv_heads"]
    n, m, longest = c["requests"], s.most, s.longest
    start, lens = s.start.long(), s.lens.long()
    new = start[1:] - start[:-1]
    i = torch.arange(longest, device="cuda")
    entry = s.table[:, i // page].long()
    slot = entry.clamp(min=0) * page + i % page                            # [n, longest]
    there = (entry >= 0) & (i < lens[:, None])
    k = s.k.view(-1, kvh, dim)[slot].float().permute(0, 2, 3, 1).contiguous()   # [n, kvh, dim, longest]
    v = s.v.view(-1, kvh, dim)[slot].float().permute(0, 2, 1, 3).contiguous()
    j = torch.arange(m, device="cuda")
    row = (start[:-1, None] + j).clamp(max=s.rows - 1)
    p = lens[:, None] - new[:, None] + j                                   # [n, m]
    seen = there[:, None] & (i <= p[..., None])
    if c["window"]:
        seen = seen & ((i + c["window"] > p[..., None]) | (i < c["sinks"]))
    q = s.q[row].float().view(n, m, kvh, -1, dim).permute(0, 2, 3, 1, 4)   # [n, kvh, G, m, dim]
    scores = torch.matmul(q.reshape(n, kvh, -1, dim), k).view(n, kvh, -1, m, longest) * dim ** -0.5
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = scores.sub_(top.masked_fill(top == -math.inf, 0)).exp_()
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(n, kvh, -1, longest), v).view(n, kvh, -1, m, dim)
    o = torch.where(total > 0, o / total, 0).permute(0, 3, 1, 2, 4).reshape(n, m, -1, dim)
    live = j < new[:, None]
    s.out[row[live]] = o[live].to(s.out.dtype)
    return s.out


# ---- the framework's calls ------------------------------------------------------------

_backend = None


def _hip():
    global _backend
    if _backend is None:
        from pokitlms_amd.backend import HipBackend
        _backend = HipBackend(0)
    return _backend


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _own_plan(s):
    from pokitlms_amd.backend import PagedPlan
    return _hip().paged_plan_async, PagedPlan(
        requests=len(s.lens), pages=s.pages, page_size=s.page, table_stride=s.table.shape[1],
        max_tokens=s.rows, lens=_ptr(s.lens), new_lens=_ptr(s.new), release=_ptr(s.release),
        block_table=_ptr(s.table), free_pages=_ptr(s.stack), free_count=_ptr(s.count),
        lens_out=_ptr(s.lens_out), free_count_out=_ptr(s.count_out), query_start=_ptr(s.start),
        positions=_ptr(s.positions), slots=_ptr(s.slots), token_request=_ptr(s.owner),
        status=_ptr(s.status)), {
            "table": s.table, "stack": s.stack, "count": s.count_out, "lens": s.lens_out,
            "start": s.start, "positions": s.positions, "slots": s.slots, "owner": s.owner,
            "status": s.status}


def _cache(c, k, v, pages):
    from pokitlms_amd.backend import PagedKV
    return PagedKV(k=_ptr(k), v=_ptr(v), gtype=GGUF[c["cache"]], pages=pages, page_size=c["page"],
                   kv_heads=c["kv_heads"], head_dim=c["dim"])


def _own_append(s):
    from pokitlms_amd.backend import PagedAppend
    c = s.case
    stride = s.q.stride(0)
    return _hip().paged_append_async, PagedAppend(
        _cache(c, s.kcache, s.vcache, s.pages), gtype=GGUF[c["type"]], tokens=c["rows"],
        heads=c["heads"], q=_ptr(s.q), k=_ptr(s.k), v=_ptr(s.v), q_out=_ptr(s.q_out),
        slots=_ptr(s.slots), q_stride=stride, k_stride=stride, v_stride=stride,
        q_norm=_ptr(s.q_norm), k_norm=_ptr(s.k_norm), rms_eps=EPS, rope_theta=THETA,
        rotary_dim=c["rotary"], positions=_ptr(s.positions), axes=c["axes"],
        position_stride=c["rows"], pair_axis=s.axis_map), {"q": s.q_out, "k": s.kcache, "v": s.vcache}


def _own_attention(s):
    from pokitlms_amd.backend import PagedAttention
    c = s.case
    return _hip().paged_attention_async, PagedAttention(
        _cache(c, s.k, s.v, s.pages), gtype=GGUF[c["type"]], heads=c["heads"], requests=c["requests"],
        max_tokens=s.rows, max_new=s.most, q=_ptr(s.q), out=_ptr(s.out), query_start=_ptr(s.start),
        lens=_ptr(s.lens), block_table=_ptr(s.table), table_stride=s.width, window=c["window"],
        sinks=c["sinks"]), s.out


def run(state):
    kind = state.case["kind"]
    if not own:
        return {"plan": _plan_plain, "append": _append_plain, "attention": _attention_plain}[kind](state)
    if state.call is None:  # the descriptor of a step's buffers, which a program makes once
        state.call = {"plan": _own_plan, "append": _own_append, "attention": _own_attention}[kind](state)
    enqueue, what, outputs = state.call
    enqueue(what, torch.cuda.current_stream().cuda_stream)
    return outputs


# ---- the definitions in 64 bits -------------------------------------------------------

def _exact_append(case, seed):
    s = _prepare_append(case, seed)
    dim, rotary = case["dim"], case["rotary"]
    q_out, kc, vc = s.q_out.double(), s.kcache.double(), s.vcache.double()
    live = torch.nonzero(s.slots >= 0).view(-1)
    page, slot = s.slots[live].long() // case["page"], s.slots[live].long() % case["page"]
    turn = torch.ones(len(live), dim // 2, dtype=torch.complex128, device="cuda")
    for i, axis in enumerate(s.axis_map):
        angle = s.positions[axis][live].double() * math.exp(-math.log(THETA) * 2 * i / rotary)
        turn[:, i] = torch.complex(torch.cos(angle), torch.sin(angle))

    def head(x, weight):
        x = x.double()
        if weight is not None:
            x = x / torch.sqrt(torch.sum(x * x, -1, keepdim=True) / dim + EPS) * weight.double()
        half = rotary // 2
        if half:
            z = torch.complex(x[:, :half], x[:, half:rotary]) * turn[:, :half]
            x = torch.cat([z.real, z.imag, x[:, rotary:]], 1)
        return x

    for h in range(case["heads"]):
        q_out[live, h * dim:(h + 1) * dim] = head(s.q[live, h * dim:(h + 1) * dim], s.q_norm)
    for h in range(case["kv_heads"]):
        kc[page, slot, h] = head(s.k[live, h * dim:(h + 1) * dim], s.k_norm)
        vc[page, slot, h] = s.v[live, h * dim:(h + 1) * dim].double()
    return {"q": q_out, "k": kc, "v": vc}


def _exact_attention(case, seed):
    s = _prepare_attention(case, seed)
    page, dim, group = case["page"], case["dim"], case["heads"] // case["kv_heads"]
    lens, new = _lengths(case)
    out, at = s.out.double(), 0
    for r in range(case["requests"]):
        n, m = int(lens[r]), int(new[r])
        where = torch.arange(n, device="cuda")
        pages = s.table[r, :-(-n // page)].long().repeat_interleave(page)[:n]
        where = where[pages >= 0]
        pages = pages[pages >= 0]
        keys, values = s.k[pages, where % page].double(), s.v[pages, where % page].double()
        for j0 in range(0, m, 1024):  # rows at a time: long prompts' weights are large
            rows = torch.arange(j0, min(m, j0 + 1024), device="cuda")
            p = (n - m + rows)[:, None]
            hidden = where[None] > p
            if case["window"]:
                hidden |= (where[None] <= p - case["window"]) & (where[None] >= case["sinks"])
            for h in range(case["heads"]):
                logit = s.q[at + rows, h].double() @ keys[:, h // group].T / math.sqrt(dim)
                weight = torch.softmax(logit.masked_fill(hidden, -math.inf), -1)
                out[at + rows, h] = weight @ values[:, h // group]
        at += m
    return out


def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers
    return (_exact_append if case["kind"] == "append" else _exact_attention)(case, seed)
