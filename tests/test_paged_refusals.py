"""What the paged-cache entry points refuse.  The arguments are checked before the context
is used, so a call without one names what is wrong with the rest."""
import ctypes

import pytest

from pokitlms_amd import _abi
from pokitlms_amd.backend import PagedAppend, PagedAttention, PagedKV, PagedPlan, rotary_axes

P = 0x10000  # an address that no call gets to use
OK = "context is required"


def call(name, desc):
    err = ctypes.create_string_buffer(256)
    status = getattr(_abi.lib(), name)(None, ctypes.byref(desc), None, err, 256)
    return status, err.value.decode()


def cache(**kw):
    args = dict(k=P, v=P, gtype=1, pages=8, page_size=16, kv_heads=2, head_dim=128)
    args.update(kw)
    return PagedKV(**args)


def plan(**kw):
    args = dict(requests=4, pages=8, page_size=16, table_stride=4, max_tokens=32, lens=P, new_lens=P + 4,
                block_table=P + 8, free_pages=P + 12, free_count=P + 16, lens_out=P, free_count_out=P + 16,
                query_start=P + 20, positions=P, slots=P, token_request=P, status=P)
    args.update(kw)
    return PagedPlan(**args).desc


def append(kv=None, **kw):
    args = dict(gtype=0, tokens=4, heads=8, q=P, k=P, v=P, q_out=P, slots=P, q_norm=P, k_norm=P,
                rms_eps=1e-6, rope_theta=1e4, rotary_dim=128, positions=P)
    args.update(kw)
    return PagedAppend(kv or cache(), **args).desc


def attention(kv=None, **kw):
    args = dict(gtype=1, heads=8, requests=4, max_tokens=32, q=P, out=2 * P, query_start=P, lens=P,
                block_table=P, table_stride=4)
    args.update(kw)
    return PagedAttention(kv or cache(), **args).desc


CACHES = [(dict(k=0), 1, "k and v"), (dict(v=P + 8), 1, "16-byte"), (dict(gtype=0), 5, "F16 or BF16"),
          (dict(gtype=8), 5, "F16 or BF16"), (dict(head_dim=96), 5, "head_dim"), (dict(pages=0), 1, "slots"),
          (dict(pages=1 << 27), 1, "slots"), (dict(page_size=24), 1, "power of two"),
          (dict(page_size=0), 1, "power of two"), (dict(page_size=2048), 1, "power of two"),
          (dict(kv_heads=0), 1, "kv_heads"), (dict(page_stride=4096, slot_stride=256, head_stride=124), 1, "multiples of 8"),
          (dict(page_stride=4096, slot_stride=256, head_stride=64), 1, "shorter"),
          (dict(page_stride=4096, slot_stride=0, head_stride=128), 1, "shorter"),
          (dict(page_stride=1 << 50, slot_stride=256, head_stride=128), 1, "range")]


@pytest.mark.parametrize("bad,status,text", CACHES)
def test_cache(bad, status, text):
    for name, desc in (("append", append), ("attention", attention)):
        got = call(f"pk_hip_paged_{name}_async", desc(cache(**bad)))
        assert got[0] == status and text in got[1], got


@pytest.mark.parametrize("good", [{}, dict(page_size=1), dict(page_size=1024), dict(gtype=30),
                                  dict(head_dim=64), dict(head_dim=256),
                                  dict(page_stride=128 * 32, slot_stride=128, head_stride=128 * 16)])
def test_caches_that_hold(good):
    for name, desc in (("append", append), ("attention", attention)):
        kw = {"rotary_dim": 64} if name == "append" else {"gtype": good.get("gtype", 1)}
        got = call(f"pk_hip_paged_{name}_async", desc(cache(**good), **kw))
        assert got[0] == 1 and OK in got[1], got


PLANS = [(dict(requests=0), "requests"), (dict(requests=8193), "requests"), (dict(pages=0), "slots"),
         (dict(page_size=3), "power of two"), (dict(table_stride=0), "positions"),
         (dict(table_stride=1 << 27), "positions"), (dict(max_tokens=0), "max_tokens"),
         (dict(max_tokens=(1 << 24) + 1), "max_tokens"), (dict(status=0), "buffers"),
         (dict(block_table=P + 2), "4-byte"), (dict(release=P + 1), "4-byte"),
         (dict(lens_out=P + 4), "outputs"), (dict(query_start=P), "outputs")]


@pytest.mark.parametrize("bad,text", PLANS)
def test_plan(bad, text):
    got = call("pk_hip_paged_plan_async", plan(**bad))
    assert got[0] == 1 and text in got[1], got


APPENDS = [(dict(gtype=8), 5, "rows are"), (dict(tokens=0), 1, "tokens"), (dict(tokens=(1 << 24) + 1), 1, "tokens"),
           (dict(heads=5000), 1, "heads"), (dict(q=0), 1, "required"), (dict(k=0), 1, "required"),
           (dict(slots=0), 1, "required"), (dict(q=P + 8), 1, "16-byte"), (dict(slots=P + 2), 1, "4-byte"),
           (dict(q_stride=1020), 1, "shorter"), (dict(q_stride=1026), 1, "16 bytes"),
           (dict(gtype=1, q_stride=1028), 1, "16 bytes"), (dict(q_stride=2048), 1, "q's stride"),
           (dict(rms_eps=0.0), 1, "epsilon"), (dict(rotary_dim=24), 1, "rotary_dim"),
           (dict(rotary_dim=144), 1, "rotary_dim"), (dict(positions=0), 1, "positions"), (dict(axes=0), 1, "axes"),
           (dict(axes=5), 1, "axes"), (dict(rope_theta=0.0), 1, "RoPE"), (dict(position_stride=3), 1, "position_stride"),
           (dict(axes=2, pair_axis=[2] * 64), 1, "pair_axis")]


@pytest.mark.parametrize("bad,status,text", APPENDS)
def test_append(bad, status, text):
    got = call("pk_hip_paged_append_async", append(**bad))
    assert got[0] == status and text in got[1], got


def test_appends_that_hold():
    for good in ({}, dict(heads=0, q=0, q_out=0), dict(rotary_dim=0, positions=0, rope_theta=0.0),
                 dict(q_norm=0, k_norm=0, rms_eps=0.0), dict(q_stride=1536, q_out_stride=1536),
                 dict(axes=3, pair_axis=rotary_axes((16, 24, 24)))):
        got = call("pk_hip_paged_append_async", append(**good))
        assert got[0] == 1 and OK in got[1], (good, got)


ATTENTIONS = [(dict(gtype=30), 5, "cache's type"), (dict(gtype=12), 5, "cache's type"), (dict(heads=0), 1, "heads"),
              (dict(heads=7), 1, "evenly"), (dict(requests=0), 1, "requests"), (dict(max_tokens=0), 1, "max_tokens"),
              (dict(q=0), 1, "required"), (dict(out=0), 1, "required"), (dict(q=P + 4), 1, "16-byte"),
              (dict(lens=P + 1), 1, "4-byte"), (dict(out=P), 1, "out may not be q"),
              (dict(scale=-1.0), 1, "scale"), (dict(scale=float("nan")), 1, "scale"),
              (dict(scale=float("inf")), 1, "scale"), (dict(table_stride=1 << 28), 1, "positions"),
              (dict(q_stride=1000), 1, "shorter"), (dict(out_stride=1028), 1, "16 bytes")]


@pytest.mark.parametrize("bad,status,text", ATTENTIONS)
def test_attention(bad, status, text):
    got = call("pk_hip_paged_attention_async", attention(**bad))
    assert got[0] == status and text in got[1], got


def test_null_descriptors():
    for name in ("plan", "append", "attention"):
        err = ctypes.create_string_buffer(64)
        assert getattr(_abi.lib(), f"pk_hip_paged_{name}_async")(None, None, None, err, 64) == 1
        assert b"is required" in err.value


def test_rotary_axes():
    assert rotary_axes((2, 3, 1)) == [0, 0, 1, 1, 1, 2]
    assert rotary_axes((4, 2, 2), interleaved=True) == [0, 1, 2, 0, 1, 2, 0, 0]
    assert rotary_axes((24, 20, 20), interleaved=True).count(0) == 24
    for bad in (((), False), ((3, -1), False), ((0, 4, 4), True)):
        with pytest.raises(ValueError):
            rotary_axes(*bad)
    with pytest.raises(ValueError):
        PagedAppend(cache(), 0, 4, 8, k=P, v=P, slots=P, rotary_dim=128, pair_axis=[0] * 63)
