"""Calls of the paged-cache entry points at the ends of their sizes, without a context: what is
too large for a launch is refused beforehand, as not covered."""
import pytest

from tests.test_paged_refusals import OK, P, attention, cache, call


@pytest.mark.parametrize("kw,kv", [
    # one 16-row tile per request and KV head, 2^25 of them
    (dict(requests=8192, max_tokens=8192, heads=4096), dict(kv_heads=4096, head_dim=64)),
    # 128-row tiles of 2^24 tokens
    (dict(requests=1024, max_tokens=1 << 24, heads=127), dict(kv_heads=127, head_dim=64))])
def test_more_tiles_than_a_launch_holds(kw, kv):
    got = call("pk_hip_paged_attention_async", attention(cache(**kv), **kw))
    assert got[0] == 5 and "launch" in got[1], got


@pytest.mark.parametrize("kw,kv", [
    (dict(requests=8192, max_tokens=8192, heads=128), dict(kv_heads=128)),
    (dict(requests=8192, max_tokens=1 << 20, heads=1024), dict(kv_heads=8)),
    (dict(requests=1, max_tokens=1 << 24, heads=64), dict(kv_heads=64)),
    (dict(requests=1, max_tokens=1 << 24, heads=127, max_new=1), dict(kv_heads=127))])
def test_large_calls_that_a_launch_holds(kw, kv):
    got = call("pk_hip_paged_attention_async", attention(cache(**kv), **kw))
    assert got[0] == 1 and OK in got[1], got


@pytest.mark.parametrize("n_new", (-1, (1 << 32) + 1, [2, -3]))
def test_counts_of_a_batch_that_are_no_counts(n_new):
    """Refused before they are cut to 32 bits (no model is needed for that)."""
    from pokitlms_amd.model import Qwen3MoeModel
    with pytest.raises(ValueError, match="n_new"):
        object.__new__(Qwen3MoeModel).generate_batch([[1, 2], [3]], n_new)
