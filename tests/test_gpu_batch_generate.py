"""Many requests at once (pk_hip_qwen3moe_generate_batch) against each on its own."""
import numpy as np
import pytest

from pokitlms_amd import synth as S
from pokitlms_amd import synth_model as SM
from pokitlms_amd.backend import HipError, Unsupported
from tests.conftest import normwise_rel
from tests.test_gpu_prompt import shape

pytestmark = pytest.mark.gpu


def compare(hip, m, lengths, n_new, seed=31):
    """Tokens and logits of the batch are those of the reference-order model, one prompt at a
    time (the bound tests/test_gpu_prompt.py holds the fast mode's own prompts to)."""
    from pokitlms_amd.model import Qwen3MoeModel
    prompts = [SM.prompt_tokens(100 + i, n, m.vocab) for i, n in enumerate(lengths)]
    news = [n_new] * len(lengths) if np.ndim(n_new) == 0 else list(n_new)
    with Qwen3MoeModel.synthetic(hip, m, seed=seed, reference_order=True) as model:
        want = [model.generate(p, n, want_logits=True) for p, n in zip(prompts, news)]
    with Qwen3MoeModel.synthetic(hip, m, seed=seed, reference_order=False) as model:
        got, logits, stats = model.generate_batch(prompts, n_new, want_logits=True)
        again, _, _ = model.generate_batch(prompts, n_new)
    for i, (tokens, wl, _) in enumerate(want):
        assert normwise_rel(logits[i], wl) <= 1e-3, (i, lengths[i])
        assert np.array_equal(got[i], tokens[:news[i]]), (i, lengths[i])
        assert np.array_equal(got[i], again[i])
    assert stats["prompt_tokens"] == sum(lengths)
    assert stats["decode_forwards"] == sum(max(n - 1, 0) for n in news)


def test_one_request(hip):
    compare(hip, shape(), [70], 6)


def test_prompts_of_many_lengths(hip):
    compare(hip, shape(), [1, 5, 33, 130, 64, 17], 5)


def test_new_tokens_of_many_counts(hip):
    """Requests that end at different steps, one that wants logits alone."""
    compare(hip, shape(), [20, 3, 40, 9], [7, 1, 0, 12])


def test_more_rows_than_a_step_takes(hip):
    """Prompts over several steps beside requests that decode already; beyond the KV window."""
    compare(hip, shape(), [700, 30, 513], 4)


@pytest.mark.parametrize("kw", (dict(head_dim=128, heads=4, kv_heads=2, attn=S.Q6_K, gate=S.Q6_K, down=S.Q4_K),
                                dict(head_dim=256, heads=2, kv_heads=1, attn=S.Q5_K, gate=S.Q5_K, down=S.Q5_K),
                                dict(head_dim=128, heads=16, kv_heads=4)), ids=("planar", "q5k", "wide"))
def test_formats(hip, kw):
    compare(hip, shape(**kw), [40, 7, 90], 4)


def test_many_requests(hip):
    """More requests than slots of the block table: pages pass from one to the next."""
    from pokitlms_amd.model import Qwen3MoeModel
    m = shape()
    lengths = [1 + (7 * i) % 23 for i in range(300)]
    prompts = [SM.prompt_tokens(i % 9, n, m.vocab) for i, n in enumerate(lengths)]
    with Qwen3MoeModel.synthetic(hip, m, seed=31, reference_order=False) as model:
        got, _, _ = model.generate_batch(prompts, 3)
        for i in (0, 37, 150, 255, 256, 257, 299):
            alone, _, _ = model.generate(prompts[i], 3)
            assert np.array_equal(got[i], alone), i


def test_refusals(hip):
    from pokitlms_amd.model import Qwen3MoeModel
    m = shape()
    p = SM.prompt_tokens(1, 10, m.vocab)
    with Qwen3MoeModel.synthetic(hip, m, seed=31, reference_order=False) as model:
        for prompts, n in (([], 1), ([np.zeros(0, np.uint32)], 1), ([p, np.array([m.vocab])], 1), ([p], m.context)):
            with pytest.raises(ValueError):
                model.generate_batch(prompts, n)
        with pytest.raises(ValueError):
            model.generate_batch([p], [1, 2])
        assert len(model.generate_batch([p], 2)[0][0]) == 2  # and the model still works
    with Qwen3MoeModel.synthetic(hip, m, seed=31, reference_order=True) as model:
        with pytest.raises(Unsupported):
            model.generate_batch([p], 2)


def test_non_finite_prompt_is_an_error(hip):
    from pokitlms_amd.model import Qwen3MoeModel
    m = shape()
    weights = Qwen3MoeModel.synthetic_weights(hip, m, 31)
    bad = np.ones(m.hidden, np.float32)
    bad[7] = np.inf
    weights["blk.0.ffn_norm.weight"].release()
    weights["blk.0.ffn_norm.weight"] = hip.upload(S.F32, m.hidden, 1, bad)
    with Qwen3MoeModel(hip, m, weights, False) as model:
        with pytest.raises(HipError, match="non-finite"):
            model.generate_batch([SM.prompt_tokens(3, 40, m.vocab)], 2)
