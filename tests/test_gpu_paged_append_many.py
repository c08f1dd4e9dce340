"""Appends of so many tokens that a workgroup takes four of them, and of just fewer."""
import numpy as np
import pytest

from tests.test_gpu_paged import append_case, check_append, f64, run_append

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", (4095, 4096, 4099))
@pytest.mark.parametrize("gtype,cache,heads,kvh,dim", [("F32", "F16", 4, 1, 64), ("F16", "F16", 3, 3, 128),
                                                       ("BF16", "BF16", 5, 1, 256), ("F32", "BF16", 2, 1, 128)])
def test_append(hip, tokens, gtype, cache, heads, kvh, dim):
    c = append_case(tokens + dim, tokens, heads, kvh, dim, gtype, cache, 16)
    before = np.full((c["rows"], c["qd"]), 3.0), f64(c["kc"]), f64(c["vc"])
    q, k, v, _ = run_append(hip, c)
    check_append(c, q, k, v, before)


@pytest.mark.parametrize("case", [dict(axes=3, rotary=128), dict(axes=4, rotary=64), dict(rotary=16), dict(rotary=0),
                                  dict(norm=False), dict(far=1 << 31, axes=2), dict(page=1), dict(layout="heads"),
                                  dict(layout="heads", pads=7, axes=3, rotary=96)], ids=str)
def test_append_forms(hip, case):
    args = dict(page=8, axes=1)
    args.update(case)
    c = append_case(7, 4101, 5, 2, 128, "F32", "F16", **args)
    before = np.full((c["rows"], c["qd"]), 3.0), f64(c["kc"]), f64(c["vc"])
    q, k, v, _ = run_append(hip, c)
    check_append(c, q, k, v, before)
