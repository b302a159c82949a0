"""A softmax over a logit of +infinity on the GPU: no gate of that token is a number, whichever experts are chosen, and
other tokens' are as without it."""

import numpy as np
import pytest

import i8_oracle as ref
from test_gpu_route import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups,top_groups,best", [(1, 1, 1), (4, 2, 1), (4, 2, 2)])
def test_softmax_of_infinity_has_no_gates(device, mc, kind, normalize, biased, groups, top_groups, best):
    rng = np.random.default_rng(3)
    dtype, tokens, experts, top_k = ref.TYPES[kind], 40, 64, 4
    bias = (rng.standard_normal(experts) * 0.1).astype(np.float32) if biased else None
    logits = rng.standard_normal((tokens, experts))
    args = (top_k, "softmax", groups, top_groups, best, normalize)
    plain = run(mc, ref.to_type(logits, dtype), dtype, bias, *args)
    at = rng.integers(0, experts, tokens)  # first and last experts among them, the chosen and others
    at[:3] = 0, experts - 1, experts // 2
    lost = np.arange(tokens) % 4 < 3
    logits[lost, at[lost]] = np.inf
    logits[5, :] = np.inf
    logits[6, 1:] = -np.inf
    logits[6, 0] = np.inf
    got = run(mc, ref.to_type(logits, dtype), dtype, bias, *args)
    assert np.all(np.isnan(got[1][lost]))
    assert np.array_equal(got[0][~lost], plain[0][~lost]) and np.array_equal(got[1][~lost], plain[1][~lost])
    assert np.all((got[0] >= 0) & (got[0] < experts))
    assert all(len(set(row)) == top_k for row in got[0])  # experts of their own all the same
    plan = ref.plan(got[0], experts)
    assert np.array_equal(got[2], plan[0]) and np.array_equal(got[3], plan[1])
