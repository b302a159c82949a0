"""The choice of experts where masks leave little, on the GPU against float64 as include/minicompiler_hip.h states it:
groups with one expert left or none, of every size."""

import numpy as np
import pytest

import i8_oracle as ref
from test_gpu_route import run

pytestmark = pytest.mark.gpu


def scores(logits, score):
    """float64, 0 where masked out; NaN where a softmax meets +infinity."""
    if score == "sigmoid":
        with np.errstate(over="ignore"):
            return 1.0 / (1.0 + np.exp(-logits))
    with np.errstate(invalid="ignore"):
        top = logits.max()
        e = np.exp(logits - top) if top > -np.inf else np.zeros_like(logits)
        return e / e.sum() if top > -np.inf else e


def choose(logits, bias, top_k, score, groups, top_groups, group_best, normalize):
    """(experts, gates) of one token's logits (float64)."""
    s = scores(logits, score)
    alone = bias is None and (groups == 1 or group_best == 1)
    key = [-np.inf if l == -np.inf else l if alone else x + (0.0 if bias is None else float(b))
           for l, x, b in zip(logits, s, logits if bias is None else bias)]
    key = [-np.inf if np.isnan(x) else x for x in key]
    each = len(key) // groups
    rank = []
    for g in range(groups):
        there = sorted((x for x in key[g * each:(g + 1) * each] if x > -np.inf), reverse=True)[:group_best]
        rank.append((not there, -sum(there), g))
    kept = {g for _, _, g in sorted(rank)[:top_groups]}
    chosen = sorted((e for e in range(len(key)) if e // each in kept), key=lambda e: (-key[e], e))[:top_k]
    gates = s[chosen]
    if normalize:
        total = gates.sum()
        gates = np.zeros(top_k) if total == 0 else gates / total
    if score == "softmax" and np.any(logits == np.inf):
        gates = np.full(top_k, np.nan)
    return chosen, gates


def check(mc, logits, kind, bias, top_k, score, groups, top_groups, group_best, normalize=True):
    dtype = ref.TYPES[kind]
    bits = ref.to_type(logits, dtype)
    args = (top_k, score, groups, top_groups, group_best, normalize)
    want = [choose(row, bias, *args) for row in ref.from_type(bits, dtype)]
    chosen, gates, order, offsets = run(mc, bits, dtype, bias, *args)
    assert np.array_equal(chosen, [w[0] for w in want])
    # One rounding to fp32; in float64 some 2^-52 for each of a few hundred sums and an exponential before it.
    wanted = np.array([w[1] for w in want])
    off = np.abs(gates - wanted)
    assert np.all((off <= (2.0 ** -24 + 2.0 ** -42) * np.abs(wanted) + 2.0 ** -150) | (np.isnan(gates) & np.isnan(wanted)))
    plan = ref.plan(chosen, logits.shape[1])
    assert np.array_equal(order, plan[0]) and np.array_equal(offsets, plan[1])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_a_group_with_one_expert_left_is_above_one_with_none(device, mc, score):
    inf = np.inf
    one = np.array([[-inf, -inf, 2.0, -inf], [-inf, -inf, -inf, -3.0], [-inf, 0.0, -inf, -inf], [-inf] * 4])
    check(mc, one, "f32", None, 1, score, 2, 1, 2)
    # One of each two masked out: the scores of what is left decide.
    two = np.array([[-inf, 0.0, -inf, 1.0, -inf, 2.0, -inf, 9.0], [5.0, -inf, -inf, 1.0, -inf, 2.0, 4.0, -inf]])
    for top_groups in (1, 2, 3):
        check(mc, two, "f32", None, 1, score, 4, top_groups, 2)


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("experts,groups", [(8, 4), (6, 2), (128, 64), (63, 21), (256, 8), (512, 64)])
def test_groups_of_which_masks_leave_little(device, mc, kind, score, biased, experts, groups):
    print(f"case masked groups {kind} {score} {biased} {experts}/{groups}", flush=True)
    rng = np.random.default_rng(experts + groups)
    tokens, each = 60, experts // groups
    logits = rng.standard_normal((tokens, experts)) * 2
    logits[rng.random(logits.shape) < 0.6] = -np.inf
    for t in range(0, tokens, 3):  # exactly one expert of each group
        left = np.arange(groups) * each + rng.integers(0, each, groups)
        masked = np.full(experts, -np.inf)
        masked[left] = rng.standard_normal(groups)
        logits[t] = masked
    logits[1] = -np.inf
    logits[2, each:] = -np.inf
    # Below -1 too: what is left of a group may score less than nothing.
    bias = (rng.standard_normal(experts) * 1.5).astype(np.float32) if biased else None
    for best in (1, 2):
        for top_groups in (1, groups // 2):
            check(mc, logits, kind, bias, min(2, each * top_groups), score, groups, top_groups, best)
