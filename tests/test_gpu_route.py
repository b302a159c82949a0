"""The choice of experts on the GPU against float64 numpy: choices and plans exactly, gates within one rounding to fp32
(and float64's own), at ties, masks, groups, NaNs and any number of tokens."""

import numpy as np
import pytest

import i8_oracle as ref
from test_gpu_mx4 import Out, device_rows

pytestmark = pytest.mark.gpu


def run(mc, bits, dtype, bias, top_k, score="softmax", groups=1, top_groups=1, group_best=1, normalize=True, scale=1.0,
        plan=True, pad=0, stream=None):
    tokens, experts = bits.shape
    x = device_rows(mc, bits, experts + pad)
    b = mc.DeviceBuffer.from_array(bias) if bias is not None else None
    chosen, gates = Out(mc, tokens * top_k * 4), Out(mc, tokens * top_k * 4)
    order, offsets = (Out(mc, tokens * top_k * 4), Out(mc, (experts + 1) * 4)) if plan else (None, None)
    space = mc.DeviceBuffer(max(256, mc.route_workspace_bytes(tokens, experts, top_k)))
    space.fill_bytes(0xCD)
    mc.synchronize()
    mc.launch_route(dtype, x.ptr, experts + pad, b.ptr if b else None, tokens, experts, top_k, score, groups, top_groups,
                    group_best, normalize, scale, chosen.ptr, gates.ptr, order.ptr if plan else None,
                    offsets.ptr if plan else None, stream, space.ptr)
    mc.synchronize()
    got = chosen.get(np.int32, (tokens, top_k)), gates.get(np.float32, (tokens, top_k))
    return (*got, order.get(np.int32, tokens * top_k), offsets.get(np.int32, experts + 1)) if plan else got


def check(mc, logits, kind, bias, top_k, score="softmax", groups=1, top_groups=1, group_best=1, normalize=True, scale=1.0,
          **kw):
    dtype = ref.TYPES[kind]
    bits = ref.to_type(logits, dtype)
    args = (top_k, score, groups, top_groups, group_best, normalize, scale)
    chosen, gates, _ = ref.route(ref.from_type(bits, dtype), bias, *args)
    got = run(mc, bits, dtype, bias, *args, **kw)
    assert np.array_equal(got[0], chosen)
    assert np.array_equal(np.isnan(got[1]), np.isnan(gates))
    # One rounding to fp32; in float64 some 2^-52 for each of a few hundred sums and an exponential before it.
    fine = ~np.isnan(gates)
    unit = 2.0 ** -24 + 2.0 ** -42
    assert np.all(np.abs(got[1] - gates)[fine] <= unit * np.abs(gates[fine]) + 2.0 ** -150)
    if len(got) == 4:
        order, offsets = ref.plan(chosen, logits.shape[1])
        assert np.array_equal(got[3], offsets) and np.array_equal(got[2], order)


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens,experts,top_k,pad", [(1, 1, 1, 0), (1, 64, 8, 0), (2, 5, 5, 3), (3, 60, 4, 0),
                                                      (7, 65, 6, 1), (64, 128, 16, 0), (65, 129, 8, 5), (100, 256, 8, 0),
                                                      (33, 257, 3, 0), (17, 512, 16, 0), (1000, 8, 2, 0),
                                                      (2500, 31, 4, 2)])
def test_choices(device, mc, kind, score, tokens, experts, top_k, pad):
    print(f"case route {kind} {score} {tokens}x{experts} top {top_k}", flush=True)
    rng = np.random.default_rng(tokens + experts)
    logits = rng.standard_normal((tokens, experts)) * 2
    bias = (rng.standard_normal(experts) * 0.1).astype(np.float32)
    check(mc, logits, kind, None, top_k, score, pad=pad)
    check(mc, logits, kind, bias, top_k, score, normalize=False, scale=2.5, pad=pad)


@pytest.mark.parametrize("best", [1, 2])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,top_groups,top_k", [(8, 2, 1, 4), (64, 8, 3, 8), (256, 8, 4, 8), (160, 8, 3, 6),
                                                             (64, 64, 5, 5), (217, 7, 2, 16), (512, 2, 1, 8),
                                                             (62, 31, 31, 9), (384, 4, 4, 8), (15, 5, 2, 6)])
def test_groups(device, mc, experts, groups, top_groups, top_k, score, biased, best):
    print(f"case groups {experts}/{groups} top {top_groups} {top_k} {score} {biased} {best}", flush=True)
    rng = np.random.default_rng(experts + groups)
    logits = rng.standard_normal((50, experts)) * 1.5
    bias = (rng.standard_normal(experts) * 0.1).astype(np.float32) if biased else None
    for kind in sorted(ref.TYPES):
        check(mc, logits, kind, bias, top_k, score, groups, top_groups, best, scale=1.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_ties_go_to_the_lower_expert(device, mc, score, groups):
    rng = np.random.default_rng(3)
    for experts in (8, 64, 132, 512):
        logits = rng.integers(-1, 2, (40, experts)).astype(np.float64)
        logits[0] = 0.0
        for bias in (None, np.zeros(experts, dtype=np.float32), rng.integers(0, 2, experts).astype(np.float32)):
            for best in (1, 2):
                check(mc, logits, "f32", bias, min(8, experts // groups), score, groups, min(2, groups), best)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_scores_next_to_each_other(device, mc, score):
    """Keys that differ in float64 and hardly, or not, in fp32."""
    rng = np.random.default_rng(4)
    experts = 96
    logits = np.float64(np.float32(0.7)) + rng.permutation(experts) * 2.0 ** -24
    logits = np.stack([rng.permutation(logits) for _ in range(30)])
    check(mc, logits, "f32", None, 8, score)
    check(mc, logits, "f32", np.full(experts, 0.25, dtype=np.float32), 8, score)
    # Past where a sigmoid is 1 in fp32.
    check(mc, 18.0 + 2.0 ** -6 * rng.permutation(experts)[None], "f32", np.zeros(experts, dtype=np.float32), 8, "sigmoid")


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 2])
@pytest.mark.parametrize("biased", [False, True])
def test_masks_infinities_and_nans(device, mc, kind, score, groups, biased):
    rng = np.random.default_rng(6)
    experts = 48
    logits = rng.standard_normal((12, experts))
    low = {"f32": -3.4e38, "bf16": -3.38e38, "f16": -65504.0}[kind]
    logits[0] = -np.inf                       # a token that nothing is left for
    logits[1, 3:] = -np.inf                   # fewer than it chooses
    logits[2, ::2] = -np.inf
    logits[3] = low
    logits[4, 5:] = low
    logits[5, 7] = np.nan
    logits[6] = np.nan
    logits[7, :24] = -np.inf                  # a whole group
    logits[8, 11] = 60000.0
    logits[9] *= 30
    logits[10, 4] = np.inf                    # by softmax: no gate is a number
    bias = (rng.standard_normal(experts) * 0.3).astype(np.float32) if biased else None
    with np.errstate(over="ignore"):
        for normalize in (False, True):
            check(mc, logits, kind, bias, 8, score, groups, 1, 2, normalize)
            check(mc, logits, kind, bias, 6, score, groups, groups, 1, normalize)


def test_biases_that_are_no_numbers(device, mc):
    rng = np.random.default_rng(8)
    logits = rng.standard_normal((9, 32))
    bias = rng.standard_normal(32).astype(np.float32)
    bias[3], bias[9], bias[17] = np.nan, np.inf, -np.inf
    check(mc, logits, "f32", bias, 6, "sigmoid")
    check(mc, logits, "f32", bias, 6, "sigmoid", 4, 3, 2)


@pytest.mark.parametrize("tokens,experts,top_k", [(1, 512, 1), (4097, 4, 4), (5000, 256, 8), (20000, 64, 2),
                                                  (9000, 384, 16)])
def test_plans_of_many_pairs(device, mc, tokens, experts, top_k):
    print(f"case plan {tokens}x{experts} top {top_k}", flush=True)
    rng = np.random.default_rng(tokens)
    # Some experts that nobody chooses, and one that most do.
    logits = rng.standard_normal((tokens, experts)) + rng.standard_normal(experts) * 2
    logits[:, experts // 2] += 6
    check(mc, logits, "bf16", None, top_k)


def test_without_a_plan_and_on_a_stream(device, mc):
    rng = np.random.default_rng(9)
    check(mc, rng.standard_normal((30, 40)), "f16", None, 4, plan=False, stream=mc.Stream())
