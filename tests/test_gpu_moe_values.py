"""The mixture-of-experts MLP on the GPU on values that its arithmetic has to keep: results worked out by hand, exact in
the result's type."""

import numpy as np
import pytest

import mx4_oracle as ref
from test_gpu_moe import check, run

pytestmark = pytest.mark.gpu


def weights_of(mc, weights, *arrays):
    """The net of test_gpu_moe.run without biases, from W1 [experts, rows, d] and W2 [experts, d, h], exact in the type."""
    net = {"keep": [], "b1": None, "b2": None, "s1": None, "s2": None}
    for name, w in zip("12", arrays):
        if weights == ref.MX4:
            codes, scales, values = ref.quantize(w.reshape(-1, w.shape[2]))
            bufs = [mc.DeviceBuffer.from_array(codes), mc.DeviceBuffer.from_array(scales)]
            net["s" + name] = bufs[1].ptr
        else:
            bits = ref.to_type(w, weights)
            values = ref.from_type(bits, weights)
            bufs = [mc.DeviceBuffer.from_array(bits)]
        assert np.array_equal(values.reshape(w.shape), w)
        net["w" + name] = bufs[0].ptr
        net["keep"] += bufs
    return net


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("weights", [ref.BF16, ref.F16, ref.MX4])
@pytest.mark.parametrize("tokens", [1, 12])
@pytest.mark.parametrize("bits", [18, 21])
def test_hidden_activations_keep_the_bits_of_fp32(device, mc, kind, weights, tokens, bits):
    """h = 1 + 2^-8 + 2^-bits and 1 + 2^-8, which W2 takes from each other: every partial sum is exact in fp32, and so is
    the result, of any of the types. Blocks of mx4 rows hold one element each."""
    print(f"case moe hidden {kind} weights {weights} tokens {tokens} bits {bits}", flush=True)
    d, h = 96, 64
    x = np.zeros((tokens, d))
    x[:, [0, 32, 64]] = 1.0
    w1, w2 = np.zeros((1, h, d)), np.zeros((1, d, h))
    w1[0, 0, [0, 32, 64]] = 1.0, 2.0 ** -8, 2.0 ** -bits
    w1[0, 32, [0, 32]] = 1.0, 2.0 ** -8
    w2[0, 5, 0], w2[0, 5, 32] = 1.0, -1.0
    net = weights_of(mc, weights, w1, w2)
    router = np.zeros((1, d), dtype=np.float32)
    dtype = ref.TYPES[kind]
    y, chosen, gates = run(mc, net, ref.to_type(x, dtype), dtype, router, weights, h, 1, "relu", True)
    assert np.all(chosen == 0) and np.all(gates == 1.0)
    want = np.zeros((tokens, d))
    want[:, 5] = 2.0 ** -bits
    assert np.array_equal(y, want)


@pytest.mark.parametrize("weights", [ref.BF16, ref.F16, ref.MX4])
@pytest.mark.parametrize("tokens", [2, 12])
def test_an_infinite_hidden_activation(device, mc, weights, tokens):
    """Through weights of one piece an infinity is one of the sign of its weight; through fp16 weights, cut into two,
    the result is not finite."""
    print(f"case moe infinite h weights {weights} tokens {tokens}", flush=True)
    d, h = 40, 33
    sign = np.where(np.arange(d) % 3 == 0, -1.0, 1.0)
    net = weights_of(mc, weights, np.ones((1, h, d)), np.tile(sign.reshape(1, d, 1), (1, 1, h)))
    b1 = np.zeros((1, h), dtype=np.float32)
    b1[0, 30] = np.inf
    net["keep"].append(mc.DeviceBuffer.from_array(b1))
    net["b1"] = net["keep"][-1].ptr
    router = np.zeros((1, d), dtype=np.float32)
    y, _, _ = run(mc, net, np.ones((tokens, d), dtype=np.float32), ref.F32, router, weights, h, 1, "relu", True)
    if weights == ref.F16:
        assert not np.isfinite(y).any()
    else:
        assert np.array_equal(y, np.tile(np.inf * sign, (tokens, 1)))


@pytest.mark.parametrize("weights", [ref.BF16, ref.F16, ref.MX4])
@pytest.mark.parametrize("tokens", [2, 12])
def test_small_fp32_activations(device, mc, weights, tokens):
    """x and h of fp32: whole from 2^-110 up, below that the multiple of 2^-133 towards zero. W1 and W2 bring the token's
    number to its place, and 2^14 (of a type that has no more) up to where every fp32 holds the result."""
    print(f"case moe small x weights {weights} tokens {tokens}", flush=True)
    d = h = 32
    w1, w2 = np.zeros((1, h, d)), np.zeros((1, d, h))
    w1[0, 3, 7] = 1.0
    w2[0, 5, 3] = 2.0 ** 14
    net = weights_of(mc, weights, w1, w2)
    rng = np.random.default_rng(tokens)
    value = (rng.integers(1 << 23, 1 << 24, tokens) * 2.0 ** (-136 + np.arange(tokens))).astype(np.float32)
    x = np.zeros((tokens, d), dtype=np.float32)
    x[:, 7] = value
    router = np.zeros((1, d), dtype=np.float32)
    y, _, _ = run(mc, net, x, ref.F32, router, weights, h, 1, "relu", True)
    want = np.zeros((tokens, d))
    want[:, 5] = np.trunc(value.astype(np.float64) * 2.0 ** 133) * 2.0 ** -133 * 2.0 ** 14
    assert np.array_equal(y, want)


@pytest.mark.parametrize("weights", [ref.BF16, ref.F16, ref.MX4])
@pytest.mark.parametrize("tokens,d,h,experts,top_k,act", [
    (4, 64, 48, 300, 8, "swiglu"), (8, 40, 40, 512, 16, "gelu"), (1, 48, 32, 129, 3, "relu"),  # eight logits a lane, in moe_up
    (3, 4200, 40, 4, 2, "swiglu"), (20, 4200, 33, 5, 2, "gelu"),     # sums of nine parts of a logit
    (2, 9000, 24, 3, 1, "relu"), (12, 9001, 16, 3, 2, "swiglu")])    # d past 16 parts; column tiles of y past the CUs
def test_many_experts_and_long_rows(device, mc, weights, tokens, d, h, experts, top_k, act):
    print(f"case moe weights {weights} {tokens} {d} {h} {experts} {top_k} {act}", flush=True)
    for kind in ("f32", "f16"):
        check(mc, 5, kind, weights, tokens, d, h, experts, top_k, act, bias=experts % 2 == 1)


@pytest.mark.parametrize("weights", [ref.BF16, ref.F16])
@pytest.mark.parametrize("act", ["relu", "gelu", "swiglu"])
def test_odd_rows_of_every_type(device, mc, weights, act):
    print(f"case moe odd rows weights {weights} {act}", flush=True)
    for kind in sorted(ref.TYPES):
        check(mc, 6, kind, weights, 11, 133, 61, 5, 2, act)
