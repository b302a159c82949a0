"""The mixture-of-experts MLP on the GPU on values that its arithmetic has to keep: results worked out by hand, exact in
the result's type."""

import numpy as np
import pytest

import mx4_oracle as ref
from test_gpu_moe import run

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
