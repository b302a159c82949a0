"""The choice of experts for more tokens than one launch has threads for, on the GPU: every token's own gate, and the plan."""

import numpy as np
import pytest

import i8_oracle as ref
from test_gpu_mx4 import Out

pytestmark = pytest.mark.gpu


def test_more_tokens_than_a_launch_takes(device, mc):
    tokens = (1 << 28) + 37
    # One expert; bf16 logits between -2 and 2, other ones for the tokens a launch further on.
    t = np.arange(tokens, dtype=np.uint32)
    bits = ((t * np.uint32(2654435761)) >> np.uint32(16)).astype(np.uint16) & np.uint16(0xBFFF)
    del t
    x = mc.DeviceBuffer.from_array(bits)
    chosen, gates, order = (Out(mc, tokens * 4) for _ in range(3))
    offsets = Out(mc, 8)
    space = mc.DeviceBuffer(mc.route_workspace_bytes(tokens, 1, 1))
    mc.launch_route(ref.BF16, x.ptr, 1, None, tokens, 1, 1, "sigmoid", 1, 1, 1, False, 2.5, chosen.ptr, gates.ptr, order.ptr,
                    offsets.ptr, None, space.ptr)
    mc.synchronize()
    assert not chosen.get(np.int32, tokens).any()
    every = 2.5 / (1.0 + np.exp(-ref.from_type(np.arange(0xC000, dtype=np.uint16) & np.uint16(0xBFFF), ref.BF16)))
    got = gates.get(np.float32, tokens)
    for at in range(0, tokens, 1 << 24):  # one rounding to fp32, and float64's own
        want = every[bits[at:at + (1 << 24)]]
        assert np.all(np.abs(got[at:at + (1 << 24)] - want) <= (2.0 ** -24 + 2.0 ** -42) * want), at
    assert np.array_equal(order.get(np.int32, tokens), np.arange(tokens, dtype=np.int32))
    assert np.array_equal(offsets.get(np.int32, 2), [0, tokens])
