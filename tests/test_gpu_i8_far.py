"""The experts' first product with 2 GiB of tokens and more on the GPU: rows gathered from below and past 2^31 bytes against
float64, every form of its kernel, experts without tokens and with few."""

import numpy as np
import pytest

import i8_oracle as ref
from test_gpu_i8 import compare, operand, random_operand
from test_gpu_mx4 import Out, bits_type

pytestmark = pytest.mark.gpu

TOKENS, EXPERTS, TOP_K, K, FAR = (1 << 19) + 77, 6, 1, 4096, 5


@pytest.fixture(scope="module")
def far(mc):
    """Tokens [rows, K] on the host and on the GPU, and a plan of them: one expert with two tokens, one with none, one with
    the last of its tile in a half."""
    rng = np.random.default_rng(31)
    x = np.frombuffer(rng.bytes(TOKENS * K), dtype=np.int8).reshape(TOKENS, K)
    sx = (rng.uniform(0.5, 2.0, TOKENS) / 127 / np.sqrt(K)).astype(np.float32)
    chosen = rng.choice([0, 1, 4, 5], TOKENS).astype(np.int32)
    chosen[[5, TOKENS - 1]] = 3  # of expert 3 the only ones, 2^31 bytes apart
    order, offsets = ref.plan(chosen[:, None], EXPERTS)
    return x, sx, operand(mc, x, sx), order, offsets


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("n", [264, 258])
@pytest.mark.parametrize("act", ["gelu", "swiglu"])
def test_up_of_tokens_past_2_gib(device, mc, far, kind, n, act):
    print(f"case far {kind} {n} {act}", flush=True)
    x, sx, dx, order, offsets = far
    rng = np.random.default_rng(n)
    dtype = ref.TYPES[kind]
    n = n // 2 if act == "swiglu" else n
    rows = 2 * n if act == "swiglu" else n
    assert mc.library().mchip_experts_i8_plan(0, 2 if act == "swiglu" else 1, TOKENS, TOP_K, EXPERTS, n, K,
                                              device["cu_count"]) == FAR
    w, sw = random_operand(rng, EXPERTS * rows, K)
    sw *= np.float32(4.0)
    b = rng.standard_normal((EXPERTS, rows)).astype(np.float32)
    dw, db, do, df = operand(mc, w, sw), *(mc.DeviceBuffer.from_array(v) for v in (b, order, offsets))
    c = Out(mc, TOKENS * n * (4 if dtype == ref.F32 else 2))
    mc.launch_experts_up_i8(dx[0].ptr, dx[1].ptr, dw[0].ptr, dw[1].ptr, db.ptr, act, dtype, c.ptr, do.ptr, df.ptr, TOKENS,
                            TOP_K, EXPERTS, n, K)
    mc.synchronize()
    got = c.get(bits_type(dtype), (TOKENS, n))
    w, sw = w.reshape(EXPERTS, rows, -1), sw.reshape(EXPERTS, rows)
    for e in range(EXPERTS):
        first, end = offsets[e], offsets[e + 1]
        # Both ends of the expert's slots, and some between them.
        slots = np.unique(np.r_[first:min(first + 300, end), max(end - 300, first):end, rng.integers(first, max(end, first + 1), 200)])
        slots = slots[(slots >= first) & (slots < end)]
        t = order[slots] // TOP_K
        want, err = ref.activate(*ref.scaled(x[t], sx[t], w[e], sw[e], b[e]), act)
        compare(got[slots], want, ref.rounded(want, err, dtype), dtype)
