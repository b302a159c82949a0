"""Products of 8-bit integer operands whose scales lie far apart, on the GPU: a power of two moved from one operand's scales
to the other's changes no bit of the result, wherever a partial product would have left fp32's range; and results past that
range are infinities, with zeros where the sum is zero."""

import numpy as np
import pytest

import i8_oracle as ref
from test_gpu_experts_i8 import at, random_plan, upload
from test_gpu_i8 import compare, random_operand
from test_gpu_mx4 import Out, bits_type

pytestmark = pytest.mark.gpu

# To A's scales (2^-13 and more before: up to 2^119, rows of the largest fp32 numbers have 2^121), its inverse to B's (2^-11
# before: down to 2^-141, subnormal).
MOVED = (-115, -64, 64, 90, 100, 125, 130)


def scales(rng, rows, about):
    """Of two significant bits, so that subnormal ones keep them."""
    return (rng.choice([1.0, 1.25, 1.5, 1.75], rows) * about).astype(np.float32)


def moved(s, power):
    r = np.ldexp(s, power)
    assert np.array_equal(np.ldexp(r.astype(np.float64), -power), s)  # exactly
    return r


@pytest.mark.parametrize("act", ref.ACTS)
@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("m,n,k", [(5, 40, 300), (40, 1056, 512), (250, 4090, 260), (600, 4104, 384), (3850, 4096, 300),
                                   (3850, 4090, 128)])
def test_products_of_scales_far_apart(device, mc, m, n, k, kind, act):
    print(f"case far scales {kind} {m}x{n}x{k} {act}", flush=True)
    rng = np.random.default_rng(m + n)
    dtype = ref.TYPES[kind]
    n = n // 2 if act == "swiglu" else n
    rows = 2 * n if act == "swiglu" else n
    a, _ = random_operand(rng, m, k)
    b, _ = random_operand(rng, rows, k)
    sa, sb = scales(rng, m, 2.0 ** -13), scales(rng, rows, 2.0 ** -11)
    bias = rng.standard_normal(rows).astype(np.float32)
    da, db, dv = mc.DeviceBuffer.from_array(a), mc.DeviceBuffer.from_array(b), mc.DeviceBuffer.from_array(bias)

    def product(sa, sb):
        ca, cb = mc.DeviceBuffer.from_array(sa), mc.DeviceBuffer.from_array(sb)
        c = Out(mc, m * n * (4 if dtype == ref.F32 else 2))
        mc.launch_matmul_i8(da.ptr, ca.ptr, db.ptr, cb.ptr, dv.ptr, act, dtype, c.ptr, m, n, k)
        mc.synchronize()
        return c.get(bits_type(dtype), (m, n))

    plain = product(sa, sb)
    want, err = ref.activate(*ref.scaled(a, sa, b, sb, bias), act)
    compare(plain, want, ref.rounded(want, err, dtype), dtype)
    for power in MOVED if m < 3000 else MOVED[::2]:
        assert np.array_equal(product(moved(sa, power), moved(sb, -power)), plain), power


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("tokens,experts,top_k,n,k", [(3, 4, 2, 40, 200), (100, 4, 2, 960, 512), (700, 8, 4, 264, 512),
                                                      (4200, 8, 4, 2056, 384)])
def test_experts_of_scales_far_apart(device, mc, kind, tokens, experts, top_k, n, k):
    print(f"case experts of far scales {kind} {tokens} {n}x{k}", flush=True)
    rng = np.random.default_rng(tokens)
    dtype = ref.TYPES[kind]
    size = 4 if dtype == ref.F32 else 2
    order, offsets = random_plan(rng, tokens, experts, top_k)
    slots = tokens * top_k
    x, _ = random_operand(rng, tokens, k)
    h, _ = random_operand(rng, slots, k)
    w, _ = random_operand(rng, experts * n, k)
    sx, sh, sw = scales(rng, tokens, 2.0 ** -13), scales(rng, slots, 2.0 ** -13), scales(rng, experts * n, 2.0 ** -11)
    bias = rng.standard_normal(experts * n).astype(np.float32)
    gates = rng.uniform(0, 1, (tokens, top_k)).astype(np.float32)
    held = [upload(mc, v) for v in (order, offsets, x, h, w, bias, gates)]
    do, df, dx, dh, dw, db, dg = (at(v) for v in held)
    space = Out(mc, mc.experts_down_i8_workspace_bytes(dtype, tokens, top_k, n, k))

    def layer(sx, sh, sw):
        cx, ch, cw = (mc.DeviceBuffer.from_array(s) for s in (sx, sh, sw))
        c, y = Out(mc, slots * n * size), Out(mc, tokens * n * size)
        mc.launch_experts_up_i8(dx, cx.ptr, dw, cw.ptr, db, "gelu", dtype, c.ptr, do, df, tokens, top_k, experts, n, k)
        mc.launch_experts_down_i8(dh, ch.ptr, dw, cw.ptr, db, dtype, y.ptr, do, df, dg, tokens, top_k, experts, n, k, None,
                                  space.ptr)
        mc.synchronize()
        return c.get(bits_type(dtype), (slots, n)), y.get(bits_type(dtype), (tokens, n))

    plain = layer(sx, sh, sw)
    w3, sw2, b2 = w.reshape(experts, n, -1), sw.reshape(experts, n), bias.reshape(experts, n)
    compare(plain[0], *ref.experts_up(x, sx, w3, sw2, b2, "gelu", order, offsets, top_k, dtype), dtype)
    compare(plain[1], *ref.experts_down(h, sh, w3, sw2, b2, order, offsets, gates, top_k, dtype), dtype)
    for power in MOVED[::2] if tokens > 1000 else MOVED:
        got = layer(moved(sx, power), moved(sh, power), moved(sw, -power))
        assert all(np.array_equal(g, p) for g, p in zip(got, plain)), power


@pytest.mark.parametrize("m", [3, 40, 250, 600, 3850])
def test_results_past_the_range(device, mc, m):
    """Scales of 2^100 on both sides: infinities with the sum's sign, zeros where it is zero."""
    rng = np.random.default_rng(m)
    n, k = 2056, 128
    a, _ = random_operand(rng, m, k, 1)
    b, _ = random_operand(rng, n, k, 1)
    a[:, 20:] = 0  # short sums, many of them zero
    sums = a.astype(np.int32) @ b.astype(np.int32).T
    assert np.any(sums == 0)
    da, db = mc.DeviceBuffer.from_array(a), mc.DeviceBuffer.from_array(b)
    ca, cb = (mc.DeviceBuffer.from_array(np.full(r, 2.0 ** 100, dtype=np.float32)) for r in (m, n))
    c = Out(mc, m * n * 4)
    mc.launch_matmul_i8(da.ptr, ca.ptr, db.ptr, cb.ptr, None, None, 0, c.ptr, m, n, k)
    mc.synchronize()
    assert np.array_equal(c.get(np.float32, (m, n)), np.where(sums == 0, 0.0, np.copysign(np.inf, sums)))
