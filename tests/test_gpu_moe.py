"""The mixture-of-experts MLP on the GPU against float64 numpy: the chosen experts exactly, gates and outputs within
the bound of its fp32 arithmetic; types, activations, sizes off every tile, ties, NaN, reuse of a workspace."""

import numpy as np
import pytest

import mx4_oracle as ref
from test_gpu_mx4 import Out, bits_type, device_rows, within

pytestmark = pytest.mark.gpu


def layer(mc, rng, weights, d, h, experts, act, bias):
    """Device weights (addresses in a dict, buffers kept) and their float64 values."""
    rows = 2 * h if act == "swiglu" else h
    out = {"keep": [], "b1": None, "b2": None, "vb1": None, "vb2": None, "s1": None, "s2": None}
    for name, shape in (("1", (experts, rows, d)), ("2", (experts, d, h))):
        w = rng.standard_normal(shape) * shape[2] ** -0.5
        if weights == ref.MX4:
            codes, scales, values = ref.quantize(w.reshape(-1, shape[2]))
            bufs = [mc.DeviceBuffer.from_array(codes), mc.DeviceBuffer.from_array(scales)]
            out["s" + name] = bufs[1].ptr
            out["v" + name] = values.reshape(shape)
        else:
            bits = ref.to_type(w, weights)
            bufs = [mc.DeviceBuffer.from_array(bits)]
            out["v" + name] = ref.from_type(bits, weights)
        out["w" + name] = bufs[0].ptr
        out["keep"] += bufs
        if bias:
            b = (rng.standard_normal(shape[:2]) * 0.2).astype(np.float32)
            out["keep"].append(mc.DeviceBuffer.from_array(b))
            out["b" + name], out["vb" + name] = out["keep"][-1].ptr, b.astype(np.float64)
    return out


def workspace_for(mc, *sizes):
    ws = mc.DeviceBuffer(mc.moe_workspace_bytes(*sizes))
    ws.fill_bytes(0)
    return ws


def run(mc, net, bits, dtype, router, weights, h, top_k, act, normalize, pad=0, stream=None, workspace=None):
    tokens, d = bits.shape
    experts = router.shape[0]
    x = device_rows(mc, bits, d + pad)
    r = mc.DeviceBuffer.from_array(router)
    y = Out(mc, tokens * d * (4 if dtype == ref.F32 else 2))
    chosen, gates = Out(mc, tokens * top_k * 4), Out(mc, tokens * top_k * 4)
    ws = workspace or workspace_for(mc, dtype, tokens, d, h, experts, top_k)
    mc.launch_moe(dtype, x.ptr, d + pad, r.ptr, weights, net["w1"], net["s1"], net["b1"], net["w2"], net["s2"],
                  net["b2"], y.ptr, chosen.ptr, gates.ptr, tokens, d, h, experts, top_k, act, normalize, stream, ws.ptr)
    mc.synchronize()
    return (ref.from_type(y.get(bits_type(dtype), (tokens, d)), dtype), chosen.get(np.int32, (tokens, top_k)),
            gates.get(np.float32, (tokens, top_k)).astype(np.float64))


def inputs(rng, tokens, d, experts, dtype, top_k, normalize):
    """x and a router whose decisions are clear of fp32 error (drawn again until they are)."""
    while True:
        bits = ref.to_type(rng.standard_normal((tokens, d)) * np.exp(0.3 * rng.standard_normal(d)), dtype)
        router = (rng.standard_normal((experts, d)) * d ** -0.5).astype(np.float32)
        routed = ref.route(ref.from_type(bits, dtype), router.astype(np.float64), top_k, normalize)
        if routed[2] > 2 * routed[3]:
            return bits, router, routed


def check(mc, seed, kind, weights, tokens, d, h, experts, top_k, act, normalize=True, bias=True, pad=0, **kw):
    dtype = ref.TYPES[kind]
    rng = np.random.default_rng(seed)
    net = layer(mc, rng, weights, d, h, experts, act, bias)
    bits, router, (chosen, gates, _, _, gate_err) = inputs(rng, tokens, d, experts, dtype, top_k, normalize)
    y, got_chosen, got_gates = run(mc, net, bits, dtype, router, weights, h, top_k, act, normalize, pad, **kw)
    assert np.array_equal(got_chosen, chosen)
    assert np.all(np.abs(got_gates - gates) <= gate_err * gates)
    exact, bound = ref.moe(ref.from_type(bits, dtype), net["v1"], net["vb1"], net["v2"], net["vb2"], chosen, gates, act,
                           gate_err, dtype)
    within(y, exact, bound)


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("weights", [ref.BF16, ref.F16, ref.MX4])
@pytest.mark.parametrize("act", ["relu", "gelu", "swiglu"])
def test_every_type_and_activation(device, mc, kind, weights, act):
    print(f"case moe {kind} weights {weights} {act}", flush=True)
    check(mc, 1, kind, weights, 5, 96, 80, 6, 2, act)


@pytest.mark.parametrize("weights", [ref.BF16, ref.F16, ref.MX4])
@pytest.mark.parametrize("tokens,d,h,experts,top_k,act", [
    (1, 1, 1, 1, 1, "relu"), (1, 256, 128, 64, 8, "swiglu"), (1, 130, 257, 5, 5, "gelu"), (2, 33, 31, 3, 1, "swiglu"),
    (15, 128, 100, 2, 2, "swiglu"), (16, 200, 136, 8, 2, "gelu"), (17, 257, 65, 31, 4, "swiglu"),
    (33, 64, 64, 1, 1, "relu"), (48, 100, 120, 16, 16, "swiglu"), (64, 96, 72, 7, 3, "gelu"),
    (64, 72, 40, 500, 8, "swiglu"), (64, 40, 48, 2, 1, "relu"), (3, 1000, 300, 4, 2, "gelu")])
def test_sizes(device, mc, weights, tokens, d, h, experts, top_k, act):
    print(f"case moe weights {weights} {tokens} {d} {h} {experts} {top_k} {act}", flush=True)
    for kind in ("f32", "bf16"):
        check(mc, 2, kind, weights, tokens, d, h, experts, top_k, act, normalize=tokens % 2 == 0, bias=experts % 2 == 1)


@pytest.mark.parametrize("weights", [ref.BF16, ref.F16])
def test_rows_that_start_at_odd_elements(device, mc, weights):
    """Weights a 2-byte step past a dword, and subnormal fp16 ones among them."""
    tokens, d, h, experts, top_k = 9, 150, 90, 5, 2
    rng = np.random.default_rng(21)
    net = layer(mc, rng, weights, d, h, experts, "gelu", True)
    for name, shape in (("1", (experts, h, d)), ("2", (experts, d, h))):
        w = rng.standard_normal(shape) * shape[2] ** -0.5
        w[:, ::3] *= 2.0 ** -14
        bits = ref.to_type(w, weights)
        buf = mc.DeviceBuffer.from_array(np.concatenate([np.zeros(1, bits.dtype), bits.reshape(-1)]))
        net["keep"].append(buf)
        net["w" + name], net["v" + name] = buf.ptr + 2, ref.from_type(bits, weights)
    bits, router, (chosen, gates, _, _, err) = inputs(rng, tokens, d, experts, ref.F16, top_k, True)
    y, got, _ = run(mc, net, bits, ref.F16, router, weights, h, top_k, "gelu", True)
    assert np.array_equal(got, chosen)
    exact, bound = ref.moe(ref.from_type(bits, ref.F16), net["v1"], net["vb1"], net["v2"], net["vb2"], chosen, gates, "gelu",
                           err, ref.F16)
    within(y, exact, bound)


def test_strided_rows_on_a_stream(device, mc):
    s = mc.Stream()
    for pad in (1, 8):
        check(mc, 3, "bf16", ref.MX4, 7, 160, 96, 4, 2, "swiglu", pad=pad, stream=s)


def test_a_workspace_serves_calls_of_other_sizes(device, mc):
    ws = workspace_for(mc, ref.F32, 64, 256, 256, 32, 8)
    for seed, (tokens, d, h, experts, top_k) in enumerate([(64, 256, 256, 32, 8), (1, 200, 100, 8, 2), (40, 130, 256, 32, 4),
                                                           (1, 200, 100, 8, 2)]):
        check(mc, seed, "f32", ref.BF16, tokens, d, h, experts, top_k, "gelu", workspace=ws)


def test_equal_logits_go_to_the_lower_experts(device, mc):
    tokens, d, h, experts, top_k = 3, 64, 32, 70, 6
    rng = np.random.default_rng(11)
    net = layer(mc, rng, ref.BF16, d, h, experts, "relu", False)
    bits = ref.to_type(rng.standard_normal((tokens, d)), ref.F32)
    router = np.tile((rng.standard_normal((1, d)) * 0.1).astype(np.float32), (experts, 1))
    _, chosen, gates = run(mc, net, bits, ref.F32, router, ref.BF16, h, top_k, "relu", True)
    assert np.array_equal(chosen, np.tile(np.arange(top_k), (tokens, 1)))
    assert np.all(np.abs(gates - 1.0 / top_k) <= 16 * 2.0 ** -24)


def test_every_token_to_the_same_expert(device, mc):
    tokens, d, h, experts = 64, 96, 64, 9
    rng = np.random.default_rng(12)
    net = layer(mc, rng, ref.MX4, d, h, experts, "swiglu", True)
    x = np.abs(rng.standard_normal((tokens, d))) + 0.1
    bits = ref.to_type(x, ref.BF16)
    router = np.zeros((experts, d), dtype=np.float32)
    router[7] = 0.05
    chosen, gates, gap, off, err = ref.route(ref.from_type(bits, ref.BF16), router.astype(np.float64), 1, False)
    assert np.all(chosen == 7) and gap > 2 * off
    y, got, got_gates = run(mc, net, bits, ref.BF16, router, ref.MX4, h, 1, "swiglu", False)
    assert np.all(got == 7) and np.all(np.abs(got_gates - gates) <= err * gates)
    exact, bound = ref.moe(ref.from_type(bits, ref.BF16), net["v1"], net["vb1"], net["v2"], net["vb2"], chosen, gates,
                           "swiglu", err, ref.BF16)
    within(y, exact, bound)


@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_a_token_that_is_no_number_leaves_the_others_alone(device, mc, value):
    tokens, d, h, experts, top_k = 20, 64, 48, 8, 3
    rng = np.random.default_rng(13)
    net = layer(mc, rng, ref.BF16, d, h, experts, "gelu", True)
    bits, router, (chosen, gates, _, _, err) = inputs(rng, tokens, d, experts, ref.F32, top_k, True)
    bits = bits.copy()
    bits[4, 10] = value
    y, got, got_gates = run(mc, net, bits, ref.F32, router, ref.BF16, h, top_k, "gelu", True)
    assert np.all(np.isnan(y[4])) and np.all(np.isnan(got_gates[4]))
    assert len(set(got[4])) == top_k and got[4].min() >= 0 and got[4].max() < experts
    others = np.arange(tokens) != 4
    assert np.array_equal(got[others], chosen[others])
    x = ref.from_type(bits, ref.F32)
    x[4] = 0.0
    exact, bound = ref.moe(x, net["v1"], net["vb1"], net["v2"], net["vb2"], chosen, gates, "gelu", err, ref.F32)
    within(y[others], exact[others], bound[others])


def test_the_same_bits_every_time_and_in_a_captured_graph(device, mc):
    tokens, d, h, experts, top_k = 24, 256, 192, 16, 4
    rng = np.random.default_rng(14)
    net = layer(mc, rng, ref.MX4, d, h, experts, "swiglu", False)
    bits = ref.to_type(rng.standard_normal((tokens, d)), ref.BF16)
    router = mc.DeviceBuffer.from_array((rng.standard_normal((experts, d)) * d ** -0.5).astype(np.float32))
    x = mc.DeviceBuffer.from_array(bits)
    y = mc.DeviceBuffer(2 * tokens * d)
    ws = workspace_for(mc, ref.BF16, tokens, d, h, experts, top_k)
    s = mc.Stream()

    def call(stream):
        mc.launch_moe(ref.BF16, x.ptr, d, router.ptr, ref.MX4, net["w1"], net["s1"], None, net["w2"], net["s2"], None,
                      y.ptr, None, None, tokens, d, h, experts, top_k, "swiglu", True, stream, ws.ptr)

    call(s)
    s.synchronize()
    first = y.download(np.uint16)
    graph = mc.CapturedGraph(s, call)
    for _ in range(4):
        y.fill_bytes(0)
        mc.synchronize()
        graph.launch()
        s.synchronize()
        assert np.array_equal(y.download(np.uint16), first)
        call(s)
        s.synchronize()
        assert np.array_equal(y.download(np.uint16), first)
