"""The experts' products on a plan on the GPU against float64 numpy: both products, every activation and type, experts
without tokens and with most of them, parts of a plan, and a whole layer from the router on, captured and replayed."""

import numpy as np
import pytest

import i8_oracle as ref
from test_gpu_i8 import compare, operand, random_operand
from test_gpu_mx4 import Out, bits_type

pytestmark = pytest.mark.gpu


def random_plan(rng, tokens, experts, top_k, skew=1.0):
    keys = rng.standard_normal((tokens, experts)) + skew * rng.standard_normal(experts)
    chosen = np.argsort(-keys, axis=1)[:, :top_k].astype(np.int32)
    return ref.plan(chosen, experts)


def weights(rng, experts, rows, k, bias):
    w, sw = random_operand(rng, experts * rows, k)
    sw *= np.float32(4.0)
    b = rng.standard_normal((experts, rows)).astype(np.float32) if bias else None
    return w.reshape(experts, rows, -1), sw.reshape(experts, rows), b


def upload(mc, a):
    return mc.DeviceBuffer.from_array(np.ascontiguousarray(a)) if a is not None else None


def at(buf):
    return buf.ptr if buf is not None else None


def check_up(mc, seed, tokens, experts, top_k, n, k, kind, act, bias=False, skew=1.0, part=None):
    rng = np.random.default_rng(seed)
    dtype = ref.TYPES[kind]
    order, offsets = random_plan(rng, tokens, experts, top_k, skew)
    a, sa = random_operand(rng, tokens, k)
    w, sw, b = weights(rng, experts, 2 * n if act == "swiglu" else n, k, bias)
    e0, e1 = part or (0, experts)
    want, bound = ref.experts_up(a, sa, w[e0:e1], sw[e0:e1], None if b is None else b[e0:e1], act, order,
                                 offsets[e0:e1 + 1], top_k, dtype)
    da, dw = operand(mc, a, sa), operand(mc, w[e0:e1], sw[e0:e1])
    db, do, df = upload(mc, None if b is None else b[e0:e1]), upload(mc, order), upload(mc, offsets[e0:e1 + 1])
    c = Out(mc, tokens * top_k * n * (4 if dtype == ref.F32 else 2))
    mc.launch_experts_up_i8(da[0].ptr, da[1].ptr, dw[0].ptr, dw[1].ptr, at(db), act, dtype, c.ptr, do.ptr, df.ptr, tokens,
                            top_k, e1 - e0, n, k)
    mc.synchronize()
    got = c.get(bits_type(dtype), (tokens * top_k, n))
    mine = slice(offsets[e0], offsets[e1])
    compare(got[mine], want[mine], bound[mine], dtype)
    rest = np.delete(got, np.r_[mine], axis=0)
    assert np.all(rest.view(np.uint8) == 0xAB)  # left as they were


def check_down(mc, seed, tokens, experts, top_k, n, k, kind, bias=False, skew=1.0):
    rng = np.random.default_rng(seed)
    dtype = ref.TYPES[kind]
    order, offsets = random_plan(rng, tokens, experts, top_k, skew)
    a, sa = random_operand(rng, tokens * top_k, k)
    w, sw, b = weights(rng, experts, n, k, bias)
    gates = rng.uniform(0, 1, (tokens, top_k)).astype(np.float32)
    want, bound = ref.experts_down(a, sa, w, sw, b, order, offsets, gates, top_k, dtype)
    da, dw = operand(mc, a, sa), operand(mc, w, sw)
    db, do, df, dg = upload(mc, b), upload(mc, order), upload(mc, offsets), upload(mc, gates)
    y = Out(mc, tokens * n * (4 if dtype == ref.F32 else 2))
    space = Out(mc, mc.experts_down_i8_workspace_bytes(dtype, tokens, top_k, n, k))
    mc.launch_experts_down_i8(da[0].ptr, da[1].ptr, dw[0].ptr, dw[1].ptr, at(db), dtype, y.ptr, do.ptr, df.ptr, dg.ptr,
                              tokens, top_k, experts, n, k, None, space.ptr)
    mc.synchronize()
    space.get(np.uint8, space.nbytes)  # its guards
    compare(y.get(bits_type(dtype), (tokens, n)), want, bound, dtype)


SIZES = [(1, 4, 1, 16, 64), (1, 64, 8, 96, 256), (2, 5, 5, 33, 100), (5, 31, 4, 48, 513), (16, 8, 2, 130, 300),
         (17, 128, 3, 64, 128), (40, 4, 4, 50, 200), (64, 16, 8, 200, 384), (100, 7, 3, 65, 1000), (300, 8, 2, 96, 520)]


@pytest.mark.parametrize("act", ref.ACTS)
@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("tokens,experts,top_k,n,k", SIZES)
def test_up(device, mc, kind, tokens, experts, top_k, n, k, act):
    print(f"case up {kind} {tokens} of {experts} top {top_k} {n}x{k} {act}", flush=True)
    check_up(mc, tokens + n, tokens, experts, top_k, n, k, kind, act, bias=tokens % 2 == 0)


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("tokens,experts,top_k,n,k", SIZES)
def test_down(device, mc, kind, tokens, experts, top_k, n, k):
    print(f"case down {kind} {tokens} of {experts} top {top_k} {n}x{k}", flush=True)
    check_down(mc, tokens + n, tokens, experts, top_k, n, k, kind, bias=tokens % 2 == 0)


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("tokens,experts,top_k,n,k,skew", [(700, 4, 2, 264, 512, 0.3), (1000, 8, 4, 300, 640, 3.0),
                                                           (2000, 64, 8, 256, 256, 1.0), (513, 3, 1, 520, 384, 5.0),
                                                           (3000, 16, 2, 136, 300, 0.5)])
def test_many_tokens(device, mc, kind, tokens, experts, top_k, n, k, skew):
    print(f"case many {kind} {tokens} of {experts} top {top_k} {n}x{k}", flush=True)
    check_up(mc, 1, tokens, experts, top_k, n, k, kind, "swiglu", skew=skew)
    check_up(mc, 2, tokens, experts, top_k, n, k, kind, "gelu", bias=True, skew=skew)
    check_down(mc, 3, tokens, experts, top_k, n, k, kind, bias=True, skew=skew)


# Each kernel by sizes that its rule gives it: blocks of 16x32, 32x32 and 32x64, tiles of 128x128, and of 256x256 with
# whole, half and short last tiles; even plans and one expert with nearly all.
VARIANTS = [(40, 16, 4, 520, 256, 1.0), (100, 4, 2, 960, 512, 0.3), (90, 4, 2, 520, 256, 0.5),
            (200, 4, 2, 1032, 256, 0.5), (700, 8, 4, 1030, 256, 1.0),
            (1500, 4, 2, 2056, 128, 0.3), (1300, 3, 2, 4100, 256, 4.0), (4000, 2, 1, 4104, 128, 0.3),
            (4200, 8, 4, 2056, 384, 1.0), (2100, 4, 2, 4096, 1600, 0.4), (2100, 3, 2, 4100, 1500, 3.0)]


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("tokens,experts,top_k,n,k,skew", VARIANTS)
def test_by_every_kernel(device, mc, kind, tokens, experts, top_k, n, k, skew):
    for act in (ref.ACTS[(tokens // 10 + sorted(ref.TYPES).index(kind)) % 3], "swiglu"):
        print(f"case kernel {kind} {tokens} of {experts} top {top_k} {n}x{k} {act}", flush=True)
        check_up(mc, n, tokens, experts, top_k, n // 2 if act == "swiglu" else n, k, kind, act, bias=k == 256, skew=skew)
    check_down(mc, n + 1, tokens, experts, top_k, n, k, kind, bias=k == 128, skew=skew)


@pytest.mark.parametrize("tokens", [3, 60, 900])
@pytest.mark.parametrize("part", [(0, 3), (2, 7), (7, 8), (4, 4 + 1)])
def test_a_part_of_a_plan_leaves_the_others_alone(device, mc, tokens, part):
    check_up(mc, tokens, tokens, 8, 2, 72, 200, "bf16", "relu", part=part)
    check_up(mc, tokens, tokens, 8, 2, 72, 200, "f32", "swiglu", bias=True, part=part)


@pytest.mark.parametrize("tokens", [1, 16, 400])
def test_a_layer_from_its_router_on(device, mc, tokens):
    """Router's product, choice, quantisation, both products: each step against float64 of what the step before wrote; then
    captured into a graph and replayed for other tokens, with the same bits as launched one by one."""
    print(f"case layer {tokens}", flush=True)
    rng = np.random.default_rng(tokens)
    d, h, experts, top_k = 256, 136, 16, 4
    slots = tokens * top_k
    router = mc.DeviceBuffer.from_array((rng.standard_normal((d, experts)) * d ** -0.5).astype(np.float32))
    bias = (rng.standard_normal(experts) * 0.05).astype(np.float32)
    dbias = mc.DeviceBuffer.from_array(bias)
    dense = [(rng.standard_normal(s) * s[1] ** -0.5).astype(np.float32) for s in ((experts, d, 2 * h), (experts, h, d))]
    held = []
    for w, (k, n) in zip(dense, ((d, 2 * h), (h, d))):
        codes, scales = mc.DeviceBuffer(mc.i8_code_bytes(experts * n, k)), mc.DeviceBuffer(experts * n * 4)
        for e in range(experts):  # stored [k, n], as the matmuls take B
            x = mc.DeviceBuffer.from_array(w[e])
            mc.quantize_i8_columns(0, x.ptr, n, codes.ptr + mc.i8_code_bytes(e * n, k) if e else codes.ptr,
                                   scales.ptr + e * n * 4, k, n)
            mc.synchronize()
        held.append((codes, scales))
    (w1, s1), (w2, s2) = held
    x = mc.DeviceBuffer(tokens * d * 4)
    logits, chosen, gates = mc.DeviceBuffer(tokens * experts * 4), mc.DeviceBuffer(slots * 4), mc.DeviceBuffer(slots * 4)
    order, offsets = mc.DeviceBuffer(slots * 4), mc.DeviceBuffer((experts + 1) * 4)
    xc, xs = mc.DeviceBuffer(mc.i8_code_bytes(tokens, d)), mc.DeviceBuffer(tokens * 4)
    hidden, y = mc.DeviceBuffer(slots * h * 2), mc.DeviceBuffer(tokens * d * 4)
    hc, hs = mc.DeviceBuffer(mc.i8_code_bytes(slots, h)), mc.DeviceBuffer(slots * 4)
    route_space = mc.DeviceBuffer(max(256, mc.route_workspace_bytes(tokens, experts, top_k)))
    down_space = mc.DeviceBuffer(mc.experts_down_i8_workspace_bytes(0, tokens, top_k, d, h))

    def layer(s):
        mc.launch_matmul("naive", x.ptr, router.ptr, logits.ptr, tokens, experts, d, s)
        mc.launch_route(0, logits.ptr, experts, dbias.ptr, tokens, experts, top_k, "sigmoid", 4, 2, 2, True, 1.5,
                        chosen.ptr, gates.ptr, order.ptr, offsets.ptr, s, route_space.ptr)
        mc.quantize_i8(0, x.ptr, d, xc.ptr, xs.ptr, tokens, d, None, s)
        mc.launch_experts_up_i8(xc.ptr, xs.ptr, w1.ptr, s1.ptr, None, "swiglu", 1, hidden.ptr, order.ptr, offsets.ptr,
                                tokens, top_k, experts, h, d, s)
        mc.quantize_i8(1, hidden.ptr, h, hc.ptr, hs.ptr, slots, h, None, s)
        mc.launch_experts_down_i8(hc.ptr, hs.ptr, w2.ptr, s2.ptr, None, 0, y.ptr, order.ptr, offsets.ptr, gates.ptr,
                                  tokens, top_k, experts, d, h, s, down_space.ptr)

    stream = mc.Stream()
    graph = mc.CapturedGraph(stream, layer)
    outputs = (logits, chosen, gates, order, offsets, xc, xs, hidden, hc, hs, y)
    for _ in range(3):
        rows = rng.standard_normal((tokens, d)).astype(np.float32)
        assert mc.library().mc_memcpy_htod(x.ptr, rows.ctypes.data, rows.nbytes) == 0
        for buf in outputs:
            buf.fill_bytes(0xEE)
        mc.synchronize()
        layer(stream)
        stream.synchronize()
        eager = [buf.download(np.uint8) for buf in outputs]
        for buf in outputs:
            buf.fill_bytes(0x77)
        mc.synchronize()
        graph.launch()
        stream.synchronize()
        for one, buf in zip(eager, outputs):
            assert np.array_equal(one, buf.download(np.uint8))
    host = lambda buf, t, shape: buf.download(np.uint8).view(t).reshape(shape)  # noqa: E731
    l = host(logits, np.float32, (tokens, experts))
    pick, gate, _ = ref.route(l.astype(np.float64), bias, top_k, "sigmoid", 4, 2, 2, True, 1.5)
    assert np.array_equal(host(chosen, np.int32, (tokens, top_k)), pick)
    want_order, want_offsets = ref.plan(pick, experts)
    assert np.array_equal(host(order, np.int32, -1), want_order)
    assert np.array_equal(host(offsets, np.int32, -1), want_offsets)
    a, sa = ref.quantize(rows.astype(np.float64))
    assert np.array_equal(host(xc, np.int8, a.shape), a) and np.array_equal(host(xs, np.float32, -1), sa)
    q = [[ref.quantize(w[e].T.astype(np.float64)) for e in range(experts)] for w in dense]
    (c1, t1), (c2, t2) = ((np.stack([o[0] for o in ops]), np.stack([o[1] for o in ops])) for ops in q)
    assert np.array_equal(host(w1, np.int8, c1.shape), c1) and np.array_equal(host(s2, np.float32, t2.shape), t2)
    want, bound = ref.experts_up(a, sa, c1, t1, None, "swiglu", want_order, want_offsets, top_k, ref.BF16)
    bits = host(hidden, np.uint16, (slots, h))
    compare(bits, want, bound, ref.BF16)
    a, sa = ref.quantize(ref.from_type(bits, ref.BF16))
    assert np.array_equal(host(hc, np.int8, a.shape), a) and np.array_equal(host(hs, np.float32, -1), sa)
    g = host(gates, np.float32, (tokens, top_k))
    want, bound = ref.experts_down(a, sa, c2, t2, None, want_order, want_offsets, g, top_k, ref.F32)
    compare(host(y, np.float32, (tokens, d)), want, bound, ref.F32)
