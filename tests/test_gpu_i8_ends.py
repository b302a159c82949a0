"""The calls on 8-bit integers and experts where users push them: addresses aligned to their elements alone, two calls at
once on streams of their own, and calls after another call's failure."""

import numpy as np
import pytest

import i8_oracle as ref
import test_gpu_experts_i8 as experts
import test_gpu_i8 as operators
import test_gpu_route as routing
from test_gpu_mx4 import Out, bits_type

pytestmark = pytest.mark.gpu


class Odd(Out):
    """An output `shift` bytes past an aligned address."""

    def __init__(self, mc, nbytes, shift):
        super().__init__(mc, nbytes + shift)
        self.shift = shift
        self.ptr += shift

    def get(self, dtype, shape):
        raw = super().get(np.uint8, self.nbytes)
        assert np.all(raw[:self.shift] == 0xAB)
        return np.frombuffer(raw[self.shift:].tobytes(), dtype).reshape(shape)


def odd(mc, a):
    """An array one element past an aligned address, what lies before it no number; the buffer and the address."""
    a = np.ascontiguousarray(a).reshape(-1)
    buf = mc.DeviceBuffer.from_array(np.concatenate([np.full(1, -1, a.dtype) if a.dtype.kind == "i" else
                                                     np.full(1, np.nan, a.dtype), a]))
    return buf, buf.ptr + a.itemsize


# A size for each kernel: blocks of 16x32, 32x32 and 32x64, tiles of 128x128 and of 256x256; columns in eights and not.
@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("m,n,k", [(3, 40, 200), (32, 4104, 200), (250, 4090, 260), (600, 4104, 384), (600, 4099, 129),
                                   (3850, 4096, 300), (3850, 4090, 300)])
@pytest.mark.parametrize("act", [None, "swiglu"])
def test_products_between_odd_addresses(device, mc, kind, m, n, k, act):
    print(f"case odd addresses {kind} {m}x{n}x{k} {act}", flush=True)
    rng = np.random.default_rng(m + n)
    dtype = ref.TYPES[kind]
    n = n // 2 if act else n
    rows = 2 * n if act else n
    a, sa = operators.random_operand(rng, m, k)
    b, sb = operators.random_operand(rng, rows, k)
    v = rng.standard_normal(rows).astype(np.float32)
    want, err = ref.activate(*ref.scaled(a, sa, b, sb, v), act)
    da, db = operators.operand(mc, a, sa), operators.operand(mc, b, sb)
    (osa, psa), (osb, psb), (ov, pv) = odd(mc, sa), odd(mc, sb), odd(mc, v)
    size = 4 if dtype == ref.F32 else 2
    c = Odd(mc, m * n * size, size)
    mc.launch_matmul_i8(da[0].ptr, psa, db[0].ptr, psb, pv, act, dtype, c.ptr, m, n, k)
    mc.synchronize()
    operators.compare(c.get(bits_type(dtype), (m, n)), want, ref.rounded(want, err, dtype), dtype)


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("tokens,n,k", [(3, 40, 200), (40, 264, 200), (700, 264, 512), (1500, 1024, 512)])
def test_experts_between_odd_addresses(device, mc, kind, tokens, n, k):
    print(f"case experts at odd addresses {kind} {tokens} {n}x{k}", flush=True)
    count, top_k = 4, 2
    rng = np.random.default_rng(tokens)
    dtype = ref.TYPES[kind]
    size = 4 if dtype == ref.F32 else 2
    order, offsets = experts.random_plan(rng, tokens, count, top_k)
    (oo, po), (of, pf) = odd(mc, order), odd(mc, offsets)
    x, sx = operators.random_operand(rng, tokens, k)
    w, sw, bias = experts.weights(rng, count, n, k, True)
    dx, dw = operators.operand(mc, x, sx), operators.operand(mc, w, sw)
    (osx, psx), (osw, psw), (ob, pb) = odd(mc, sx), odd(mc, sw), odd(mc, bias)
    c = Odd(mc, tokens * top_k * n * size, size)
    mc.launch_experts_up_i8(dx[0].ptr, psx, dw[0].ptr, psw, pb, "gelu", dtype, c.ptr, po, pf, tokens, top_k, count, n, k)
    mc.synchronize()
    want, bound = ref.experts_up(x, sx, w, sw, bias, "gelu", order, offsets, top_k, dtype)
    operators.compare(c.get(bits_type(dtype), (tokens * top_k, n)), want, bound, dtype)

    h, sh = operators.random_operand(rng, tokens * top_k, k)
    gates = rng.uniform(0, 1, (tokens, top_k)).astype(np.float32)
    dh, (osh, psh), (og, pg) = operators.operand(mc, h, sh), odd(mc, sh), odd(mc, gates)
    y = Odd(mc, tokens * n * size, size)
    space = Out(mc, mc.experts_down_i8_workspace_bytes(dtype, tokens, top_k, n, k))
    mc.launch_experts_down_i8(dh[0].ptr, psh, dw[0].ptr, psw, pb, dtype, y.ptr, po, pf, pg, tokens, top_k, count, n, k,
                              None, space.ptr)
    mc.synchronize()
    want, bound = ref.experts_down(h, sh, w, sw, bias, order, offsets, gates, top_k, dtype)
    operators.compare(y.get(bits_type(dtype), (tokens, n)), want, bound, dtype)


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("columns", [False, True])
@pytest.mark.parametrize("rows,k", [(3, 40), (1200, 600), (40, 5000), (2, 20001)])
def test_quantisation_between_odd_addresses(device, mc, kind, columns, rows, k):
    dtype = ref.TYPES[kind]
    size = 4 if dtype == ref.F32 else 2
    bits = ref.to_type(np.random.default_rng(rows).standard_normal((rows, k)), dtype)
    stored = np.ascontiguousarray(bits.T) if columns else bits
    x = mc.DeviceBuffer.from_array(np.concatenate([np.full(1, 0x7FFF if size == 2 else np.nan, bits.dtype),
                                                   stored.reshape(-1)]))
    codes, scales, v = Out(mc, mc.i8_code_bytes(rows, k)), Odd(mc, rows * 4, 4), Odd(mc, rows * k * size, size)
    call = mc.quantize_i8_columns if columns else mc.quantize_i8
    call(dtype, x.ptr + size, stored.shape[1], codes.ptr, scales.ptr, *stored.shape, v.ptr)
    mc.synchronize()
    want = ref.quantize(ref.from_type(bits, dtype))
    assert np.array_equal(codes.get(np.int8, (rows, ref.padded(k))), want[0])
    assert np.array_equal(scales.get(np.float32, rows), want[1])
    back = np.ascontiguousarray(v.get(bits_type(dtype), stored.shape))
    wanted = ref.from_type(ref.values(*want, k, dtype), dtype)
    assert np.array_equal(ref.from_type(back, dtype), wanted.T if columns else wanted)


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("tokens,count", [(1, 64), (7, 60), (100, 256), (40, 512)])
def test_choices_between_odd_addresses(device, mc, kind, tokens, count):
    dtype, top_k = ref.TYPES[kind], 4
    size = 4 if dtype == ref.F32 else 2
    rng = np.random.default_rng(tokens)
    bits = ref.to_type(rng.standard_normal((tokens, count)), dtype)
    bias = rng.standard_normal(count).astype(np.float32)
    x = mc.DeviceBuffer.from_array(np.concatenate([np.zeros(1, bits.dtype), bits.reshape(-1)]))
    ob, pb = odd(mc, bias)
    chosen, gates, order = (Odd(mc, tokens * top_k * 4, 4) for _ in range(3))
    offsets = Odd(mc, (count + 1) * 4, 4)
    space = mc.DeviceBuffer(max(256, mc.route_workspace_bytes(tokens, count, top_k)))
    mc.launch_route(dtype, x.ptr + size, count, pb, tokens, count, top_k, "sigmoid", 2, 1, 2, True, 2.5, chosen.ptr,
                    gates.ptr, order.ptr, offsets.ptr, None, space.ptr)
    mc.synchronize()
    want = ref.route(ref.from_type(bits, dtype), bias, top_k, "sigmoid", 2, 1, 2, True, 2.5)
    got = chosen.get(np.int32, (tokens, top_k))
    assert np.array_equal(got, want[0])
    # One rounding to fp32, and float64's own before it.
    assert np.all(np.abs(gates.get(np.float32, got.shape) - want[1]) <= (2.0 ** -24 + 2.0 ** -42) * np.abs(want[1]))
    plan = ref.plan(got, count)
    assert np.array_equal(order.get(np.int32, tokens * top_k), plan[0])
    assert np.array_equal(offsets.get(np.int32, count + 1), plan[1])


def test_calls_at_once(device, mc):
    """The same calls on four streams, each with its own workspace, over and over: the results of each by itself."""
    tokens, count, top_k, n, k = 500, 8, 2, 264, 512
    rng = np.random.default_rng(9)
    jobs = []
    for i in range(4):
        logits = rng.standard_normal((tokens, count)).astype(np.float32)
        h, sh = operators.random_operand(rng, tokens * top_k, k)
        w, sw, _ = experts.weights(rng, count, n, k, False)
        jobs.append({"stream": mc.Stream(), "logits": mc.DeviceBuffer.from_array(logits),
                     "h": operators.operand(mc, h, sh), "w": operators.operand(mc, w, sw),
                     "out": [mc.DeviceBuffer(tokens * top_k * 4) for _ in range(3)] + [mc.DeviceBuffer((count + 1) * 4)],
                     "y": mc.DeviceBuffer(tokens * n * 4),
                     "route": mc.DeviceBuffer(mc.route_workspace_bytes(tokens, count, top_k)),
                     "down": mc.DeviceBuffer(mc.experts_down_i8_workspace_bytes(0, tokens, top_k, n, k))})

    def run(j):
        chosen, gates, order, offsets = (o.ptr for o in j["out"])
        mc.launch_route(0, j["logits"].ptr, count, None, tokens, count, top_k, "softmax", 1, 1, 1, True, 1.0, chosen, gates,
                        order, offsets, j["stream"], j["route"].ptr)
        mc.launch_experts_down_i8(j["h"][0].ptr, j["h"][1].ptr, j["w"][0].ptr, j["w"][1].ptr, None, 0, j["y"].ptr, order,
                                  offsets, gates, tokens, top_k, count, n, k, j["stream"], j["down"].ptr)

    def results(j):
        return [o.download(np.uint8) for o in (*j["out"], j["y"])]

    alone = []
    for j in jobs:
        run(j)
        mc.synchronize()
        alone.append(results(j))
        for o in (*j["out"], j["y"]):
            o.fill_bytes(0)
        mc.synchronize()
    for _ in range(5):
        for j in jobs:
            run(j)
    mc.synchronize()
    for j, want in zip(jobs, alone):
        assert all(np.array_equal(a, b) for a, b in zip(results(j), want))


@pytest.fixture
def failed(device, mc):
    """A copy to nowhere, refused by the runtime; forgotten after the test."""
    a = np.zeros(4, dtype=np.float32)

    def fail():
        assert mc.library().mc_memcpy_htod(None, a.ctypes.data, a.nbytes) != 0

    yield fail
    mc.library().hipGetLastError()  # of the runtime that the library is linked with


def before(mc, monkeypatch, name, fail):
    """The package's function with a failure before each call."""
    call = getattr(mc, name)

    def both(*args, **kw):
        fail()
        return call(*args, **kw)

    monkeypatch.setattr(mc, name, both)


@pytest.mark.parametrize("columns", [False, True])
@pytest.mark.parametrize("k", [200, 3000])
def test_quantisation_after_a_failure(mc, failed, columns, k, monkeypatch):
    before(mc, monkeypatch, "quantize_i8_columns" if columns else "quantize_i8", failed)
    operators.check_quantize(mc, np.random.default_rng(1).standard_normal((5, k)), ref.F32, columns=columns)


@pytest.mark.parametrize("m", [3, 600])
def test_product_after_a_failure(mc, failed, m, monkeypatch):
    before(mc, monkeypatch, "launch_matmul_i8", failed)
    operators.check_product(mc, 1, m, 4104, 300)


@pytest.mark.parametrize("tokens", [3, 100])
def test_experts_after_a_failure(mc, failed, tokens, monkeypatch):
    for name in ("launch_route", "launch_experts_up_i8", "launch_experts_down_i8"):
        before(mc, monkeypatch, name, failed)
    routing.check(mc, np.random.default_rng(2).standard_normal((tokens, 64)), "f32", None, 4)
    experts.check_up(mc, 3, tokens, 4, 2, 64, 100, "bf16", "swiglu")
    experts.check_down(mc, 4, tokens, 4, 2, 64, 100, "bf16")
