"""Arguments that the 4-bit and mixture-of-experts calls refuse, before anything reaches a device: code 1 and a message
that names the argument."""

import pytest

P = 1 << 20  # an aligned address that is never read


def refused(mc, match, fn, *args, **kw):
    with pytest.raises(mc.HipError, match=match) as e:
        fn(*args, **kw)
    assert e.value.code == 1


def test_operand_sizes(mc):
    assert mc.mx4_code_bytes(3, 1) == 3 * 64 and mc.mx4_scale_bytes(3, 1) == 3 * 4
    assert mc.mx4_code_bytes(2, 128) == 2 * 64 and mc.mx4_code_bytes(2, 129) == 2 * 128
    assert mc.mx4_scale_bytes(2, 4096) == 256 and mc.mx4_code_bytes(1 << 20, 1 << 14) == 1 << 33
    assert mc.mx4_code_bytes(0, 8) == 0 and mc.mx4_scale_bytes(8, -1) == 0


@pytest.mark.parametrize("columns", [False, True])
def test_quantize(mc, columns):
    fn = mc.quantize_mx4_columns if columns else mc.quantize_mx4
    good = dict(dtype=0, x=P, ld=64, codes=P, scales=P, a=64, b=64, values=P)

    def call(**kw):
        g = {**good, **kw}
        fn(g["dtype"], g["x"], g["ld"], g["codes"], g["scales"], g["a"], g["b"], g["values"])

    for match, kw in [("type", {"dtype": 4}), ("type", {"dtype": -1}), ("size", {"a": 0}), ("size", {"b": -5}),
                      ("closer", {"ld": 63}), ("null", {"x": None}), ("null", {"codes": None}),
                      ("null", {"scales": None}), ("codes", {"codes": P + 8}), ("scales", {"scales": P + 2}),
                      ("element", {"x": P + 2}), ("element", {"values": P + 1})]:
        refused(mc, match, call, **kw)


def test_product(mc):
    def call(ac=P, as_=P, bc=P, bs=P, dt=0, c=P, m=4, n=4, k=4):
        mc.launch_matmul_mx4(ac, as_, bc, bs, dt, c, m, n, k)

    for match, kw in [("type", {"dt": 3}), ("size", {"m": 0}), ("size", {"n": 0}), ("size", {"k": 0}),
                      ("2\\^24", {"k": (1 << 24) + 1}), ("null", {"ac": None}), ("null", {"bs": None}),
                      ("null", {"c": None}), ("codes", {"bc": P + 4}), ("scales", {"as_": P + 1}),
                      ("aligned", {"c": P + 2})]:
        refused(mc, match, call, **kw)


def test_weights(mc):
    def call(dt=1, a=P, lda=8, bc=P, bs=P, ct=1, c=P, m=4, n=4, k=8, ws=P):
        mc.launch_matmul_mx4_weights(dt, a, lda, bc, bs, ct, c, m, n, k, None, ws)

    for match, kw in [("type", {"dt": 4}), ("type", {"ct": 7}), ("size", {"m": 0}), ("closer", {"lda": 7}),
                      ("null", {"a": None}), ("null", {"bc": None}), ("codes", {"bc": P + 1}),
                      ("scales", {"bs": P + 2}), ("element", {"a": P + 1}), ("element", {"c": P + 1}),
                      ("workspace", {"m": 17, "ws": None}), ("workspace", {"m": 100, "ws": P + 128})]:
        refused(mc, match, call, **kw)
    assert mc.matmul_mx4_weights_workspace_bytes(1, 16, 64, 64) == 0  # few rows need none
    assert mc.matmul_mx4_weights_workspace_bytes(9, 4, 4, 4) == 0


def test_moe(mc):
    good = dict(dtype=1, x=P, ldx=64, router=P, weights=4, w1=P, w1_scales=P, b1=None, w2=P, w2_scales=P, b2=None, y=P,
                chosen=None, gates=None, tokens=2, d=64, h=64, experts=4, top_k=2, activation="swiglu", normalize=True,
                stream=None, workspace=P)

    def call(**kw):
        mc.launch_moe(**{**good, **kw})

    for match, kw in [("type", {"dtype": 4}), ("weights' type", {"weights": 0}), ("activation", {"activation": 3}),
                      ("size", {"tokens": 0}), ("size", {"h": 0}), ("64 tokens", {"tokens": 65}),
                      ("512 experts", {"experts": 513}), ("16 experts", {"experts": 32, "top_k": 17}),
                      ("than there are", {"top_k": 5}), ("closer", {"ldx": 63}), ("null", {"router": None}),
                      ("null", {"workspace": None}), ("scales", {"w2_scales": None}), ("address", {"w1": P + 8}),
                      ("address", {"x": P + 1}), ("address", {"b1": P + 2}), ("workspace", {"workspace": P + 16})]:
        refused(mc, match, call, **kw)
    assert mc.moe_workspace_bytes(1, 65, 64, 64, 4, 2) == 0 and mc.moe_workspace_bytes(1, 2, 64, 64, 4, 2) > 0
