"""Arguments that the 8-bit integer calls, the router and the experts' products refuse, before anything reaches a device:
code 1 and a message that names the argument."""

import pytest

P = 1 << 20  # an aligned address that is never read


def refused(mc, match, fn, *args, **kw):
    with pytest.raises(mc.HipError, match=match) as e:
        fn(*args, **kw)
    assert e.value.code == 1


def test_operand_sizes(mc):
    assert mc.i8_code_bytes(3, 1) == 3 * 128 and mc.i8_code_bytes(2, 128) == 256 and mc.i8_code_bytes(2, 129) == 512
    assert mc.i8_code_bytes(1 << 20, 1 << 14) == 1 << 34
    assert mc.i8_code_bytes(0, 8) == 0 and mc.i8_code_bytes(8, -1) == 0


@pytest.mark.parametrize("columns", [False, True])
def test_quantize(mc, columns):
    fn = mc.quantize_i8_columns if columns else mc.quantize_i8
    good = dict(dtype=0, x=P, ld=64, codes=P, scales=P, a=64, b=64, values=P)

    def call(**kw):
        g = {**good, **kw}
        fn(g["dtype"], g["x"], g["ld"], g["codes"], g["scales"], g["a"], g["b"], g["values"])

    for match, kw in [("type", {"dtype": 4}), ("type", {"dtype": -1}), ("size", {"a": 0}), ("size", {"b": -5}),
                      ("closer", {"ld": 63}), ("null", {"x": None}), ("null", {"codes": None}),
                      ("null", {"scales": None}), ("codes", {"codes": P + 8}), ("scales", {"scales": P + 2}),
                      ("element", {"x": P + 2}), ("element", {"values": P + 1}),
                      ("2\\^28", {"a" if columns else "b": (1 << 28) + 1, "ld": 1 << 29})]:
        refused(mc, match, call, **kw)


def test_product(mc):
    def call(ac=P, as_=P, bc=P, bs=P, bias=None, act=None, dt=0, c=P, m=4, n=4, k=4):
        mc.launch_matmul_i8(ac, as_, bc, bs, bias, act, dt, c, m, n, k)

    for match, kw in [("type", {"dt": 3}), ("activation", {"act": "tanh"}), ("activation", {"act": 4}),
                      ("size", {"m": 0}), ("size", {"n": 0}), ("size", {"k": 0}), ("131071", {"k": 131072}),
                      ("2\\^30", {"n": (1 << 30) + 1}), ("null", {"ac": None}), ("null", {"bs": None}),
                      ("null", {"c": None}), ("codes", {"bc": P + 4}), ("scales", {"as_": P + 1}),
                      ("bias", {"bias": P + 2}), ("aligned", {"c": P + 2})]:
        refused(mc, match, call, **kw)


def test_route(mc):
    good = dict(dtype=0, logits=P, ld=64, bias=None, tokens=4, experts=64, top_k=8, score="softmax", groups=1,
                top_groups=1, group_best=1, normalize=True, scale=1.0, chosen=P, gates=P, order=P, offsets=P,
                workspace=P)

    def call(**kw):
        mc.launch_route(**{**good, **kw})

    for match, kw in [("type", {"dtype": 4}), ("score", {"score": "tanh"}), ("size", {"tokens": 0}),
                      ("size", {"top_k": 0}), ("size", {"groups": 0}), ("size", {"top_groups": -1}),
                      ("512", {"experts": 513, "ld": 513}), ("16 experts", {"top_k": 17}),
                      ("evenly", {"groups": 7}), ("64 groups", {"groups": 128, "experts": 128, "ld": 128}),
                      ("more groups", {"groups": 4, "top_groups": 5}), ("group's score", {"group_best": 3}),
                      ("than the chosen groups", {"groups": 16, "top_groups": 1}), ("closer", {"ld": 63}),
                      ("pairs", {"tokens": 1 << 28}), ("null", {"logits": None}), ("null", {"gates": None}),
                      ("one half", {"order": None}), ("one half", {"offsets": None}), ("element", {"logits": P + 2}),
                      ("aligned", {"bias": P + 2}), ("aligned", {"order": P + 1}),
                      ("workspace", {"tokens": 64, "workspace": None}), ("workspace", {"tokens": 64, "workspace": P + 64})]:
        refused(mc, match, call, **kw)
    assert mc.route_workspace_bytes(1, 64, 8) == 0 and mc.route_workspace_bytes(64, 64, 8) > 0
    assert mc.route_workspace_bytes(0, 64, 8) == 0 and mc.route_workspace_bytes(64, 64, 17) == 0


@pytest.mark.parametrize("down", [False, True])
def test_experts(mc, down):
    good = dict(x=P, xs=P, w=P, ws=P, bias=None, c_dtype=0, c=P, order=P, offsets=P, tokens=4, top_k=2, experts=8, n=64,
                k=64, gates=P, workspace=P, activation=None)

    def call(**kw):
        g = {**good, **kw}
        plan = (g["order"], g["offsets"])
        sizes = (g["tokens"], g["top_k"], g["experts"], g["n"], g["k"])
        if down:
            mc.launch_experts_down_i8(g["x"], g["xs"], g["w"], g["ws"], g["bias"], g["c_dtype"], g["c"], *plan,
                                      g["gates"], *sizes, None, g["workspace"])
        else:
            mc.launch_experts_up_i8(g["x"], g["xs"], g["w"], g["ws"], g["bias"], g["activation"], g["c_dtype"], g["c"],
                                    *plan, *sizes)

    bad = [("type", {"c_dtype": 4}), ("size", {"tokens": 0}), ("size", {"n": 0}), ("size", {"experts": 0}),
           ("512", {"experts": 513}), ("16 experts", {"top_k": 17, "experts": 32}), ("131071", {"k": 131072}),
           ("pairs", {"tokens": 1 << 30}), ("null", {"x": None}), ("null", {"ws": None}), ("null plan", {"order": None}), ("null plan", {"offsets": None}), ("plan that", {"offsets": P + 2}),
           ("codes", {"w": P + 8}), ("bias", {"bias": P + 1}), ("aligned", {"c": P + 2})]
    if down:
        bad += [("than there are", {"top_k": 9}), ("gates", {"gates": None}), ("workspace", {"workspace": None}), ("gates", {"gates": P + 2}),
                ("workspace", {"workspace": P + 16})]
    else:
        bad += [("activation", {"activation": "tanh"})]
    for match, kw in bad:
        refused(mc, match, call, **kw)
    assert mc.experts_down_i8_workspace_bytes(0, 4, 2, 0, 64) == 0 and mc.experts_down_i8_workspace_bytes(0, 4, 2, 64, 64) > 0
