"""Refusals of the 4-bit and mixture-of-experts calls whose reason, or whose being refused at all, depends on more than
one argument; before anything reaches a device."""

import pytest

from test_mx4_refusals import P, refused


def moe(mc, **kw):
    good = dict(dtype=1, x=P, ldx=64, router=P, weights=4, w1=P, w1_scales=P, b1=None, w2=P, w2_scales=P, b2=None, y=P,
                chosen=None, gates=None, tokens=2, d=64, h=64, experts=4, top_k=2, activation="swiglu", normalize=True,
                stream=None, workspace=P)
    mc.launch_moe(**{**good, **kw})


@pytest.mark.parametrize("name", ["w1_scales", "w2_scales"])
@pytest.mark.parametrize("offset", [1, 2, 3])
def test_moe_scales_off_their_dwords(mc, name, offset):
    """Four scales at a time are read."""
    refused(mc, "scales.*4", moe, mc, **{name: P + offset})


@pytest.mark.parametrize("dtype,n,most", [(0, 4194241, 4194240), (0, 8388482, 4194240), (1, 4194241, 4194240),
                                          (1, 8388482, 8388480), (2, 1 << 30, 8388480)])
def test_columns_beyond_a_launch(mc, dtype, n, most):
    """16-bit columns are taken in pairs where their number is even: twice as many."""
    refused(mc, f"columns.*\\({most}\\)", mc.quantize_mx4_columns, dtype, P, n, P, P, 40, n)


@pytest.mark.parametrize("m,n,k", [(1 << 30, 1 << 30, 32), (1 << 24, 1 << 24, 32)])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_more_tiles_than_a_launch(mc, dtype, m, n, k):
    """Refused before A is cut into pieces, too."""
    refused(mc, "more tiles of C", mc.launch_matmul_mx4, P, P, P, P, dtype, P, m, n, k)
    refused(mc, "more tiles of C", mc.launch_matmul_mx4_weights, dtype, P, k, P, P, dtype, P, m, n, k, None, P)


def test_more_rows_than_are_cut(mc):
    refused(mc, "cuts", mc.launch_matmul_mx4_weights, 0, P, 1 << 24, P, P, 0, P, 1 << 24, 1, 1 << 24, None, P)


@pytest.mark.parametrize("activation", ["silu", "", -1, 3])
def test_moe_activations_that_are_none(mc, activation):
    """An unknown name as an unknown number."""
    refused(mc, "activation", moe, mc, activation=activation)
