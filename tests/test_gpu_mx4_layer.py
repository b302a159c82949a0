"""The example that serves a layer on 4-bit weights: its parts agree with the same functions in float64."""

import json

import pytest

from minicompiler_amd import mx4_layer

# bf16 outputs: at most half a unit of 2^-8 of each element; the experts' input and sums add fp32 and 16-bit cuts, far below.
BF16_ERROR = 2.0 ** -8


@pytest.mark.gpu
@pytest.mark.parametrize("d,h,experts,top_k,prompt,batch", [(256, 128, 8, 2, 40, 3), (130, 70, 5, 5, 1, 1), (384, 96, 16, 4, 129, 24)])
def test_layer_matches_float64(mc, d, h, experts, top_k, prompt, batch):
    r = mx4_layer.run(d, h, experts, top_k, prompt, batch, steps=3)
    assert r["prompt_error"] <= BF16_ERROR
    assert r["projection_error"] <= BF16_ERROR
    assert r["experts_error"] <= BF16_ERROR
    assert r["router_gap"] <= 1e-4 and r["gate_error"] <= 1e-4
    # Rounding x to two or three significant bits: between a unit and a few hundredths.
    assert 0.01 < r["prompt_quantisation_error"] < 0.25


@pytest.mark.gpu
def test_command_prints_one_line(mc, capsys):
    assert mx4_layer.main(["--d", "128", "--h", "64", "--experts", "4", "--top-k", "2", "--prompt", "16", "--batch", "2",
                           "--steps", "2"]) == 0
    assert json.loads(capsys.readouterr().out)["decode_us"] > 0


def test_command_refuses_a_batch_beyond_the_operator():
    with pytest.raises(SystemExit):
        mx4_layer.main(["--batch", "65"])


def test_decoded_codes():
    import numpy as np

    codes = np.array([[0x21, 0xF7] + [0] * 62], dtype=np.uint8)
    scales = np.array([[128, 0, 0, 0]], dtype=np.uint8)
    assert mx4_layer.decoded(codes, scales, 5).tolist() == [[1.0, 2.0, 12.0, -12.0, 0.0]]
