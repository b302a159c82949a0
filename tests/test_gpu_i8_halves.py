"""Products of 8-bit integers on 256x256 tiles whose last round has too few for the chip, so that its tiles run as two of
128 rows, on the GPU against float64: whole and short last rows among them, columns in eights and not, SwiGLU."""

import ctypes

import pytest

import i8_oracle as ref
from test_gpu_i8 import check_product

pytestmark = pytest.mark.gpu

# m, n, k, activation, tiles that run as halves on 256 CUs. Behind the last whole 256 rows of m: 40, 140, all of them.
SIZES = [(9000, 4352, 1700, None, 100), (9000, 4346, 1700, "gelu", 100), (9100, 4352, 1800, "relu", 100),
         (9100, 4346, 1800, None, 100), (9000, 2176, 1700, "swiglu", 100), (9100, 2170, 1700, "swiglu", 100),
         (8300, 8150, 1600, None, 32), (4096, 14336, 900, None, 128), (4000, 7168, 900, "swiglu", 128)]


@pytest.mark.parametrize("m,n,k,act,halves", SIZES)
def test_tiles_that_run_as_halves(device, mc, m, n, k, act, halves):
    split = ctypes.c_int(-1)
    mc.library().mchip_matmul_i8_plan(2 if act == "swiglu" else 3, m, n, k, device["cu_count"], ctypes.byref(split))
    assert split.value > 0
    for kind in sorted(ref.TYPES) if (m, n) in ((9000, 4352), (9100, 2170)) else ("bf16",) if n % 8 else ("f32",):
        print(f"case halves {kind} {m}x{n}x{k} {act} {split.value}", flush=True)
        check_product(mc, m + n + k, m, n, k, kind, act, bias=act is not None)
