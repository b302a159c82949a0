"""Which kernel a product of 8-bit integers runs (host logic, no GPU), on a chip of 256 CUs: the sizes that the GPU tests
give to each kernel reach it, so that a new rule cannot take a kernel out of them unseen."""

import ctypes

import pytest

import test_gpu_experts_i8 as experts
import test_gpu_i8 as operators
import test_gpu_i8_halves as halves

BLOCKS_16X32, BLOCKS_32X32, BLOCKS_32X64, TILES_128, TILES_256, TILES_FAR = range(6)


def dense(mc, m, n, k, gated):
    split = ctypes.c_int(-1)
    kernel = mc.library().mchip_matmul_i8_plan(2 if gated else 3, m, n, k, 256, ctypes.byref(split))
    return kernel, split.value


def on_plan(mc, down, gated, tokens, count, top_k, n, k):
    return mc.library().mchip_experts_i8_plan(int(down), 2 if gated else 3, tokens, top_k, count, n, k, 256)


DENSE = [BLOCKS_16X32, BLOCKS_32X32, BLOCKS_32X64, BLOCKS_32X64, BLOCKS_32X64, TILES_128, TILES_128, TILES_128, TILES_128,
         TILES_128, TILES_256, TILES_128]


@pytest.mark.parametrize("at", range(len(operators.VARIANTS)))
def test_dense_sizes_of_every_kernel(mc, at):
    m, n, k = operators.VARIANTS[at]
    assert dense(mc, m, n, k, False) == (DENSE[at], 0)
    assert dense(mc, m, n // 2, k, True) == (DENSE[at], 0)


@pytest.mark.parametrize("m,n,k,act,count", halves.SIZES)
def test_dense_sizes_with_halves(mc, m, n, k, act, count):
    assert dense(mc, m, n, k, act == "swiglu") == (TILES_256, count)


EXPERTS = [BLOCKS_32X64, BLOCKS_32X32, BLOCKS_16X32, BLOCKS_32X64, TILES_128, TILES_128, TILES_128, TILES_128, TILES_128,
           TILES_256, TILES_256]


@pytest.mark.parametrize("at", range(len(experts.VARIANTS)))
def test_plans_of_every_kernel(mc, at):
    tokens, count, top_k, n, k, _ = experts.VARIANTS[at]
    for down, gated, columns in ((False, False, n), (False, True, n // 2), (True, False, n)):
        assert on_plan(mc, down, gated, tokens, count, top_k, columns, k) == EXPERTS[at]


@pytest.mark.parametrize("m,n,k,kernel,split", [
    (1, 4096, 4096, BLOCKS_16X32, 0), (32, 4096, 4096, BLOCKS_16X32, 0), (256, 4096, 4096, BLOCKS_32X64, 0),
    (512, 4096, 4096, TILES_128, 0), (4096, 4096, 4096, TILES_256, 0), (8192, 8192, 8192, TILES_256, 0),
    (4096, 14336, 4096, TILES_256, 128), (1, 1, 1, BLOCKS_16X32, 0)])
def test_the_rule(mc, m, n, k, kernel, split):
    assert dense(mc, m, n, k, False) == (kernel, split)


# Gathered rows whose bytes reach 2 GiB: as large tiles as below it, from one row to the next, and never more blocks than
# a launch takes.
@pytest.mark.parametrize("tokens,count,top_k,n,k,gated,kernel", [
    (524287, 64, 8, 2048, 4096, True, TILES_256), (524288, 64, 8, 2048, 4096, True, TILES_FAR),
    (524288, 8, 2, 14336, 4096, True, TILES_FAR), (1 << 27, 8, 8, 128, 128, False, TILES_FAR),
    (16383, 4, 2, 1000, 131071, False, TILES_256), (16384, 4, 2, 1000, 131071, False, TILES_FAR),
    (2000000, 512, 16, 4096, 4096, True, TILES_FAR)])
def test_gathered_rows_past_2_gib(mc, tokens, count, top_k, n, k, gated, kernel):
    assert on_plan(mc, False, gated, tokens, count, top_k, n, k) == kernel
    # The second product reads its rows in their order, wherever they lie.
    assert on_plan(mc, True, False, tokens, count, top_k, n, k) in (TILES_128, TILES_256)
