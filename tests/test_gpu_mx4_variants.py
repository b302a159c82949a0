"""Products of 4-bit operands on the GPU at the sizes that lead to each compiled form of a kernel (on 256 CUs): columns
per block, a second step of k for every wave, 16-bit and fp32 rows and results, rows at odd distances."""

import numpy as np
import pytest

import mx4_oracle as ref
from test_gpu_mx4 import Out, bits_type, device_rows, operand, upload_at, within

pytestmark = pytest.mark.gpu


# Columns for blocks of 32 by few rows and, of 64, by none; two rows of blocks; 64x64 and 32x64 blocks; k past one step for each
# of eight waves.
@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("m,n,k", [(1, 8200, 300), (16, 14336, 1100), (7, 16321, 130), (17, 8200, 300), (32, 14336, 1100),
                                   (30, 16321, 130), (64, 4100, 1100), (1000, 1001, 1100), (700, 1030, 1100),
                                   (40, 700, 2200)])
def test_quantised_operands(device, mc, kind, m, n, k):
    print(f"case mx4 product {kind} {m}x{n}x{k}", flush=True)
    dtype = ref.TYPES[kind]
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    ac, as_, a = operand(mc, rng, m, k)
    bc, bs, b = operand(mc, rng, n, k, k ** -0.5)
    c = Out(mc, m * n * (4 if dtype == ref.F32 else 2))
    mc.launch_matmul_mx4(ac.ptr, as_.ptr, bc.ptr, bs.ptr, dtype, c.ptr, m, n, k)
    mc.synchronize()
    exact, bound = ref.product_bound(a, b, k, dtype)
    within(ref.from_type(c.get(bits_type(dtype), (m, n)), dtype), exact, bound)


# Few rows by 16, 32 and 64 columns a block, at even and odd distances, k past a step for each of 16 waves; up to 64 rows.
@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("m,n,k,pad", [(1, 14336, 2100, 0), (2, 14336, 300, 1), (9, 8200, 300, 1), (16, 14336, 2100, 0),
                                       (16, 14336, 2101, 2), (12, 4200, 2100, 3), (16, 8200, 2100, 0), (32, 14336, 1100, 0),
                                       (20, 8200, 1101, 1), (64, 8192, 2048, 0), (33, 4200, 1101, 0), (64, 4096, 2200, 0),
                                       (16, 4096, 2100, 0), (11, 1000, 2201, 1), (20, 8000, 1100, 2), (33, 1000, 1100, 0),
                                       (40, 5000, 1100, 2), (5, 300, 700, 0), (5, 300, 701, 0), (9, 8200, 300, 0),
                                       (100, 300, 129, 0), (130, 4500, 201, 0), (2050, 2060, 390, 0),
                                       (9, 8000, 300, 0), (20, 1000, 300, 0)])
def test_quantised_weights(device, mc, kind, m, n, k, pad):
    print(f"case mx4 weights {kind} {m}x{n}x{k} pad {pad}", flush=True)
    dtype = ref.TYPES[kind]
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    bits = ref.to_type(rng.standard_normal((m, k)) * np.exp(rng.standard_normal(k)), dtype)
    a = device_rows(mc, bits, k + pad)
    bc, bs, b = operand(mc, rng, n, k, k ** -0.5)
    workspace = mc.DeviceBuffer(max(1, mc.matmul_mx4_weights_workspace_bytes(dtype, m, n, k)))
    for out in (ref.F32, ref.BF16, ref.F16):
        c = Out(mc, m * n * (4 if out == ref.F32 else 2))
        mc.launch_matmul_mx4_weights(dtype, a.ptr, k + pad, bc.ptr, bs.ptr, out, c.ptr, m, n, k, None, workspace.ptr)
        mc.synchronize()
        # Up to three pieces of A per product.
        exact, bound = ref.product_bound(ref.from_type(bits, dtype), b, 3 * k, out)
        within(ref.from_type(c.get(bits_type(out), (m, n)), out), exact, bound)


@pytest.mark.parametrize("n", [40, 8200])
def test_few_fp32_rows_more_than_2_gib_apart(device, mc, n):
    m, k, lda = 2, 200, (1 << 29) + 3
    print(f"case mx4 weights, fp32 rows far apart {n}", flush=True)
    rng = np.random.default_rng(n)
    bits = ref.to_type(rng.standard_normal((m, k)), ref.F32)
    a = mc.DeviceBuffer(4 * ((m - 1) * lda + k))
    for i in range(m):
        upload_at(mc, a, 4 * i * lda, bits[i])
    bc, bs, b = operand(mc, rng, n, k)
    for out in (ref.F32, ref.BF16, ref.F16):
        c = Out(mc, m * n * (4 if out == ref.F32 else 2))
        mc.launch_matmul_mx4_weights(ref.F32, a.ptr, lda, bc.ptr, bs.ptr, out, c.ptr, m, n, k)
        mc.synchronize()
        exact, bound = ref.product_bound(ref.from_type(bits, ref.F32), b, 3 * k, out)
        within(ref.from_type(c.get(bits_type(out), (m, n)), out), exact, bound)
