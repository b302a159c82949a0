"""A call after another call's failure: the HIP runtime remembers the last error of a thread, which is not this call's."""

import numpy as np
import pytest

import mx4_oracle as ref
import test_gpu_moe as experts
import test_gpu_mx4 as operators

pytestmark = pytest.mark.gpu


@pytest.fixture
def failed(device, mc):
    """A copy to nowhere, refused by the runtime; forgotten after the test."""
    a = np.zeros(4, dtype=np.float32)

    def fail():
        assert mc.library().mc_memcpy_htod(None, a.ctypes.data, a.nbytes) != 0

    yield fail
    mc.library().hipGetLastError()  # of the runtime that the library is linked with


@pytest.mark.parametrize("columns", [False, True])
def test_quantisation(mc, failed, columns, monkeypatch):
    rng = np.random.default_rng(1)
    before(mc, monkeypatch, "quantize_mx4_columns" if columns else "quantize_mx4", failed)
    operators.check_quantize(mc, rng.standard_normal((5, 200)), ref.F32, columns=columns)


@pytest.mark.parametrize("m", [3, 200])
def test_product(mc, failed, m, monkeypatch):
    before(mc, monkeypatch, "launch_matmul_mx4", failed)
    operators.test_product_of_quantised_operands(None, mc, "f32", m, 100, 300)


@pytest.mark.parametrize("m", [3, 20, 200, 2050])
def test_weights(mc, failed, m, monkeypatch):
    before(mc, monkeypatch, "launch_matmul_mx4_weights", failed)
    operators.test_product_with_quantised_weights(None, mc, "bf16", m, 2060 if m == 2050 else 100, 200, 0)


def test_experts(mc, failed, monkeypatch):
    before(mc, monkeypatch, "launch_moe", failed)
    experts.check(mc, 1, "bf16", ref.MX4, 5, 96, 80, 6, 2, "swiglu")


def before(mc, monkeypatch, name, fail):
    """The package's function with a failure before each call."""
    call = getattr(mc, name)

    def both(*args, **kw):
        fail()
        return call(*args, **kw)

    monkeypatch.setattr(mc, name, both)
