"""A layer on 4-bit weights served end to end: a projection and a mixture-of-experts MLP.

    python -m minicompiler_amd.mx4_layer [--d 2048] [--h 1024] [--experts 64] [--top-k 8]
                                         [--prompt 512] [--batch 4] [--steps 100]

At load the weights, made in fp32 as a model file holds them ([k, n], as the matmuls take B), are quantised on the GPU
with quantize_mx4_columns: one mx4 operand for the projection, one per expert and matrix for the SwiGLU experts, side
by side in one array as launch_moe reads them. Then

  prompt   x [prompt, d] in bf16 is quantised by rows and multiplied by the quantised projection (launch_matmul_mx4);
  decode   x [batch, d] in bf16 goes through the projection as it is (launch_matmul_mx4_weights) and through the
           experts, router included (launch_moe), captured once into a HIP graph and replayed for every step.

Each part's output is compared with the same function in float64 on the host, of the same quantised numbers, and its
time printed, per call over the steps. All on synthetic data."""

from __future__ import annotations

import argparse
import json
import sys

import numpy as np

import minicompiler_amd as mc

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def bf16(x: np.ndarray) -> np.ndarray:
    """Finite fp32 rounded to bf16 bits."""
    u = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32)
    return ((u + np.uint32(0x7FFF) + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def wide(bits: np.ndarray) -> np.ndarray:
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def decoded(codes: np.ndarray, scales: np.ndarray, k: int) -> np.ndarray:
    """mx4 rows as float64."""
    four = np.stack([codes & 15, codes >> 4], axis=-1).reshape(codes.shape[0], -1)
    values = MAGNITUDES[four & 7] * np.where(four & 8, -1.0, 1.0)
    return (values * np.repeat(np.ldexp(1.0, scales.astype(int) - 127), 32, axis=1))[:, :k]


class Quantised:
    """`count` matrices [k, n] as mx4 operands of n rows each, one after the other."""

    def __init__(self, count: int, k: int, n: int):
        self.count, self.k, self.n = count, k, n
        self.codes = mc.DeviceBuffer(mc.mx4_code_bytes(count * n, k))
        self.scales = mc.DeviceBuffer(mc.mx4_scale_bytes(count * n, k))

    def put(self, i: int, weights: mc.DeviceBuffer, stream=None) -> None:
        """Matrix i from fp32 [k, n] on the device."""
        mc.quantize_mx4_columns(mc.DTYPE_F32, weights.ptr, self.n, self.codes.ptr + mc.mx4_code_bytes(i * self.n, self.k),
                                self.scales.ptr + mc.mx4_scale_bytes(i * self.n, self.k), self.k, self.n, stream=stream)

    def host(self) -> np.ndarray:
        rows = self.count * self.n
        return decoded(self.codes.download(np.uint8, mc.mx4_code_bytes(rows, self.k)).reshape(rows, -1),
                       self.scales.download(np.uint8, mc.mx4_scale_bytes(rows, self.k)).reshape(rows, -1), self.k)


def quantised(rng, count: int, k: int, n: int) -> Quantised:
    out = Quantised(count, k, n)
    for i in range(count):
        w = mc.DeviceBuffer.from_array((rng.standard_normal((k, n)) * k ** -0.5).astype(np.float32))
        out.put(i, w)
        mc.synchronize()  # before its memory goes
    return out


def timed(stream: mc.Stream, call, steps: int) -> float:
    """Microseconds per call."""
    for _ in range(max(3, steps // 5)):
        call()
    first, last = mc.Event(), mc.Event()
    first.record(stream)
    for _ in range(steps):
        call()
    last.record(stream)
    stream.synchronize()
    return first.elapsed_ms(last) * 1e3 / steps


def difference(got: np.ndarray, want: np.ndarray) -> float:
    return float(np.linalg.norm(got - want) / np.linalg.norm(want))


def run(d: int, h: int, experts: int, top_k: int, prompt: int, batch: int, steps: int, seed: int = 0) -> dict:
    rng = np.random.default_rng(seed)
    stream = mc.Stream()
    projection = quantised(rng, 1, d, d)
    # An expert's gate and up rows lie together: SwiGLU's W1 is [2 h, d].
    up, down = quantised(rng, experts, d, 2 * h), quantised(rng, experts, h, d)
    router = (rng.standard_normal((experts, d)) * d ** -0.5).astype(np.float32)
    device_router = mc.DeviceBuffer.from_array(router)
    result = {"d": d, "h": h, "experts": experts, "top_k": top_k, "prompt": prompt, "batch": batch, "data": "synthetic"}

    # The prompt.
    x = bf16(rng.standard_normal((prompt, d)))
    device_x = mc.DeviceBuffer.from_array(x)
    codes, scales = mc.DeviceBuffer(mc.mx4_code_bytes(prompt, d)), mc.DeviceBuffer(mc.mx4_scale_bytes(prompt, d))
    y = mc.DeviceBuffer(prompt * d * 2)

    def prefill():
        mc.quantize_mx4(mc.DTYPE_BF16, device_x.ptr, d, codes.ptr, scales.ptr, prompt, d, stream=stream)
        mc.launch_matmul_mx4(codes.ptr, scales.ptr, projection.codes.ptr, projection.scales.ptr, mc.DTYPE_BF16, y.ptr,
                             prompt, d, d, stream)

    result["prompt_us"] = timed(stream, prefill, steps)
    weights = projection.host()
    quantised_x = decoded(codes.download(np.uint8).reshape(prompt, -1), scales.download(np.uint8).reshape(prompt, -1), d)
    got = wide(y.download(np.uint16).reshape(prompt, d))
    result["prompt_error"] = difference(got, quantised_x @ weights.T)
    result["prompt_quantisation_error"] = difference(got, wide(x) @ weights.T)

    # A decoding step.
    x = bf16(rng.standard_normal((batch, d)))
    device_x = mc.DeviceBuffer.from_array(x)
    projected, y = mc.DeviceBuffer(batch * d * 2), mc.DeviceBuffer(batch * d * 2)
    chosen, gates = mc.DeviceBuffer(batch * top_k * 4), mc.DeviceBuffer(batch * top_k * 4)
    product_space = mc.DeviceBuffer(mc.matmul_mx4_weights_workspace_bytes(mc.DTYPE_BF16, batch, d, d))
    moe_space = mc.DeviceBuffer(mc.moe_workspace_bytes(mc.DTYPE_BF16, batch, d, h, experts, top_k))
    moe_space.fill_bytes(0)
    mc.synchronize()

    def step(s):
        mc.launch_matmul_mx4_weights(mc.DTYPE_BF16, device_x.ptr, d, projection.codes.ptr, projection.scales.ptr,
                                     mc.DTYPE_BF16, projected.ptr, batch, d, d, s, product_space.ptr)
        mc.launch_moe(mc.DTYPE_BF16, projected.ptr, d, device_router.ptr, mc.DTYPE_MX4, up.codes.ptr, up.scales.ptr, None,
                      down.codes.ptr, down.scales.ptr, None, y.ptr, chosen.ptr, gates.ptr, batch, d, h, experts, top_k,
                      "swiglu", True, s, moe_space.ptr)

    graph = mc.CapturedGraph(stream, step)
    result["decode_us"] = timed(stream, graph.launch, steps)
    got = wide(projected.download(np.uint16).reshape(batch, d))
    result["projection_error"] = difference(got, wide(x) @ weights.T)
    w1, w2 = up.host().reshape(experts, 2 * h, d), down.host().reshape(experts, d, h)
    picked, gate = chosen.download(np.int32).reshape(batch, top_k), gates.download(np.float32).reshape(batch, top_k)
    logits = got @ router.astype(np.float64).T
    # A pick in place i is one of the i largest logits, but for their rounding.
    ranked = -np.sort(-logits, axis=1)[:, :top_k]
    result["router_gap"] = float(np.abs(np.take_along_axis(logits, picked, axis=1) - ranked).max())
    want = np.zeros((batch, d))
    for t in range(batch):
        p = np.exp(logits[t, picked[t]] - logits[t].max())
        for e, g in zip(picked[t], p / p.sum()):
            a, b = np.split(w1[e] @ got[t], 2)
            want[t] += g * (w2[e] @ (a / (1.0 + np.exp(-a)) * b))
        result["gate_error"] = max(result.get("gate_error", 0.0), float(np.abs(gate[t] - p / p.sum()).max()))
    result["experts_error"] = difference(wide(y.download(np.uint16).reshape(batch, d)), want)
    return result


def main(argv=None) -> int:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("d", 2048), ("h", 1024), ("experts", 64), ("top-k", 8), ("prompt", 512), ("batch", 4),
                        ("steps", 100)):
        p.add_argument("--" + name, type=int, default=value)
    a = p.parse_args(argv)
    if not 1 <= a.batch <= 64:
        p.error("a decoding step has 1 to 64 tokens")
    print(json.dumps(run(a.d, a.h, a.experts, a.top_k, a.prompt, a.batch, a.steps)))
    return 0


if __name__ == "__main__":
    sys.exit(main())
