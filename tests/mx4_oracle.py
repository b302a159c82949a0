"""The microscaled 4-bit format and the mixture-of-experts MLP in float64 numpy, with error bounds of the kernels'
arithmetic (fp32 sums of exact products), for the tests."""

from __future__ import annotations

import numpy as np

from helpers import U32, gamma

F32, BF16, F16, MX4 = 0, 1, 2, 4
TYPES = {"f32": F32, "bf16": BF16, "f16": F16}
UNIT = {F32: U32, BF16: 2.0 ** -8, F16: 2.0 ** -11}  # the largest relative error of rounding to the type
TINY = {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25}  # ... below its smallest normal number
MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def to_type(x, dtype: int) -> np.ndarray:
    """The array as the type's bits (fp32: floats), rounded to nearest even."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    if dtype == F32:
        return x
    if dtype == F16:
        return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32)
    r = ((u + np.uint32(0x7FFF) + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_type(bits, dtype: int) -> np.ndarray:
    if dtype == F32:
        return np.asarray(bits, dtype=np.float32).astype(np.float64)
    if dtype == F16:
        return np.asarray(bits).view(np.float16).astype(np.float64)
    return (np.asarray(bits).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def padded(k: int) -> int:
    return (k + 127) // 128 * 128


def quantize(x):
    """Rows x [rows, k] (float64) to (codes [rows, kp / 2], scales [rows, kp / 32], values [rows, k])."""
    rows, k = x.shape
    b = np.zeros((rows, padded(k)))
    b[:, :k] = x
    b = b.reshape(rows, -1, 32)
    top = np.max(np.abs(b), axis=-1)
    lost = ~np.isfinite(top)
    top = np.where(lost, 1.0, top)
    scale = np.where(top > 0, np.frexp(top)[1] - 1 - 2 + 127, 0)
    scale = np.maximum(scale, 0)
    with np.errstate(invalid="ignore"):
        v = np.where(lost[..., None], 0.0, np.ldexp(np.abs(b), (127 - scale)[..., None]))
    # Halfway between two codes the even one: below and at .25, from .75 on, ...
    code = ((v > 0.25).astype(int) + (v >= 0.75) + (v > 1.25) + (v >= 1.75) + (v > 2.5) + (v >= 3.5) + (v > 5.0))
    sign = np.signbit(b) & ~lost[..., None]
    scale = np.where(lost, 255, scale)
    code = (code | (sign.astype(int) << 3)).astype(np.uint8).reshape(rows, -1)
    packed = code[:, 0::2] | (code[:, 1::2] << 4)
    return packed, scale.astype(np.uint8), decode(packed, scale, k)


def decode(packed, scales, k: int):
    code = np.empty((packed.shape[0], packed.shape[1] * 2), dtype=np.uint8)
    code[:, 0::2] = packed & 15
    code[:, 1::2] = packed >> 4
    v = MAGNITUDES[code & 7] * np.where(code & 8, -1.0, 1.0)
    s = np.asarray(scales, dtype=np.int64)
    f = np.where(s == 255, np.nan, np.ldexp(1.0, s - 127))
    return (v * np.repeat(f, 32, axis=1))[:, :k]


def product_bound(a, b, k: int, dtype: int):
    """(exact, bound) of fp32 sums of exact products of the rows of a and b, rounded to dtype."""
    exact, absdot = a @ b.T, np.abs(a) @ np.abs(b).T
    err = gamma(padded(k)) * absdot
    return exact, err + rounding(exact, err, dtype)


def rounding(value, err, dtype: int):
    return UNIT[dtype] * (np.abs(value) + err) + TINY[dtype]


def activate(u, act: str):
    if act == "relu":
        return np.maximum(u, 0.0)
    if act == "gelu":
        return 0.5 * u * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * (u + 0.044715 * u ** 3)))
    gate, up = np.split(u, 2)
    return gate / (1.0 + np.exp(-gate)) * up


def route(x, router, top_k: int, normalize: bool):
    """(chosen, gates, smallest gap between neighbouring logits that decide, relative error bound of the gates)."""
    logits = x @ router.T
    absdot = np.abs(x) @ np.abs(router).T
    order = np.argsort(-logits, axis=1, kind="stable")
    chosen = order[:, :top_k]
    p = np.exp(logits - logits.max(axis=1, keepdims=True))
    p /= p.sum(axis=1, keepdims=True)
    gates = np.take_along_axis(p, chosen, axis=1)
    if normalize:
        gates = gates / gates.sum(axis=1, keepdims=True)
    ranked = np.take_along_axis(logits, order, axis=1)
    gaps = np.diff(-ranked[:, :top_k + 1], axis=1)
    off = gamma(padded(x.shape[1])) * absdot.max()
    # Each logit is off by `off`; the difference to the largest by twice that and a rounding; then exp, sums, quotients.
    relative = 2 * (2 * off + U32 * np.abs(logits).max() * 2) + 64 * U32
    return chosen, gates, (gaps.min() if gaps.size else np.inf), off, relative


def moe(x, w1, b1, w2, b2, chosen, gates, act: str, gate_err: float, dtype: int):
    """(y, bound): x [tokens, d], w1 [experts, rows, d], w2 [experts, d, h] in float64. The bound follows fp32 sums
    of exact products through the activation (slopes at most 1.13 for GELU, 1.1 for SiLU; its functions within 16
    units), h cut to 16 bits (24 for fp32), and the second sums."""
    tokens, d = x.shape
    h = w2.shape[2]
    y, bound = np.zeros((tokens, d)), np.zeros((tokens, d))
    cut = 2.0 ** -23 if dtype == F32 else 2.0 ** -15
    for t in range(tokens):
        for e, g in zip(chosen[t], gates[t]):
            u, du = w1[e] @ x[t], gamma(padded(d) + 1) * (np.abs(w1[e]) @ np.abs(x[t]))
            if b1 is not None:
                u = u + b1[e]
                du = du + U32 * (np.abs(u) + np.abs(b1[e]) + du)
            a = activate(u, act)
            if act == "swiglu":
                gate, up = np.split(u, 2)
                dgate, dup = np.split(du, 2)
                silu = gate / (1.0 + np.exp(-gate))
                da = 1.1 * dgate * (np.abs(up) + dup) + np.abs(silu) * dup + 16 * U32 * np.abs(a)
            else:
                # GELU's own argument is a polynomial: its rounding matters where tanh is steep.
                da = 1.13 * du + 16 * U32 * (np.abs(a) + np.abs(u) * (act == "gelu"))
            da = da + cut * np.abs(a)
            o = w2[e] @ a
            do = np.abs(w2[e]) @ da + gamma(padded(h) + 16) * (np.abs(w2[e]) @ (np.abs(a) + da))
            if b2 is not None:
                o = o + b2[e]
                do = do + U32 * (np.abs(o) + np.abs(b2[e]) + do)
            y[t] += g * o
            bound[t] += abs(g) * do + abs(g) * gate_err * (np.abs(o) + do) + 24 * U32 * abs(g) * (np.abs(o) + do)
    return y, bound + rounding(y, bound, dtype)
