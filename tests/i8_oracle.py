"""8-bit integer operands, the choice of experts and the experts' products on a plan in float64 numpy, with error bounds
of the kernels' arithmetic, for the tests."""

from __future__ import annotations

import numpy as np

from helpers import U32
from mx4_oracle import BF16, F16, F32, TINY, TYPES, UNIT, from_type, padded, to_type  # noqa: F401

ACTS = (None, "relu", "gelu", "swiglu")
EXP_ENDS = 1e-36  # the fp32 exponential passes its range where a sigmoid is below this


def quantize(x):
    """Rows x [rows, k] (float64, of at most 24 bits) to (codes int8 [rows, kp], scales fp32 [rows])."""
    rows, k = x.shape
    top = np.max(np.abs(x), axis=-1)
    lost = ~np.isfinite(top)
    with np.errstate(under="ignore"):
        scale = (np.where(lost, 0.0, top) / 127.0).astype(np.float32)
    s = scale.astype(np.float64)
    # A quotient of two 24-bit numbers is no nearer to a half, unless it is one, than 2^-33: float64 keeps its side.
    with np.errstate(invalid="ignore", over="ignore"):
        code = np.rint(np.where(lost[:, None], 0.0, x) / np.where(s > 0, s, 1.0)[:, None])
    code = np.where((s > 0)[:, None], np.clip(code, -127, 127), 0.0)
    codes = np.zeros((rows, padded(k)), dtype=np.int8)
    codes[:, :k] = code
    return codes, np.where(lost, np.float32(np.nan), scale)


def values(codes, scales, k, dtype):
    """What the codes stand for, as the type's bits: the product rounded to fp32, then to the type."""
    with np.errstate(invalid="ignore", over="ignore"):
        v = codes[:, :k].astype(np.float32) * np.asarray(scales, dtype=np.float32)[:, None]
    return to_type(v, dtype)


def sigmoid(z):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-z))


def scaled(a, sa, b, sb, bias):
    """(a b^T scaled + bias, its bound) for integer a [m, k], b [n, k]: the sum's rounding to fp32, two products and the
    bias, one rounding each."""
    s = (a.astype(np.float64) @ b.astype(np.float64).T) * sa.astype(np.float64)[:, None] * sb.astype(np.float64)
    err = 3.01 * U32 * np.abs(s) + 3 * 2.0 ** -149
    if bias is not None:
        s = s + bias.astype(np.float64)
        err = err + 1.01 * U32 * (np.abs(s) + err)
    return s, err


def activate(u, err, act):
    """(act(u), its bound) of fp32 numbers within err of u. An exponential of z is off by its last bits and by z rounded
    before, as is a constant: (2 |z| + 4) units; the rest of a sigmoid and the products around it 6 roundings."""
    if act == "relu":
        return np.maximum(u, 0.0), err
    if act == "gelu":
        z = 1.5957691216057308 * (u + 0.044715 * u ** 3)
        y = u * sigmoid(z)
        # |d/du| <= 1.13; z itself carries 6 roundings, which count like z's in the exponent.
        return y, 1.13 * err + U32 * (10 + 8 * np.abs(z)) * np.abs(y) + EXP_ENDS * np.abs(u)
    if act == "swiglu":
        n = u.shape[-1] // 2
        g, up, eg, eu = u[..., :n], u[..., n:], err[..., :n], err[..., n:]
        silu = g * sigmoid(g)
        y = silu * up
        e = 1.1 * eg * (np.abs(up) + eu) + eu * np.abs(silu) + U32 * (10 + 2 * np.abs(g)) * np.abs(y)
        return y, e + EXP_ENDS * np.abs(g * up)
    return u, err


def rounded(y, err, dtype):
    """The bound after rounding to the stored type."""
    return err + UNIT[dtype] * (np.abs(y) + err) * 1.001 + TINY[dtype] * 1.01


def route(logits, bias, top_k, score, groups, top_groups, group_best, normalize, scale):
    """(chosen, gates float64, keys): logits float64 [tokens, experts]."""
    bad = np.isnan(logits).any(-1)
    l = np.where(np.isnan(logits), -np.inf, logits)
    tokens, experts = l.shape
    with np.errstate(invalid="ignore", over="ignore"):
        if score == "softmax":
            top = l.max(-1, keepdims=True)
            e = np.where(top == -np.inf, 0.0, np.exp(l - np.where(top == -np.inf, 0.0, top)))
            e = np.where(l == -np.inf, 0.0, e)
            total = e.sum(-1, keepdims=True)
            s = np.where(total == 0, 0.0, e / np.where(total == 0, 1.0, total))
        else:
            s = sigmoid(l)
    if bias is None and (groups == 1 or group_best == 1):
        key = l.copy()
    else:
        with np.errstate(invalid="ignore"):
            key = np.where(l == -np.inf, -np.inf, s + (0.0 if bias is None else bias.astype(np.float64)))
        key = np.where(np.isnan(key), -np.inf, key)
    chosen = np.zeros((tokens, top_k), dtype=np.int32)
    each = experts // groups
    for t in range(tokens):
        allowed = range(experts)
        if groups > 1:
            with np.errstate(invalid="ignore"):
                sums = [np.sort(key[t, g * each:(g + 1) * each])[::-1][:group_best].sum() for g in range(groups)]
            sums = [-np.inf if np.isnan(x) else x for x in sums]
            kept = sorted(range(groups), key=lambda g: (-sums[g], g))[:top_groups]
            allowed = [e for e in range(experts) if e // each in kept]
        chosen[t] = sorted(allowed, key=lambda e: (-key[t, e], e))[:top_k]
    gates = np.take_along_axis(s, chosen, axis=1)
    if normalize:
        total = gates.sum(-1, keepdims=True)
        gates = np.where(total == 0, 0.0, gates / np.where(total == 0, 1.0, total))
    gates = gates * np.float64(np.float32(scale))
    gates[bad] = np.nan
    return chosen, gates, key


def plan(chosen, experts):
    """(order, offsets) of chosen [tokens, top_k]."""
    flat = chosen.reshape(-1)
    order = np.argsort(flat, kind="stable").astype(np.int32)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat, minlength=experts))]).astype(np.int32)
    return order, offsets


def experts_up(a, sa, w, sw, bias, act, order, offsets, top_k, dtype):
    """(C by slot, its bound): a int8 [tokens, kp], w int8 [experts, rows, kp]. NaN where no expert has the slot."""
    n = w.shape[1] // (2 if act == "swiglu" else 1)
    out, bound = np.full((len(order), n), np.nan), np.zeros((len(order), n))
    for e in range(len(w)):
        at = slice(offsets[e], offsets[e + 1])
        t = order[at] // top_k
        y, err = activate(*scaled(a[t], sa[t], w[e], sw[e], None if bias is None else bias[e]), act)
        out[at], bound[at] = y, rounded(y, err, dtype)
    return out, bound


def experts_down(a, sa, w, sw, bias, order, offsets, gates, top_k, dtype):
    """(y by token, its bound): a int8 [slots, kp]; gates [tokens, top_k] fp32."""
    tokens = len(order) // top_k
    y, size, err = (np.zeros((tokens, w.shape[1])) for _ in range(3))
    g = gates.reshape(-1).astype(np.float64)
    for e in range(len(w)):
        at = slice(offsets[e], offsets[e + 1])
        pair = order[at]
        u, eu = scaled(a[at], sa[at], w[e], sw[e], None if bias is None else bias[e])
        np.add.at(y, pair // top_k, u * g[pair, None])
        np.add.at(size, pair // top_k, np.abs(u * g[pair, None]))
        np.add.at(err, pair // top_k, eu * np.abs(g[pair, None]))
    # One rounding by the gate, top_k - 1 sums.
    err = err * 1.01 + 1.01 * (top_k + 1) * U32 * size + top_k * 2.0 ** -149
    return y, rounded(y, err, dtype)
