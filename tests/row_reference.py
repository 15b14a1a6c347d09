"""Plain 64-bit forms of the row operators, and what their tests share."""
from __future__ import annotations

import numpy as np

from darknet_amd import api

F32, F16, BF16, I8 = 0, 1, 2, 3
# half a step of the type, relative to the value
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
# half of the smallest step there is (what is left of a value below the normal range)
HALF_TINY = {F32: 2.0 ** -150, F16: 2.0 ** -25, BF16: 2.0 ** -134}


def to_type(x, t):
    """The bits of float32 values rounded to a type (nearest even)."""
    x = np.ascontiguousarray(x, np.float32)
    if t == F32:
        return x
    if t == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    b = x.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_type(bits, t):
    """float32 values of what to_type made."""
    if t == F32:
        return bits
    if t == F16:
        return bits.astype(np.float32)
    return (bits.astype(np.uint32) << 16).view(np.float32)


class Buffer:
    """Device memory of any element type, with room in front (to shift its alignment) and a guard behind."""

    GUARD = 64

    def __init__(self, data=None, shape=None, dtype=None, shift=0):
        data = np.full(shape, 0, dtype) if data is None else np.ascontiguousarray(data)
        if shape is not None:   # an output: its old contents must not pass for a result
            data = np.frombuffer(b"\xa5" * data.nbytes, data.dtype).reshape(data.shape)
        self.shape, self.dtype, self.nbytes, self.shift = data.shape, data.dtype, data.nbytes, shift
        raw = b"\x5a" * shift + data.tobytes() + b"\x5a" * self.GUARD
        raw += b"\x5a" * (-len(raw) % 4)
        self.raw = len(raw)
        self.mem = api.DeviceArray(np.frombuffer(raw, np.int32), dtype=np.int32)
        self.ptr = self.mem.ptr + shift

    def get(self):
        raw = self.mem.numpy().tobytes()
        assert raw[:self.shift] == b"\x5a" * self.shift, "memory in front of a buffer was written"
        assert set(raw[self.shift + self.nbytes:]) == {0x5A}, "memory behind a buffer was written"
        return np.frombuffer(raw[self.shift:self.shift + self.nbytes], self.dtype).reshape(self.shape).copy()


STORE = {F32: np.float32, F16: np.float16, BF16: np.uint16}


# ---- norm ------------------------------------------------------------------------------------
def rmsnorm(x, add, scales, eps, t):
    """(s as stored, y in 64 bits) for the bits x, add of type t."""
    s = from_type(x, t)
    if add is not None:
        with np.errstate(over="ignore", invalid="ignore"):
            s = s + from_type(add, t)
        s = from_type(to_type(s, t), t)
    v = s.astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        y = v / np.sqrt((v * v).mean(1, keepdims=True) + np.float64(np.float32(eps)))
        return s, y if scales is None else y * scales.astype(np.float64)


def q8(y, group):
    """(codes, scales) of rows of 64-bit values."""
    rows, n = y.shape
    group = group or n
    groups = -(-n // group)
    codes, scales = np.zeros((rows, n), np.int8), np.zeros((rows, groups), np.float32)
    for g in range(groups):
        v = y[:, g * group:(g + 1) * group]
        c = (np.abs(v).max(1) / 127).astype(np.float32)
        c[~np.isfinite(v).all(1)] = np.nan
        scales[:, g] = c
        ok = c > 0
        codes[ok, g * group:(g + 1) * group] = np.clip(np.rint(v[ok] / c[ok, None].astype(np.float64)), -127, 127)
    return codes, scales


# ---- 4-bit weights ---------------------------------------------------------------------------
def q4_codes(seed, outputs, inputs, group, zeros=True):
    """(codes 0..15, scales, zeros) of a layer."""
    r = np.random.default_rng(seed)
    groups = -(-inputs // group)
    codes = r.integers(0, 16, (outputs, inputs), dtype=np.uint8)
    scales = ((0.5 + r.random((outputs, groups))) * 0.02).astype(np.float32)
    return codes, scales, r.integers(0, 16, (outputs, groups), dtype=np.uint8) if zeros else None


def q4_bytes(codes):
    """Two codes to a byte, the even input in the lower half; what an odd length leaves over is set to ones."""
    outputs, inputs = codes.shape
    even, odd = codes[:, 0::2], np.full((outputs, (inputs + 1) // 2), 15, np.uint8)
    odd[:, :inputs // 2] = codes[:, 1::2]
    return even | (odd << 4)


def q4_weights(codes, scales, zeros, group):
    """The weights in 64 bits."""
    at = np.arange(codes.shape[1]) // group
    z = 8.0 if zeros is None else zeros.astype(np.float64)[:, at]
    return (codes.astype(np.float64) - z) * scales.astype(np.float64)[:, at]


ACTIVATE = {3: lambda v: v, 1: lambda v: v * (v > 0), 7: lambda v: np.where(v > 0, v, .1 * v),
            0: lambda v: 1 / (1 + np.exp(-v))}


def q4_products(x, w, bias, activation):
    y = x @ w.T
    return ACTIVATE[activation](y if bias is None else y + bias.astype(np.float64))


def q4_bound(x, w, group, t_out, y, bias=None):
    """How far an output may be off: the input is held in fixed point relative to the largest of its group
    (to 2^-22 of it, to 2^-15 where the output has 16 bits), products within a group are exact, and each of
    the groups, the bias and the epilogue rounds to 2^-24 of what has been added up."""
    k = x.shape[1]
    step = 2.0 ** -22 if t_out == F32 else 2.0 ** -15
    held = np.zeros_like(y)
    for lo in range(0, k, group):
        top = np.abs(x[:, lo:lo + group]).max(1)
        held += step * top[:, None] * np.abs(w[:, lo:lo + group]).sum(1)[None]
    size = np.abs(x) @ np.abs(w).T + (0 if bias is None else np.abs(bias.astype(np.float64)))
    rounds = (-(-k // group) + 16) * 2.0 ** -24
    return held + rounds * size + HALF_STEP[t_out] * np.abs(y) * 1.01 + HALF_TINY[t_out]


# ---- sampling --------------------------------------------------------------------------------
def sample(logits, temperature, top_k, top_p, min_p, uniform):
    """(token, probability, margin) of one row of float32 logits; the margin is how near to a border, relative to
    the mass, the draw and the nucleus' end lie (a result within 1e-9 of one says nothing)."""
    n = len(logits)
    l = logits.astype(np.float64)
    l[np.isnan(l)] = -np.inf
    order = np.lexsort((np.arange(n), -l))
    order = order[l[order] > -np.inf]
    if not len(order):
        return -1, 0.0, 1.0
    greedy = not temperature > 0
    top = l[order[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(l[order] == top, 1.0, np.exp((l[order] - top) / (1.0 if greedy else np.float64(temperature))))
    if greedy:
        top_k = 1
    margin = 1.0
    if top_k > 0:
        w = w[:top_k]
    if top_p < 1:
        running, target = np.cumsum(w), np.float64(top_p) * w.sum()
        margin = np.abs(running - target).min() / w.sum()
        w = w[:max(1, int((running < target).sum()) + 1)]
    if min_p > 0:
        w = w[w >= min(np.float64(min_p), 1.0)]
    at = np.argsort(order[:len(w)], kind="stable")
    running, total = np.cumsum(w[at]), w.sum()
    u = min(max(np.float64(uniform), 0.0), 1.0) if uniform == uniform else 0.0
    if 0 < u < 1:
        margin = min(margin, np.abs(running - u * running[-1]).min() / total)
    pick = at[int((running < u * running[-1]).sum())]
    return int(order[pick]), float(w[pick] / total), margin
