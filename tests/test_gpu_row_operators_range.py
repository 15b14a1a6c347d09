"""Row operators on the device where values of very different sizes meet, or lie on a border: products of rows with a few
large inputs, of small inputs and scales, 8-bit codes between two steps, one token far above many."""
import numpy as np
import pytest

import row_reference as R
from row_reference import BF16, F16, F32, Buffer
from test_gpu_row_operators import check_draw, draw

pytestmark = pytest.mark.gpu


class Weights:
    """A layer whose codes, scales and zeros are given."""

    def __init__(self, dn, codes, scales, zeros, group):
        (self.n, self.k), self.group = codes.shape, group
        self.w = R.q4_weights(codes, scales, zeros, group)
        self.packed = Buffer(shape=(dn.q4_packed_bytes(self.k, self.n, group),), dtype=np.uint8, shift=16)
        src = [Buffer(R.q4_bytes(codes)), Buffer(scales), Buffer(zeros)]
        assert dn.q4_pack_codes_gpu(src[0].ptr, src[1].ptr, src[2].ptr, self.packed.ptr, self.k, self.n, group) == 0
        dn.hip_synchronize()

    def product(self, dn, bits, tx, scales=None, x_group=0, t_out=F32, bias=None, act=3):
        """What the library gives for the rows `bits` of type tx."""
        batch = len(bits)
        size = dn.connected_q4_workspace_bytes(tx, batch, self.k, self.n, self.group)
        ws = Buffer(shape=(size,), dtype=np.uint8, shift=16) if size else None
        bx, bs, bb = Buffer(bits), Buffer(scales) if scales is not None else None, Buffer(bias) if bias is not None else None
        out = Buffer(shape=(batch, self.n), dtype=R.STORE[t_out])
        assert dn.forward_connected_q4_gpu(bx.ptr, tx, bs.ptr if bs else None, x_group, self.packed.ptr, bb.ptr if bb else None, out.ptr, t_out,
                                           batch, self.k, self.n, self.group, act, ws.ptr if ws else None) == 0
        dn.hip_synchronize()
        if ws:
            ws.get()
        return R.from_type(out.get(), t_out).astype(np.float64)


def single_weights(seed, n, k, group, scale=0.02):
    """(codes, scales, zeros, column of each output): each output has one weight that is not 0."""
    r = np.random.default_rng(seed)
    groups = -(-k // group)
    zeros = r.integers(0, 16, (n, groups), dtype=np.uint8)
    scales = ((0.5 + r.random((n, groups))) * scale).astype(np.float32)
    codes = zeros[:, np.arange(k) // group].copy()
    column = r.integers(0, k, n)
    codes[np.arange(n), column] = (codes[np.arange(n), column] + r.integers(1, 16, n)) % 16
    return codes, scales, zeros, column


# rows, inputs, outputs: few rows; 16 rows a workgroup; the inputs cut over workgroups; many outputs, one to four tiles of rows
FORMS = [(1, 700, 90), (4, 700, 90), (3, 5003, 3000), (5, 700, 90), (20, 700, 90), (5, 8200, 60), (5, 300, 40000), (20, 300, 20000), (40, 200, 14000), (64, 200, 11300)]


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("batch,k,n", FORMS)
def test_q4_every_value_keeps_its_bits(dn, batch, k, n, t, group):
    """Values of all sizes in a row, each alone in the outputs that have its weight: fp32 is held to 2^-23 of a value, the
    other types exactly; the sum of one product with the group's scale and the scaling takes at most four roundings more."""
    r = np.random.default_rng(batch + k + n)
    codes, scales, zeros, column = single_weights(k, n, k, group)
    low, high = (-24, 15.99) if t == F16 else (-110, 120)
    x = (np.sign(r.standard_normal((batch, k))) * 2.0 ** r.uniform(low, high, (batch, k))).astype(np.float32)
    x[:, r.random(k) < 0.02] = 0
    x[batch // 2] = r.standard_normal(k)                       # one row as usual
    bits = R.to_type(x, t)
    x = R.from_type(bits, t).astype(np.float64)
    m = Weights(dn, codes, scales, zeros, group)
    got = m.product(dn, bits, t)
    want = x[:, column] * m.w[np.arange(n), column]
    tol = np.abs(want) * ((2.0 ** -23 if t == F32 else 0) + 5 * 2.0 ** -24)
    bad = np.abs(got - want) > tol
    assert not bad.any(), (int(bad.sum()), float((np.abs(got - want) / np.maximum(np.abs(want), 1e-300)).max()))


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("batch", [1, 4, 5, 64])
@pytest.mark.parametrize("outlier", [1e6, 1e9, 2.0 ** 60, 3e38])
def test_q4_an_outlier_whose_weight_is_zero(dn, batch, outlier, t):
    """Ordinary rows and weights but for one large input that no output has.  Each value is held to 2^-23 (fp32), a group's
    sum takes a rounding for each of its eight matrix instructions and eight within one, and each group is added once."""
    k, n, group = 4096, 600, 128
    r = np.random.default_rng(batch)
    codes, scales, zeros = R.q4_codes(batch, n, k, group)
    x = r.standard_normal((batch, k)).astype(np.float32)
    for b in range(batch):
        at = 37 + 61 * b
        x[b, at] = outlier
        codes[:, at] = zeros[:, at // group]
    bits = R.to_type(x, t)
    x = R.from_type(bits, t).astype(np.float64)
    m = Weights(dn, codes, scales, zeros, group)
    got = m.product(dn, bits, t)
    want = x @ m.w.T
    size = np.abs(x) @ np.abs(m.w).T
    tol = size * ((2.0 ** -23 if t == F32 else 0) + (64 + k // group + 8) * 2.0 ** -24)
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / size).max() * 2 ** 24)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("batch", [1, 2, 4, 6, 30])
def test_q4_small_inputs_with_small_scales(dn, batch, group):
    """Rows near the least fp32 values, weights whose scales are small too: outputs are within the range of fp32 although
    the product of a row's factor and a scale is not.  Bounds as above; what is below the normal range has its own step."""
    k, n = 700, 45
    r = np.random.default_rng(batch + group)
    codes, scales, zeros = R.q4_codes(batch, n, k, group)
    for size, small in ((1e-33, 1e-3), (1e-36, 1.0), (1e-28, 1e-8), (1e-14, 1e-20), (1e-30, 1e20), (1e10, 1e-25)):
        sc = (scales * np.float32(small)).astype(np.float32)
        m = Weights(dn, codes, sc, zeros, group)
        x = (r.standard_normal((batch, k)) * size).astype(np.float32)
        got, want = m.product(dn, x, F32), x.astype(np.float64) @ m.w.T
        tol = np.abs(x.astype(np.float64)) @ np.abs(m.w).T * (2.0 ** -23 + (64 + -(-k // group) + 8) * 2.0 ** -24) + (k // group + 8) * 2.0 ** -149
        assert (np.abs(got - want) <= tol).all(), (size, small)
        # 8 bits: whole numbers, so that only scales and sums round
        bits = r.integers(-127, 128, (batch, k), dtype=np.int8)
        for xg in (0, group):
            xs = ((0.5 + r.random((batch, -(-k // xg) if xg else 1))) * size).astype(np.float32)
            v = bits * xs.astype(np.float64)[:, np.arange(k) // xg if xg else np.zeros(k, int)]
            got, want = m.product(dn, bits, R.I8, xs, xg), v @ m.w.T
            tol = np.abs(v) @ np.abs(m.w).T * (-(-k // group) + 16) * 2.0 ** -24 + (k // group + 8) * 2.0 ** -149
            assert (np.abs(got - want) <= tol).all(), (size, small, xg)


@pytest.mark.parametrize("batch", [1, 3, 5, 20])
@pytest.mark.parametrize("n", [40, 12000])
def test_q4_scales_of_8_bit_rows_that_are_not_finite(dn, batch, n):
    """A row with an infinite or NaN scale: all its sums are NaN, whatever its codes; the other rows are as without it."""
    k, group = 300, 32
    codes, scales, zeros = R.q4_codes(batch, n, k, group)
    m = Weights(dn, codes, scales, zeros, group)
    r = np.random.default_rng(n)
    bits = r.integers(-127, 128, (batch, k), dtype=np.int8)
    for value in (np.inf, -np.inf, np.nan):
        for xg in (0, group):
            xs = (0.5 + r.random((batch, -(-k // xg) if xg else 1))).astype(np.float32)
            fine = m.product(dn, bits, R.I8, xs, xg)
            xs[batch // 2, -1] = value
            got = m.product(dn, bits, R.I8, xs, xg)
            assert np.isnan(got[batch // 2]).all()
            rest = np.arange(batch) != batch // 2
            assert np.array_equal(got[rest], fine[rest])


# ---- norm ------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("n", [64, 300, 1000, 4096, 20000])
def test_norm_codes_between_two_steps(dn, n, t):
    """Rows whose root mean square is a whole number, scales that put values half-way between two steps: ties go to even."""
    r = np.random.default_rng(n)
    for rms in (1, 2, 3, 5, 7, 0.75):
        x = (rms * r.choice([-1, 1], (2, n))).astype(np.float32)
        for group in (0, 32, 128):
            g = np.empty(n, np.float32)
            for lo in range(0, n, group or n):
                part = g[lo:lo + (group or n)]
                step = np.float32(r.integers(1, 1 << 12) * 2.0 ** r.integers(-8, 3))
                part[:] = step * (r.integers(-127, 127, len(part)) + np.float32(0.5))
                part[r.integers(len(part))] = step * 127
            bx, bg = Buffer(R.to_type(x, t)), Buffer(g)
            q, c = Buffer(shape=(2, n), dtype=np.int8), Buffer(shape=(2, -(-n // (group or n))), dtype=np.float32)
            assert dn.forward_rmsnorm_gpu(bx.ptr, None, bg.ptr, None, None, q.ptr, c.ptr, t, 2, n, group, 0.0) == 0
            dn.hip_synchronize()
            _, y = R.rmsnorm(R.to_type(x, t), None, g, 0.0, t)
            assert np.array_equal(np.abs(y), np.abs(np.broadcast_to(g, y.shape)).astype(np.float64))    # exact
            codes, want = R.q8(y, group)
            assert np.array_equal(c.get(), want) and np.array_equal(q.get(), codes), (rms, group, int((q.get() != codes).sum()))


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("n", [40, 1000, 20000])
def test_norm_values_and_scales_of_all_sizes(dn, n, t):
    """Elements far below their row with large scales, large rows with small scales: the result is within the range of
    fp32, and right to two roundings, although a product on the way to it in 32 bits would not be."""
    r = np.random.default_rng(n)
    for size, small, scale in ((1.0, 1e-38, 1e6), (1e30, 1e-8, 1e-9), (1e-25, 1e-12, 1e20), (1e35, 1.0, 1e-30), (3e3, 1e-30, 1e12)):
        x = (r.standard_normal((3, n)) * size).astype(np.float32)
        x[:, r.random(n) < 0.5] *= np.float32(small)
        bits, g = R.to_type(x, t), ((0.5 + r.random(n)) * scale).astype(np.float32)
        bx, bg, out = Buffer(bits), Buffer(g), Buffer(shape=(3, n), dtype=bits.dtype)
        assert dn.forward_rmsnorm_gpu(bx.ptr, None, bg.ptr, None, out.ptr, None, None, t, 3, n, 0, 0.0) == 0
        dn.hip_synchronize()
        _, y = R.rmsnorm(bits, None, g, 0.0, t)
        tol = np.abs(y) * (R.HALF_STEP[t] + 4 * 2.0 ** -24) + R.HALF_TINY[t]
        assert (np.abs(R.from_type(out.get(), t) - y) <= tol).all(), (size, small, scale)


# ---- sampling --------------------------------------------------------------------------------
def mass_bits(n):
    """The largest token's weight is 2^this in a row of n tokens."""
    return min(48, 63 - max(1, (n - 1).bit_length()))


@pytest.mark.parametrize("n,below", [(5000, 20.0), (8192, 27.0), (30000, 24.0), (131072, 25.0), (262144, 27.05), (1 << 20, 26.0), (1500001, 24.0), (1 << 24, 22.0)])
@pytest.mark.parametrize("settings", ["none", "p", "min"])
def test_sample_one_token_above_a_flat_vocabulary(dn, n, below, settings):
    """One token, and all the others alike far below it, whose masses add up: each is a whole multiple of 2^-bits of the
    largest, so the share of the others is known to n * 2^-(bits + 1), and the place of a draw among them accordingly."""
    x = np.full((1, n), -below, np.float32)
    top = n // 3
    x[0, top] = 0
    w = np.exp(-np.float64(np.float32(below)))
    off = n * 2.0 ** -(mass_bits(n) + 1)
    total = 1 + (n - 1) * w
    u = np.float32([0.5, 1 - total ** -1 * (n - 1) * w * 0.5, 1 - 2.0 ** -24, total ** -1 * (top * w) * 0.5, 1.0])
    rows = np.repeat(x, len(u), 0) if n < 1 << 20 else x
    kw = dict(p=dict(top_p=[1 - 2.0 ** -24] * len(u)), min=dict(min_p=[w * 0.99] * len(u)), none={})[settings]
    kept = n - 1                                             # of the others
    if settings == "p":                                      # of the others the first by index
        kept = max(0, min(n - 1, int(np.ceil((float(np.float32(1 - 2.0 ** -24)) * total - 1) / w))))
    slack = off / w + 2
    place = lambda rank: rank if rank < top else rank + 1    # noqa: E731  (of the others, by index)
    for i in range(len(u)):
        one = {a: v[:1] for a, v in kw.items()}
        tok, prob = (draw(dn, rows[i:i + 1], F32, u[i:i + 1], **one) if len(rows) > 1 else draw(dn, x, F32, u[i:i + 1], **one))
        if u[i] == 0.5 or kept == 0:
            assert tok[0] == top
            share = 1 / (1 + kept * w)
            room = off + (slack * w if settings == "p" else 0)
            assert abs(prob[0] - share) <= 2.0 ** -24 + room
            continue
        mass = float(u[i]) * (1 + kept * w)
        rank = mass / w if mass < top * w else None if mass <= top * w + 1 else (mass - 1) / w
        if rank is None or (settings == "p" and abs(mass - top * w - 1) < 2 * off):
            continue
        room = slack * (2 if settings == "p" else 1) + float(u[i]) * 2.0 ** -52 * n
        assert abs(int(tok[0]) - place(min(kept - 1, max(0, int(rank))))) <= room + 1, (u[i], tok[0], rank)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("n", [(1 << 20) + 1, (1 << 21) + 5000, 1 << 24])
def test_sample_rows_beyond_a_million(dn, n, t):
    """Blocks of several strips of 2048 tokens: draws into the first, the second and the last strips of a block."""
    r = np.random.default_rng(n)
    x = (r.standard_normal((1, n)) * 2).astype(np.float32)
    x[0, r.integers(0, n, 40)] += 6
    held = R.from_type(R.to_type(x, t), t)[0].astype(np.float64)
    w = np.exp(held - held.max())
    running = np.cumsum(w)
    block = -(-n // (2048 * 512)) * 2048
    places = [0, 2047, 2048, block - 1, block, 3 * block + 2048 + 77, n - 1, (n // block) * block, n - n // 7]
    u = np.float32([(running[p] - 0.5 * w[p]) / running[-1] for p in places if p < n])
    off = n * 2.0 ** -(mass_bits(n) + 1) + 2.0 ** -24 * running[-1]     # of masses; u in 32 bits
    for one in u:
        tok, prob = draw(dn, x, t, [one])
        lo, hi = np.searchsorted(running, float(one) * running[-1] - off), np.searchsorted(running, float(one) * running[-1] + off)
        assert lo <= tok[0] <= hi
        assert abs(prob[0] - w[tok[0]] / running[-1]) <= 2.0 ** -24 + off
    # borders among a few, among many and among equal tokens
    for kw in (dict(top_k=[50]), dict(top_p=[0.4]), dict(top_k=[n // 2], top_p=[0.9], min_p=[1e-3])):
        check_draw(dn, x, t, np.float32([0.61]), None, **kw)
    flat = np.round(x * 0.5)
    check_draw(dn, flat, t, np.float32([0.37]), None, top_k=[n // 3])
    check_draw(dn, flat, t, np.float32([0.73]), None, top_p=[0.55])
