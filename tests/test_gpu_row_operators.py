"""Row operators on the device against plain 64-bit forms: root-mean-square norm with residual and 8-bit output,
products with 4-bit weights, sampling - alone, one after the other, on streams and in captured graphs."""
import ctypes as C

import numpy as np
import pytest

import row_reference as R
from row_reference import BF16, F16, F32, I8, Buffer

pytestmark = pytest.mark.gpu
TYPES = [F32, F16, BF16]


# ---- norm ------------------------------------------------------------------------------------
class Norm:
    def __init__(self, seed, rows, n, t, add=True, scales=True, group=None, shift=0):
        r = np.random.default_rng(seed)
        self.rows, self.n, self.t, self.group = rows, n, t, group
        self.x = R.to_type(r.standard_normal((rows, n)) * 2, t)
        self.add = R.to_type(r.standard_normal((rows, n)) * 0.5, t) if add else None
        self.g = (1 + 0.2 * r.standard_normal(n)).astype(np.float32) if scales else None
        self.shift = shift

    def run(self, dn, eps=1e-5, output=True, keep_sum=True):
        size, sh = self.x.dtype.itemsize, self.shift
        put = lambda a, s=0: None if a is None else Buffer(a, shift=s)                # noqa: E731
        bx, ba, bg = put(self.x, sh * size), put(self.add, sh * size), put(self.g)
        new = lambda s=0: Buffer(shape=(self.rows, self.n), dtype=self.x.dtype, shift=s * size)  # noqa: E731
        bs = new(sh) if self.add is not None and keep_sum else None
        bo = new(sh) if output else None
        bq = bc = None
        if self.group is not None:
            groups = -(-self.n // (self.group or self.n))
            bq = Buffer(shape=(self.rows, self.n), dtype=np.int8, shift=sh)
            bc = Buffer(shape=(self.rows, groups), dtype=np.float32)
        p = lambda b: b.ptr if b else None                                            # noqa: E731
        assert dn.forward_rmsnorm_gpu(p(bx), p(ba), p(bg), p(bs), p(bo), p(bq), p(bc), self.t, self.rows, self.n,
                                      self.group or 0, eps) == 0
        dn.hip_synchronize()
        return [b.get() if b else None for b in (bs, bo, bq, bc)]

    def check(self, dn, eps=1e-5, **kw):
        s, o, q, c = self.run(dn, eps, **kw)
        want_s, y = R.rmsnorm(self.x, self.add, self.g, eps, self.t)
        if s is not None:
            assert np.array_equal(R.from_type(s, self.t), want_s)
        if o is not None:
            # r, and two products, are rounded to 32 bits, then the result to its type
            tol = np.abs(y) * (R.HALF_STEP[self.t] + 4 * 2.0 ** -24) + R.HALF_TINY[self.t]
            assert (np.abs(R.from_type(o, self.t) - y) <= tol).all()
        if q is not None:
            codes, scales = R.q8(y, self.group)
            assert np.array_equal(c, scales) and np.array_equal(q, codes)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 7), (1, 64), (5, 129), (2, 1000), (300, 128), (1, 4096), (2, 5003), (17, 8192), (3, 16384), (2, 20001), (1, 70000)])
def test_norm(dn, t, rows, n):
    Norm(rows + n, rows, n, t).check(dn)
    Norm(rows + n + 1, rows, n, t, add=False, scales=False).check(dn)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("group", [0, 32, 64, 128])
@pytest.mark.parametrize("rows,n", [(1, 1), (2, 31), (3, 130), (70, 256), (1, 4096), (4, 5003), (2, 12544), (2, 33000)])
def test_norm_q8(dn, t, group, rows, n):
    Norm(rows * 3 + n, rows, n, t, group=group).check(dn)
    Norm(rows * 3 + n + 1, rows, n, t, add=False, group=group).check(dn, output=False)
    Norm(rows * 3 + n + 2, rows, n, t, group=group).check(dn, output=False, keep_sum=False)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shift", [1, 2, 3])
def test_norm_at_any_element_boundary(dn, t, shift):
    Norm(shift, 3, 1024, t, group=64, shift=shift).check(dn)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n", [777, 4096, 40000])
@pytest.mark.parametrize("place", ["sum on input", "sum on add, output on input", "output on input", "output on add"])
def test_norm_in_place(dn, t, n, place):
    c = Norm(n, 4, n, t, group=128)
    want = c.run(dn, keep_sum="sum" in place)
    bx, ba, bg = Buffer(c.x), Buffer(c.add), Buffer(c.g)
    new = lambda d: Buffer(shape=(4, n), dtype=d)     # noqa: E731
    bs = {"sum on input": bx, "sum on add, output on input": ba}.get(place)
    bo = {"sum on input": None, "output on add": ba}.get(place, bx) or new(c.x.dtype)
    bq, bc = new(np.int8), Buffer(shape=want[3].shape, dtype=np.float32)
    assert dn.forward_rmsnorm_gpu(bx.ptr, ba.ptr, bg.ptr, bs.ptr if bs else None, bo.ptr, bq.ptr, bc.ptr, t, 4, n, 128, 1e-5) == 0
    dn.hip_synchronize()
    for got, w in zip((bs, bo, bq, bc), want):
        if got is not None:
            assert np.array_equal(got.get().view(np.uint8), w.view(np.uint8))


def test_norm_values_that_are_not_ordinary(dn):
    """Zeros, infinities, NaN, squares beyond 32 bits and below them: each row by itself."""
    n = 300
    c = Norm(5, 8, n, F32, add=False, scales=False, group=128)
    c.x[0] = 0
    c.x[1, 200] = np.inf
    c.x[2, 5] = np.nan
    c.x[3] *= 1e30
    c.x[4] *= 1e-30
    c.x[5, :] = 0
    c.x[5, 299] = -2.5
    _, o, q, scales = c.run(dn)
    _, y = R.rmsnorm(c.x, None, None, 1e-5, F32)
    codes, want = R.q8(y, 128)
    assert np.array_equal(np.isnan(o), np.isnan(y)) and np.array_equal(scales, want, equal_nan=True) and np.array_equal(q, codes)
    fine = ~np.isnan(y)
    assert (np.abs(o - y)[fine] <= 5 * 2.0 ** -24 * np.abs(y)[fine] + 2.0 ** -149).all()
    # the sum itself may leave the type
    c = Norm(6, 1, 64, F16)
    c.x[:], c.add[:] = 60000, 10000
    s = c.run(dn)[0]
    assert np.isinf(s).all()


def test_norm_more_rows_than_a_grid(dn):
    Norm(9, 70001, 3, BF16, group=0).check(dn)


# ---- 4-bit weights ---------------------------------------------------------------------------
class Q4:
    def __init__(self, dn, seed, k, n, group, zeros=True):
        self.k, self.n, self.group = k, n, group
        codes, scales, z = R.q4_codes(seed, n, k, group, zeros)
        self.w = R.q4_weights(codes, scales, z, group)
        self.packed = Buffer(shape=(dn.q4_packed_bytes(k, n, group),), dtype=np.uint8, shift=16)
        src = [Buffer(R.q4_bytes(codes)), Buffer(scales), Buffer(z) if zeros else None]
        assert dn.q4_pack_codes_gpu(src[0].ptr, src[1].ptr, src[2].ptr if zeros else None, self.packed.ptr, k, n, group) == 0
        dn.hip_synchronize()

    def call(self, dn, bx, tx, bxs, xg, bias, out, t_out, batch, act, ws):
        return dn.forward_connected_q4_gpu(bx.ptr, tx, bxs.ptr if bxs else None, xg, self.packed.ptr, bias.ptr if bias else None, out.ptr,
                                           t_out, batch, self.k, self.n, self.group, act, ws.ptr if ws else None)

    def workspace(self, dn, tx, batch):
        size = dn.connected_q4_workspace_bytes(tx, batch, self.k, self.n, self.group)
        return Buffer(shape=(size,), dtype=np.uint8, shift=16) if size else None

    def check(self, dn, seed, batch, tx, t_out, act=3, bias=True, xg=0, shift=0):
        r = np.random.default_rng(seed)
        x = r.standard_normal((batch, self.k)).astype(np.float32)
        x[:, r.random(self.k) < 0.01] *= 20
        xs = None
        if tx == I8:
            bits = r.integers(-128, 128, x.shape, dtype=np.int8)
            xs = (0.01 + 0.02 * r.random((batch, -(-self.k // xg) if xg else 1))).astype(np.float32)
            x = bits.astype(np.float64) * xs.astype(np.float64)[:, np.arange(self.k) // xg if xg else np.zeros(self.k, int)]
        else:
            bits = R.to_type(x, tx)
            x = R.from_type(bits, tx).astype(np.float64)
        b = r.standard_normal(self.n).astype(np.float32) if bias else None
        bx, bxs, bb = Buffer(bits, shift=shift * bits.itemsize), Buffer(xs) if tx == I8 else None, Buffer(b) if bias else None
        ws, out = self.workspace(dn, tx, batch), Buffer(shape=(batch, self.n), dtype=R.STORE[t_out], shift=shift * R.STORE[t_out]().itemsize)
        assert self.call(dn, bx, tx, bxs, xg, bb, out, t_out, batch, act, ws) == 0
        dn.hip_synchronize()
        got = R.from_type(out.get(), t_out).astype(np.float64)
        linear = R.q4_products(x, self.w, b, 3)
        y = R.ACTIVATE[act](linear)
        # no activation tested here is steeper than 1
        tol = R.q4_bound(x, self.w, self.group, t_out, linear, b)
        assert (np.abs(got - y) <= tol).all(), float((np.abs(got - y) / tol).max())
        if ws:
            ws.get()
        return out


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("k,n", [(1, 1), (31, 3), (128, 16), (129, 17), (257, 40), (1000, 33), (4096, 64), (5003, 130), (12544, 50)])
def test_q4_sizes(dn, group, k, n):
    m = Q4(dn, k + n, k, n, group)
    m.check(dn, 1, 1, F32, F32)
    m.check(dn, 2, 3, BF16, F16, act=7)
    m.check(dn, 3, 2, I8, F32, xg=group, bias=False)


@pytest.mark.parametrize("batch", [1, 2, 4, 5, 6, 8, 10, 11, 15, 16, 17, 21, 31, 32, 33, 48, 64, 65, 100, 130])
def test_q4_batches(dn, batch):
    m = Q4(dn, batch, 600, 75, 64)
    m.check(dn, batch, batch, F32, F32)
    m.check(dn, batch + 1, batch, I8, BF16, xg=64)
    m.check(dn, batch + 2, batch, F16, F16, bias=False)


@pytest.mark.parametrize("tx", [F32, F16, BF16, I8])
@pytest.mark.parametrize("t_out", TYPES)
def test_q4_types(dn, tx, t_out):
    for group, zeros in ((32, True), (64, False), (128, True)):
        m = Q4(dn, tx * 3 + t_out + group, 1111, 90, group, zeros)
        for batch, act in ((1, 1), (7, 0), (20, 7)):
            m.check(dn, batch, batch, tx, t_out, act=act)
            m.check(dn, batch, batch, tx, t_out, act=act, xg=group, shift=1)


def test_q4_a_large_layer(dn):
    """The sizes where every workgroup variant is in use, many row tiles among them."""
    for k, n, group in ((4096, 5000, 128), (2048, 40000, 32), (12544, 1715, 64)):
        m = Q4(dn, k + n, k, n, group)
        for batch, tx in ((1, F32), (4, BF16), (16, I8), (40, F32)):
            m.check(dn, batch, batch, tx, F32, xg=group if tx == I8 else 0)


def test_q4_values_that_are_not_ordinary(dn):
    k, n = 300, 40
    m = Q4(dn, 3, k, n, 64)
    x = np.random.default_rng(4).standard_normal((6, k)).astype(np.float32)
    x[0] = 0
    x[1, 7], x[2, 299] = np.inf, np.nan
    x[3] *= np.float32(1e34)
    x[4] *= np.float32(1e-34)
    x[5, :64], x[5, 64:] = x[5, :64] * np.float32(1e-42), 0
    for rows in (x, np.concatenate([x] * 5)):
        out, b = Buffer(shape=(len(rows), n), dtype=np.float32), np.full(n, 0.25, np.float32)
        assert m.call(dn, Buffer(rows), F32, None, 0, Buffer(b), out, F32, len(rows), 3, m.workspace(dn, F32, len(rows))) == 0
        dn.hip_synchronize()
        got = out.get()
        want = rows.astype(np.float64) @ m.w.T + 0.25
        for i in range(len(rows)):
            if i % 6 in (1, 2):
                assert np.isnan(got[i]).all()
            else:
                tol = R.q4_bound(rows[i:i + 1].astype(np.float64), m.w, 64, F32, want[i:i + 1], b)
                assert (np.abs(got[i] - want[i]) <= tol[0] + 2.0 ** -149).all(), i


def test_q4_nan_scales_of_8_bit_rows_reach_the_outputs(dn):
    """What the norm writes for a row that is not finite."""
    m = Q4(dn, 5, 256, 20, 128)
    bits, xs = np.ones((2, 256), np.int8), np.ones((2, 2), np.float32)
    bits[1, 128:], xs[1, 1] = 0, np.nan
    out = Buffer(shape=(2, 20), dtype=np.float32)
    assert m.call(dn, Buffer(bits), I8, Buffer(xs), 128, None, out, F32, 2, 3, m.workspace(dn, I8, 2)) == 0
    dn.hip_synchronize()
    got = out.get()
    assert np.isfinite(got[0]).all() and np.isnan(got[1]).all()


@pytest.mark.parametrize("k,n,group", [(1, 1, 32), (100, 20, 32), (300, 33, 64), (1000, 17, 128)])
def test_q4_pack_weights(dn, k, n, group):
    w = np.random.default_rng(k).standard_normal((n, k)).astype(np.float32)
    w[0, :min(k, group)] = 0                                     # a group of zeros
    if n > 1:
        w[1] = np.abs(w[1])                                      # groups on one side of zero
    packed, back = Buffer(shape=(dn.q4_packed_bytes(k, n, group),), dtype=np.uint8), Buffer(shape=(n, k), dtype=np.float32)
    assert dn.q4_pack_weights_gpu(Buffer(w).ptr, packed.ptr, k, n, group) == 0
    assert dn.q4_unpack_weights_gpu(packed.ptr, back.ptr, k, n, group) == 0
    dn.hip_synchronize()
    packed.get()
    got = back.get()
    for lo in range(0, k, group):
        part = w[:, lo:lo + group].astype(np.float64)
        step = (np.maximum(part.max(1), 0) - np.minimum(part.min(1), 0)) / 15
        # half a step from rounding, as much again where the rounded zero shifts the range's end
        assert (np.abs(got[:, lo:lo + group] - part) <= step[:, None] * (1 + 1e-6)).all()
        assert (np.abs(got[:, lo:lo + group] - part).mean(1) <= step * 0.5).all()
    assert (got[0, :min(k, group)] == 0).all()


def test_q4_unpack_gives_the_codes_back(dn):
    for k, n, group in ((77, 19, 32), (640, 16, 128)):
        codes, scales, zeros = R.q4_codes(k, n, k, group)
        m = Q4(dn, k, k, n, group)
        back = Buffer(shape=(n, k), dtype=np.float32)
        assert dn.q4_unpack_weights_gpu(m.packed.ptr, back.ptr, k, n, group) == 0
        dn.hip_synchronize()
        m.packed.get()
        assert np.array_equal(back.get(), (R.q4_weights(codes, scales, zeros, group)).astype(np.float32))


# ---- sampling --------------------------------------------------------------------------------
def draw(dn, logits, t, uniform, temperature=None, top_k=None, top_p=None, min_p=None, n=None, shift=0, probs=True):
    rows, stride = logits.shape
    n = stride if n is None else n
    put = lambda a, d: None if a is None else Buffer(np.asarray(a, d))            # noqa: E731
    bl = Buffer(R.to_type(logits, t), shift=shift * R.STORE[t]().itemsize)
    params = [put(temperature, np.float32), put(top_k, np.int32), put(top_p, np.float32), put(min_p, np.float32), put(uniform, np.float32)]
    tok, prob = Buffer(shape=(rows,), dtype=np.int32), Buffer(shape=(rows,), dtype=np.float32) if probs else None
    size = dn.sample_workspace_bytes(rows, n)
    ws = Buffer(shape=(size,), dtype=np.uint8, shift=16) if size else None
    assert dn.sample_rows_gpu(bl.ptr, t, rows, n, stride, *[p.ptr if p else None for p in params], tok.ptr, prob.ptr if probs else None,
                              ws.ptr if ws else None) == 0
    dn.hip_synchronize()
    if ws:
        ws.get()
    return tok.get(), prob.get() if probs else None


def check_draw(dn, logits, t, uniform, temperature=None, top_k=None, top_p=None, min_p=None, n=None, shift=0):
    tok, prob = draw(dn, logits, t, uniform, temperature, top_k, top_p, min_p, n, shift)
    held = R.from_type(R.to_type(logits, t), t)[:, :n]
    at = lambda a, r, d: d if a is None else np.asarray(a)[r]                     # noqa: E731
    for r in range(len(logits)):
        w_tok, w_prob, margin = R.sample(held[r], np.float32(at(temperature, r, 1.0)), at(top_k, r, 0), np.float32(at(top_p, r, 1.0)),
                                         np.float32(at(min_p, r, 0.0)), np.float32(uniform[r]))
        if margin < 1e-9:
            continue
        assert tok[r] == w_tok, (r, margin)
        # masses to 2^-38 of the largest, then one rounding
        assert abs(prob[r] - w_prob) <= 2.0 ** -24 * w_prob + 2.0 ** -37, r


def logits_of(seed, rows, n, spread=2.5):
    r = np.random.default_rng(seed)
    x = r.standard_normal((rows, n)).astype(np.float32) * np.float32(spread)
    for row in x:
        row[r.integers(0, n, min(n, 12))] += 6 * r.random(min(n, 12)).astype(np.float32)
    return x, r


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 2), (4, 63), (2, 1000), (5, 4097), (3, 8192), (2, 16385), (2, 50021), (1, 131072), (2, 262147)])
def test_sample_settings(dn, t, rows, n):
    x, r = logits_of(rows + n + t, rows, n)
    u, temp = r.random(rows), 0.4 + r.random(rows)
    check_draw(dn, x, t, u)
    check_draw(dn, x, t, u, temp, top_k=r.integers(1, 60, rows))
    check_draw(dn, x, t, u, temp, top_p=0.3 + 0.69 * r.random(rows))
    check_draw(dn, x, t, u, temp, min_p=0.01 + 0.2 * r.random(rows))
    check_draw(dn, x, t, u, temp, r.integers(1, 200, rows), 0.5 + 0.4 * r.random(rows), 0.02 * r.random(rows))
    check_draw(dn, x, t, u, 3 + temp, r.integers(max(1, n // 2), n + 5, rows), 0.99 + 0.009 * r.random(rows))
    check_draw(dn, x, t, u, np.zeros(rows))


def test_sample_a_batch_with_settings_of_its_own(dn):
    rows, n = 130, 5000
    x, r = logits_of(4, rows, n)
    x[r.random(x.shape) < 0.3] = -np.inf
    k, p, m = r.integers(-2, 80, rows), 0.2 + r.random(rows), r.random(rows) * 0.2 - 0.05
    check_draw(dn, x, F32, r.random(rows), r.random(rows) * 2 - 0.2, k, p, m)
    check_draw(dn, x, BF16, r.random(rows), r.random(rows) * 2 - 0.2, k, p, m, n=4321)      # part of each row
    check_draw(dn, x, F16, r.random(rows), None, k, p, m, shift=1)


@pytest.mark.parametrize("n", [5, 700, 20000, 140000])
def test_sample_ties_go_by_index(dn, n):
    """Every logit the same, two values only, and few values: borders run through equal tokens."""
    r = np.random.default_rng(n)
    u = r.random(8)
    for x in (np.zeros((8, n), np.float32), r.integers(0, 2, (8, n)).astype(np.float32), r.integers(-4, 5, (8, n)).astype(np.float32) / 2):
        check_draw(dn, x, F32, u)
        check_draw(dn, x, BF16, u, top_k=[1, 2, 3, n // 3 + 1, n - 1, n, n + 1, 0])
        check_draw(dn, x, F16, u, top_p=[.05, .1, .3, .5001, .7, .9, .99, .001])
        check_draw(dn, x, F32, u, None, [n // 2 + 1] * 8, [.05, .1, .3, .5001, .7, .9, .99, .001], [0.5] * 8)


@pytest.mark.parametrize("n", [37, 3000, 40000])
def test_sample_ends_and_odd_settings(dn, n):
    x, r = logits_of(n, 12, n)
    nan, inf = np.nan, np.inf
    u = np.array([0, 1, .5, -1, 2, nan, 0, 1, 0, 1, .3, .6])
    ok = dict(temperature=[1, 1, nan, 1, 1, 1, -1, inf, 1, 1, 1e-30, 1e30], top_k=[0, 0, 0, -5, 0, 0, 9, 0, 1, 3, 0, 0],
              top_p=[1, 1, .5, 1, 1, 1, .1, 1, 0, -1, nan, 2], min_p=[0.2, 0.2, 0, 0.2, 0.2, 0.2, 0, 0, 0, 0, nan, 7])
    tok, prob = draw(dn, x, F32, u, **ok)
    for i in range(12):
        l = x[i].astype(np.float64)
        kept = np.flatnonzero(np.exp(l - l.max()) >= np.float64(np.float32(0.2)))
        want = {0: kept[0], 1: kept[-1], 2: l.argmax(), 3: kept[0], 4: kept[-1], 5: kept[0], 6: l.argmax(), 7: n - 1, 8: l.argmax(),
                9: l.argmax(), 10: l.argmax(), 11: R.sample(x[i], 1e30, 0, 1, 1, np.float32(.6))[0]}[i]
        assert tok[i] == want, i
    assert prob[2] == prob[6] == prob[8] == prob[9] == prob[10] == 1


@pytest.mark.parametrize("n", [6, 900, 30000])
@pytest.mark.parametrize("t", TYPES)
def test_sample_rows_without_tokens_and_infinities(dn, n, t):
    x = np.full((7, n), -np.inf, np.float32)
    x[1] = np.nan
    x[2, 4] = -3
    x[3, [1, 3, 5]] = np.inf
    x[4, :], x[4, 2] = 1, np.nan
    x[5, 0], x[5, n - 1] = -1e38 if t != F16 else -6e4, -1e38 if t != F16 else -6e4
    x[6, [0, 5]] = np.inf
    x[6, 3] = np.nan
    u = np.array([.5, .5, .5, .5, .5, .75, .2])
    for kw in (dict(), dict(top_k=[3] * 7), dict(top_p=[.999] * 7), dict(top_k=[5] * 7, top_p=[.9999] * 7, min_p=[.1] * 7)):
        tok, prob = draw(dn, x, t, u, **kw)
        assert tok[[0, 1]].tolist() == [-1, -1] and prob[[0, 1]].tolist() == [0, 0]
        assert tok[2] == 4 and prob[2] == 1
        assert tok[3] == 3 and abs(prob[3] - 1 / 3) < 1e-7
        assert tok[5] == n - 1 and prob[5] == 0.5 and tok[6] == 0 and prob[6] == 0.5
        check_draw(dn, x[4:5], t, u[4:5], None, *[v and v[4:5] for v in (kw.get("top_k"), kw.get("top_p"), kw.get("min_p"))])


def test_sample_the_same_row_anywhere(dn):
    """A row gives its token at every place of a batch and in batches of every size."""
    x, r = logits_of(8, 1, 30011)
    want = draw(dn, x, F32, [.37], [.9], [50], [.95], [.01])
    for rows in (2, 9, 64, 300):
        tok, prob = draw(dn, np.repeat(x, rows, 0), F32, [.37] * rows, [.9] * rows, [50] * rows, [.95] * rows, [.01] * rows)
        assert (tok == want[0][0]).all() and (prob == want[1][0]).all()
    assert draw(dn, x, F32, [.37], [.9], [50], [.95], [.01], probs=False)[0][0] == want[0][0]


def test_sample_follows_its_distribution(dn):
    """Evenly spaced random numbers meet each token as often as its probability says, to within one."""
    x = np.log(np.float32([[1, 5, 0.5, 3, 7, 2, 0.25, 1.25]]))
    count = 4000
    tok, _ = draw(dn, np.repeat(x, count, 0), F32, (np.arange(count) + .5) / count)
    want = np.exp(x[0].astype(np.float64)) / 20 * count
    assert (np.abs(np.bincount(tok, minlength=8) - want) <= 1 + 1e-6).all()


# ---- together, on streams, in graphs -----------------------------------------------------------
class Step:
    """One step of a served model: norm with residual to 8 bits, 4-bit product, one token a row."""

    def __init__(self, dn, seed, rows, hidden, vocab, group=128):
        r = np.random.default_rng(seed)
        self.dn, self.rows, self.hidden, self.vocab, self.group = dn, rows, hidden, vocab, group
        self.m = Q4(dn, seed, hidden, vocab, group)
        groups = -(-hidden // group)
        self.x, self.h = (r.standard_normal((2, rows, hidden)) * 0.5).astype(np.float32)
        self.g = (1 + 0.1 * r.standard_normal(hidden)).astype(np.float32)
        self.u = r.random(rows).astype(np.float32)
        self.b = [Buffer(a) for a in (self.x, self.h, self.g, self.u, np.full(rows, 0.8, np.float32), np.full(rows, 40, np.int32))]
        self.sum, self.q = Buffer(shape=(rows, hidden), dtype=np.float32), Buffer(shape=(rows, hidden), dtype=np.int8)
        self.qs, self.logits = Buffer(shape=(rows, groups), dtype=np.float32), Buffer(shape=(rows, vocab), dtype=np.float32)
        self.tok, self.prob = Buffer(shape=(rows,), dtype=np.int32), Buffer(shape=(rows,), dtype=np.float32)
        self.ws1 = self.m.workspace(dn, I8, rows)
        size = dn.sample_workspace_bytes(rows, vocab)
        self.ws2 = Buffer(shape=(size,), dtype=np.uint8, shift=16) if size else None
        dn.hip_synchronize()

    def run(self):
        dn, b = self.dn, self.b
        assert dn.forward_rmsnorm_gpu(b[0].ptr, b[1].ptr, b[2].ptr, self.sum.ptr, None, self.q.ptr, self.qs.ptr, F32, self.rows,
                                      self.hidden, self.group, 1e-6) == 0
        assert self.m.call(dn, self.q, I8, self.qs, self.group, None, self.logits, F32, self.rows, 3, self.ws1) == 0
        assert dn.sample_rows_gpu(self.logits.ptr, F32, self.rows, self.vocab, self.vocab, b[4].ptr, b[5].ptr, None, None, b[3].ptr,
                                  self.tok.ptr, self.prob.ptr, self.ws2.ptr if self.ws2 else None) == 0

    def results(self):
        return [b.get() for b in (self.sum, self.q, self.qs, self.logits, self.tok, self.prob)]

    def check(self):
        s, q, qs, logits, tok, prob = self.results()
        want_s, y = R.rmsnorm(self.x, self.h, self.g, 1e-6, F32)
        codes, scales = R.q8(y, self.group)
        assert np.array_equal(s, want_s) and np.array_equal(q, codes) and np.array_equal(qs, scales)
        x = codes.astype(np.float64) * scales.astype(np.float64)[:, np.arange(self.hidden) // self.group]
        want = R.q4_products(x, self.m.w, None, 3)
        assert (np.abs(logits - want) <= R.q4_bound(x, self.m.w, self.group, F32, want)).all()
        for i in range(self.rows):
            w_tok, w_prob, margin = R.sample(logits[i], np.float32(.8), 40, 1, 0, self.u[i])
            assert margin < 1e-9 or (tok[i] == w_tok and abs(prob[i] - w_prob) <= 2.0 ** -24 * w_prob + 2.0 ** -37)


@pytest.mark.parametrize("rows,hidden,vocab,group", [(1, 1024, 1000, 128), (3, 777, 5003, 32), (20, 2048, 33000, 64)])
def test_a_served_step(dn, rows, hidden, vocab, group):
    s = Step(dn, rows, rows, hidden, vocab, group)
    s.run()
    dn.hip_synchronize()
    s.check()


class Hip:
    def __init__(self):
        self.lib = C.CDLL("libamdhip64.so")

    def __getattr__(self, name):
        fn = getattr(self.lib, name)

        def call(*a):
            status = fn(*a)
            assert status == 0, (name, status)
        return call

    def stream(self):
        s = C.c_void_p()
        self.hipStreamCreateWithFlags(C.byref(s), C.c_uint(1))   # does not wait for the null stream
        return s


def test_two_streams_at_once(dn):
    """Two steps in flight on streams of their own; each gives what it gives alone."""
    hip = Hip()
    steps = [Step(dn, 31, 4, 1024, 33000), Step(dn, 32, 2, 2000, 20011)]
    streams = [hip.stream(), hip.stream()]
    try:
        for _ in range(3):
            for s, st in zip(steps, streams):
                dn.hip_set_stream(st)
                s.run()
        for st in streams:
            hip.hipStreamSynchronize(st)
    finally:
        dn.hip_set_stream(None)
    for s in steps:
        s.check()
    for st in streams:
        hip.hipStreamDestroy(st)


def test_captured_and_replayed(dn):
    """Two steps captured into two graphs, replayed in turn with new inputs and eager work in between: every replay
    gives what the eager calls give."""
    hip = Hip()
    steps = [Step(dn, 41, 2, 1024, 33000), Step(dn, 42, 5, 640, 3001, 32)]
    st = hip.stream()
    execs = []
    try:
        dn.hip_set_stream(st)
        for s in steps:
            graph, ex = C.c_void_p(), C.c_void_p()
            hip.hipStreamBeginCapture(st, C.c_int(2))   # relaxed
            s.run()
            hip.hipStreamEndCapture(st, C.byref(graph))
            hip.hipGraphInstantiate(C.byref(ex), graph, None, None, C.c_size_t(0))
            execs.append((graph, ex))
        for turn in range(3):
            for s, (_, ex) in zip(steps, execs):
                s.u[:] = np.random.default_rng(turn).random(s.rows)
                dn.hip_push_array(s.b[3].ptr, s.u.ctypes.data_as(C.POINTER(C.c_float)), s.rows)
                hip.hipGraphLaunch(ex, st)
                hip.hipStreamSynchronize(st)
                s.check()
                replayed = s.results()
                s.run()
                hip.hipStreamSynchronize(st)
                assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(replayed, s.results()))
    finally:
        dn.hip_set_stream(None)
    for graph, ex in execs:
        hip.hipGraphExecDestroy(ex)
        hip.hipGraphDestroy(graph)
    hip.hipStreamDestroy(st)
