"""Row operators on the device at the sizes where they change form, at the ends of the number range, and beyond
offsets of 32 bits."""
import ctypes as C
import struct

import numpy as np
import pytest

import row_reference as R
from darknet_amd import api
from row_reference import BF16, F16, F32, I8, Buffer
from test_gpu_row_operators import Norm, Q4, check_draw, logits_of

pytestmark = pytest.mark.gpu

# input type, weights' group, input_group
KINDS = [(F32, 128, 0), (F32, 32, 0), (BF16, 64, 0), (F16, 128, 0), (I8, 128, 128), (I8, 32, 32), (I8, 64, 0)]


@pytest.mark.parametrize("batch,k,n", [
    (5, 1000, 70), (20, 1000, 70), (5, 1000, 6200), (20, 1000, 6200),       # few outputs
    (16, 600, 44816), (5, 600, 49153), (32, 600, 22401), (32, 600, 49153),   # many: one and two tiles of rows
    (40, 600, 15001), (130, 600, 16401), (64, 600, 11201), (250, 600, 12293)])  # three and four
def test_q4_forms(dn, batch, k, n):
    for i in range(3):
        tx, group, xg = KINDS[(batch + n + 2 * i) % len(KINDS)]
        Q4(dn, batch + i, k, n, group).check(dn, n + i, batch, tx, F32, xg=xg, act=7)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("batch,k", [(1, 26000), (1, 28672), (1, 30000), (2, 14336), (3, 9500), (4, 7168), (4, 7169),
                                     (1, 35000), (1, 37000), (1, 70000), (1, 74000), (2, 36700), (4, 9000), (4, 18300), (4, 19000)])
def test_q4_long_rows(dn, kind, batch, k):
    tx, group, xg = kind
    Q4(dn, k + batch, k, 37, group).check(dn, k, batch, tx, F32, xg=xg)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("batch,k,n", [(5, 8064, 33), (5, 8065, 33), (16, 8192, 33), (17, 9001, 130), (33, 20787, 50), (5, 12545, 1700), (8, 16500, 2100)])
def test_q4_inputs_cut_over_workgroups(dn, kind, batch, k, n):
    tx, group, xg = kind
    Q4(dn, k + n, k, n, group).check(dn, k, batch, tx, BF16 if batch == 17 else F32, xg=xg, act=7)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("runs", [64, 128, 256, 512, 1024, 1536, 2048, 4096])
def test_norm_widths_where_the_form_changes(dn, t, runs):
    v = 4 if t == F32 else 8
    for n in (runs * v, runs * v + 1):
        Norm(n, 3, n, t, group=128).check(dn)
        Norm(n + 1, 2, n, t, add=False, group=0).check(dn)


def test_norm_rows_at_the_ends_of_the_range(dn):
    """Without eps the factor of a row leaves the range of 32 bits where the row is near its ends."""
    for size in (1e-42, 1e-39, 1e-36, 1e-30, 1e30, 3e37):
        c = Norm(7, 3, 333, F32, add=False, group=64)
        c.x *= np.float32(size)
        c.check(dn, eps=0)


@pytest.mark.parametrize("n", [1000, 8000, 20000])
def test_sample_many_tokens_kept(dn, n):
    """top-k that ends among tokens that weigh nothing, and distributions whose border shares its logits with many."""
    x, r = logits_of(n, 4, n, 6.)
    x[1, 3] += 60
    check_draw(dn, x, F32, r.random(4), 0.3 + r.random(4), top_k=np.full(4, n - n // 3))
    check_draw(dn, x, F32, r.random(4), np.full(4, 0.05), top_k=np.full(4, n // 2), top_p=np.full(4, 0.999))
    flat = (x * np.float32(0.01))
    check_draw(dn, flat, F32, r.random(4), top_p=np.full(4, 0.5), top_k=np.full(4, n - 7))
    check_draw(dn, flat, BF16, r.random(4), top_p=np.full(4, 0.9), min_p=np.full(4, 0.95))


@pytest.mark.parametrize("n", [6, 900, 30000])
def test_sample_logits_at_the_ends_of_the_range(dn, n):
    """Differences of two logits that leave 32 bits, under temperatures next to which they are small."""
    r = np.random.default_rng(n)
    x = (r.random((6, n)) * 3e38).astype(np.float32)
    x[:, ::2] *= -1
    x[:, 5] = -3e38
    t = np.float32([1e38, np.inf, 3e37, 1e36, 1.0, 2e38])
    u = np.linspace(0.02, 0.98, 6)
    check_draw(dn, x, F32, u, t)
    for k in (1, 2, n // 2, n - 1):
        check_draw(dn, x, F32, u, t, top_k=np.full(6, k))
        check_draw(dn, x, F32, u, t, top_k=np.full(6, k), top_p=np.full(6, 0.7), min_p=np.full(6, 0.01))
    check_draw(dn, x, F32, u, t, top_p=np.full(6, 0.9))


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("n", [300, 20000])
def test_norm_scales_that_are_not_finite(dn, t, n):
    """NaN and infinite scales: their outputs, and the 8-bit groups that hold them."""
    c = Norm(n, 2, n, t, group=128)
    c.g[5], c.g[200] = np.nan, np.inf
    s, o, q, scales = c.run(dn)
    with np.errstate(invalid="ignore"):
        _, y = R.rmsnorm(c.x, c.add, c.g, 1e-5, t)
        codes, want = R.q8(y, 128)
    assert np.array_equal(scales, want, equal_nan=True) and np.array_equal(q, codes)
    got = R.from_type(o, t)
    assert np.isnan(got[:, 5]).all() and np.isinf(got[:, 200]).all()
    rest = np.isfinite(y)
    assert (np.abs(got - y)[rest] <= (np.abs(y) * (R.HALF_STEP[t] + 4 * 2.0 ** -24) + R.HALF_TINY[t])[rest]).all()


@pytest.mark.parametrize("batch", [2, 20])
def test_q4_activations(dn, batch):
    """Every activation on what the product gives with none, by every way of storing: fp32 results differ from the
    formula's in 64 bits by the sum's own error (no slope here is above 1.8) and one rounding."""
    forms = {0: lambda v: 1 / (1 + np.exp(-v)), 1: lambda v: np.maximum(v, 0), 2: lambda v: np.where(v > 0, v, .01 * v), 3: lambda v: v,
             4: lambda v: np.maximum(v, 0) + .1 * v, 5: np.tanh, 7: lambda v: np.where(v > 0, v, .1 * v),
             8: lambda v: np.where(v >= 0, v, np.exp(np.minimum(v, 0)) - 1), 9: lambda v: 2 / (1 + np.exp(-v)) - 1, 11: lambda v: np.clip(v, -1, 1),
             13: lambda v: np.where(v >= 0, 1.0507 * v, 1.0507 * 1.6732 * (np.exp(np.minimum(v, 0)) - 1))}
    k = 256
    for n in (50, 24000):
        m = Q4(dn, n, k, n, 128)
        x = (np.random.default_rng(n).standard_normal((batch, k)) * 0.1).astype(np.float32)
        bx, out = Buffer(x), Buffer(shape=(batch, n), dtype=np.float32)
        ws = m.workspace(dn, F32, batch)
        v = x.astype(np.float64) @ m.w.T
        tol = R.q4_bound(x.astype(np.float64), m.w, 128, F32, v)
        for act, form in forms.items():
            assert m.call(dn, bx, F32, None, 0, None, out, F32, batch, act, ws) == 0
            dn.hip_synchronize()
            assert (np.abs(out.get() - form(v)) <= 1.8 * tol + 2.0 ** -23 * np.abs(form(v))).all(), act


def push(dn, ptr, a):
    dn.hip_push_array(ptr, np.ascontiguousarray(a, np.float32).ctypes.data_as(C.POINTER(C.c_float)), a.size)


def pull(dn, ptr, shape, dtype=np.float32):
    out = np.empty(shape, dtype)
    dn.hip_pull_array(ptr, out.ctypes.data_as(C.POINTER(C.c_float)), out.nbytes // 4)
    return out


def test_norm_beyond_32_bit_offsets(dn):
    rows, n = 70001, 16384
    x, q, qs = api.DeviceArray(n=rows * n), api.DeviceArray(n=rows * n // 4), api.DeviceArray(n=rows * (n // 128))
    dn.fill_gpu(rows * n, 2.0, x.ptr, 1)
    c = Norm(1, 1, n, F32, add=False, scales=False, group=128)
    last = (rows - 1) * n
    push(dn, x.ptr + last * 4, c.x)
    assert dn.forward_rmsnorm_gpu(x.ptr, None, None, None, x.ptr, q.ptr, qs.ptr, F32, rows, n, 128, 1e-5) == 0
    dn.hip_synchronize()
    _, y = R.rmsnorm(c.x, None, None, 1e-5, F32)
    codes, scales = R.q8(y, 128)
    assert (np.abs(pull(dn, x.ptr + last * 4, (1, n)) - y) <= 5 * 2.0 ** -24 * np.abs(y) + 2.0 ** -149).all()
    assert np.array_equal(pull(dn, q.ptr + last, (1, n), np.int8), codes)
    assert np.array_equal(pull(dn, qs.ptr + (rows - 1) * (n // 128) * 4, (1, n // 128)), scales)
    assert (np.abs(pull(dn, x.ptr + (last - n) * 4, (1, n)) - 1) <= 1e-5).all()


def test_q4_beyond_32_bit_offsets(dn):
    """Codes of whole numbers, scales of a half and inputs of small whole numbers: every sum is exact."""
    k, n = 16384, 600001
    codes, scales = api.DeviceArray(n=n * (k // 8)), api.DeviceArray(n=n * (k // 128))
    packed = api.DeviceArray(n=dn.q4_packed_bytes(k, n, 128) // 4)
    pattern = 0x3F9A2C71
    dn.fill_gpu(codes.n, struct.unpack("f", struct.pack("I", pattern))[0], codes.ptr, 1)
    dn.fill_gpu(scales.n, 0.5, scales.ptr, 1)
    marked = 0x12345678                                  # the last output's codes
    push(dn, codes.ptr + (n - 1) * (k // 2), np.full(k // 8, struct.unpack("f", struct.pack("I", marked))[0], np.float32))
    assert dn.q4_pack_codes_gpu(codes.ptr, scales.ptr, None, packed.ptr, k, n, 128) == 0
    w = [np.tile([((p >> 4 * i) & 15) - 8 for i in range(8)], k // 8) * 0.5 for p in (pattern, marked)]
    for batch in (1, 5):
        x = np.random.default_rng(batch).integers(-3, 4, (batch, k)).astype(np.float32)
        bx, out = Buffer(x), Buffer(shape=(batch, n), dtype=np.float32)
        size = dn.connected_q4_workspace_bytes(F32, batch, k, n, 128)
        ws = Buffer(shape=(size,), dtype=np.uint8, shift=16) if size else None
        assert dn.forward_connected_q4_gpu(bx.ptr, F32, None, 0, packed.ptr, None, out.ptr, F32, batch, k, n, 128, 3,
                                           ws.ptr if ws else None) == 0
        dn.hip_synchronize()
        got = out.get()
        assert (got[:, :-1] == (x @ w[0])[:, None]).all() and (got[:, -1] == x @ w[1]).all()


@pytest.mark.parametrize("n", [100, 20000])
def test_sample_beyond_32_bit_offsets(dn, n):
    rows, stride = 3, 1 << 30
    mem = api.DeviceArray(n=(rows - 1) * stride + n)
    x, r = logits_of(n, rows, n)
    for i in range(rows):
        push(dn, mem.ptr + i * stride * 4, x[i])
    u, k = r.random(rows).astype(np.float32), np.full(rows, 20, np.int32)
    bu, bk, tok = Buffer(u), Buffer(k), Buffer(shape=(rows,), dtype=np.int32)
    size = dn.sample_workspace_bytes(rows, n)
    ws = Buffer(shape=(size,), dtype=np.uint8, shift=16) if size else None
    assert dn.sample_rows_gpu(mem.ptr, F32, rows, n, stride, None, bk.ptr, None, None, bu.ptr, tok.ptr, None, ws.ptr if ws else None) == 0
    dn.hip_synchronize()
    got = tok.get()
    for i in range(rows):
        want, _, margin = R.sample(x[i], np.float32(1), 20, 1, 0, u[i])
        assert margin < 1e-9 or got[i] == want
