"""Calls of the row operators that their documentation allows and other tests leave out: the least and the most rows and
columns, few rows that are not ordinary, a workspace in use again, some activations, more rows than a grid has."""
import ctypes as C

import numpy as np
import pytest

import row_reference as R
from darknet_amd import api
from row_reference import BF16, F16, F32, Buffer
from test_gpu_row_operators import Hip, Step
from test_gpu_row_operators_range import Weights

pytestmark = pytest.mark.gpu


def ordinary_rows(seed, batch, k, t):
    """(bits, values in 64 bits) of ordinary rows of a type; 8 bits come with a scale for each row."""
    r = np.random.default_rng(seed)
    if t == R.I8:
        bits = r.integers(-128, 128, (batch, k), dtype=np.int8)
        xs = ((0.5 + r.random((batch, 1))) * 0.02 * r.choice([-1, 1], (batch, 1))).astype(np.float32)
        return bits, xs, bits * xs.astype(np.float64)
    bits = R.to_type(r.standard_normal((batch, k)).astype(np.float32), t)
    return bits, None, R.from_type(bits, t).astype(np.float64)


def close(x, w, group, t, t_out, y):
    """How far an output y may be off: fp32 input is held to 2^-23 of each value; a group's sum takes a rounding for each
    of its eight matrix instructions and eight within one, and each group, the row's factor, bias and type one more."""
    size = np.abs(x) @ np.abs(w).T
    held = 2.0 ** -23 if t == F32 else 0
    return size * (held + (64 + -(-x.shape[1] // group) + 8) * 2.0 ** -24) + R.HALF_STEP[t_out] * np.abs(y) * 1.01 + R.HALF_TINY[t_out]


@pytest.mark.parametrize("t", [F32, BF16, F16, R.I8])
@pytest.mark.parametrize("batch,k,n", [(1, 7, 1), (2, 8, 3), (4, 9, 17), (5, 1, 1), (6, 3, 20), (17, 7, 40), (40, 8, 5), (64, 9, 11300), (5, 5, 49153), (33, 129, 1), (1500, 64, 33), (4099, 40, 700)])
@pytest.mark.parametrize("t_out", [F32, F16])
def test_q4_least_and_most_rows_and_columns(dn, batch, k, n, t, t_out):
    """Rows shorter than an access, single outputs, thousands of rows; 8-bit rows with scales of either sign."""
    group = 32
    codes, scales, zeros = R.q4_codes(k + n, n, k, group)
    bits, xs, x = ordinary_rows(batch, batch, k, t)
    m = Weights(dn, codes, scales, zeros, group)
    got, y = m.product(dn, bits, t, xs, 0, t_out), x @ m.w.T
    assert (np.abs(got - y) <= close(x, m.w, group, t, t_out, y)).all()


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("batch", [1, 2, 3, 4])
def test_q4_few_rows_that_are_not_ordinary(dn, batch, t):
    """Rows of zeros, with an infinity, with NaN, of very large, very small and subnormal values, by themselves and together."""
    k, n, group = 300, 40, 64
    codes, scales, zeros = R.q4_codes(batch, n, k, group)
    m = Weights(dn, codes, scales, zeros, group)
    base = np.random.default_rng(4).standard_normal((7, k)).astype(np.float32)
    base[0] = 0
    base[1, 7], base[2, 299] = np.inf, np.nan
    base[3] *= np.float32(1e34 if t != F16 else 1e4)
    base[4] *= np.float32(1e-34 if t != F16 else 1e-5)
    base[5] *= np.float32(1e-41 if t != F16 else 1e-6)
    for first in range(7):
        rows = base[(first + np.arange(batch)) % 7]
        bits = R.to_type(rows, t)
        x = R.from_type(bits, t).astype(np.float64)
        got = m.product(dn, bits, t)
        for i in range(batch):
            if not np.isfinite(x[i]).all():
                assert np.isnan(got[i]).all()
                continue
            y = x[i:i + 1] @ m.w.T
            assert (np.abs(got[i] - y) <= close(x[i:i + 1], m.w, group, t, F32, y) + (k // group + 8) * 2.0 ** -149).all(), (first, i)


@pytest.mark.parametrize("batch,k,n", [(5, 700, 90), (5, 8200, 60), (20, 300, 20000)])
def test_q4_a_workspace_in_use_again(dn, batch, k, n):
    """What a call with an outlier in each row leaves in the workspace does not touch the next call, nor the other way round;
    every call of a kind gives the same bits."""
    group = 64
    codes, scales, zeros = R.q4_codes(k, n, k, group)
    m = Weights(dn, codes, scales, zeros, group)
    r = np.random.default_rng(k)
    plain = r.standard_normal((batch, k)).astype(np.float32)
    far = plain.copy()
    far[np.arange(batch), r.integers(0, k, batch)] = 1e12
    size = dn.connected_q4_workspace_bytes(F32, batch, k, n, group)
    ws, first = Buffer(shape=(size,), dtype=np.uint8, shift=16), {}
    for _ in range(3):
        for name, rows in (("plain", plain), ("far", far)):
            out = Buffer(shape=(batch, n), dtype=np.float32)
            assert dn.forward_connected_q4_gpu(Buffer(rows).ptr, F32, None, 0, m.packed.ptr, None, out.ptr, F32, batch, k, n, group, 3, ws.ptr) == 0
            dn.hip_synchronize()
            got = out.get()
            x = rows.astype(np.float64)
            y = x @ m.w.T
            assert (np.abs(got - y) <= close(x, m.w, group, F32, F32, y)).all()
            assert np.array_equal(first.setdefault(name, got), got)


@pytest.mark.parametrize("batch,n", [(2, 50), (20, 50), (20, 24000)])
def test_q4_the_other_activations(dn, batch, n):
    """plse, stair and lhtan on what the product gives with none (the same call but for the activation)."""
    k, group = 256, 128
    codes, scales, zeros = R.q4_codes(n, n, k, group)
    m = Weights(dn, codes, scales * 4, zeros, group)
    bits, _, _ = ordinary_rows(n, batch, k, F32)
    v = m.product(dn, bits, F32)
    floor = np.floor(v)
    forms = {6: np.where(v < -4, .01 * (v + 4), np.where(v > 4, .01 * (v - 4) + 1, .125 * v + .5)),
             10: np.where(floor % 2 == 0, np.floor(v / 2), (v - floor) + np.floor(v / 2)),
             12: np.where(v < 0, .001 * v, np.where(v > 1, .001 * (v - 1) + 1, v))}
    for act, want in forms.items():
        got = m.product(dn, bits, F32, act=act)
        # from the same fp32 sum: the steps' differences and the result are rounded to 32 bits
        assert (np.abs(got - want) <= 2.0 ** -23 * np.maximum(np.abs(want), 1)).all(), act


def test_products_with_workspaces_on_two_streams(dn):
    """Steps of five rows and more, whose products have workspaces, in flight on two streams; each gives what it gives alone."""
    hip = Hip()
    steps = [Step(dn, 51, 6, 9000, 1000), Step(dn, 52, 40, 1024, 9001)]
    assert all(s.ws1 for s in steps)
    streams = [hip.stream(), hip.stream()]
    try:
        for _ in range(4):
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


@pytest.mark.parametrize("n", [9, 8200])
def test_sample_more_rows_than_a_grid(dn, n):
    """Logits that are all the same: the token is the place of the random number, in each of 70000 rows."""
    rows = 70000
    logits = api.DeviceArray(n=rows * n // 2)                # zeros, as bf16
    u = ((np.random.default_rng(n).integers(0, n, rows) + 0.5) / n).astype(np.float32)
    bu, tok, prob = Buffer(u), Buffer(shape=(rows,), dtype=np.int32), Buffer(shape=(rows,), dtype=np.float32)
    size = dn.sample_workspace_bytes(rows, n)
    ws = api.DeviceArray(n=size // 4 + 4) if size else None
    assert dn.sample_rows_gpu(logits.ptr, BF16, rows, n, n, None, None, None, None, bu.ptr, tok.ptr, prob.ptr, ws.ptr if ws else None) == 0
    dn.hip_synchronize()
    assert np.array_equal(tok.get(), np.floor(u.astype(np.float64) * n).astype(np.int32))
    assert (np.abs(prob.get() - 1 / n) <= 2.0 ** -24 / n).all()


@pytest.mark.parametrize("batch,k,n", [(3, 2000, 300), (6, 700, 90), (5, 8200, 60), (20, 300, 20000)])
def test_q4_captured_rows_that_change_their_kind(dn, batch, k, n):
    """A captured product replayed with ordinary rows, rows with outliers and rows of all sizes in turn, eager work between:
    every replay gives the bits that the eager call gives, and they are right."""
    group = 128
    codes, scales, zeros = R.q4_codes(n, n, k, group)
    m = Weights(dn, codes, scales, zeros, group)
    r = np.random.default_rng(n)
    kinds = [r.standard_normal((batch, k)).astype(np.float32) for _ in range(3)]
    kinds[1][np.arange(batch), r.integers(0, k, batch)] = 1e15
    kinds[2] *= (2.0 ** r.uniform(-90, 60, (batch, k))).astype(np.float32)
    size = dn.connected_q4_workspace_bytes(F32, batch, k, n, group)
    ws = Buffer(shape=(size,), dtype=np.uint8, shift=16) if size else None
    x, out = Buffer(kinds[0]), Buffer(shape=(batch, n), dtype=np.float32)
    call = lambda: dn.forward_connected_q4_gpu(x.ptr, F32, None, 0, m.packed.ptr, None, out.ptr, F32, batch, k, n, group, 3,  # noqa: E731
                                               ws.ptr if ws else None)
    hip = Hip()
    st, graph, ex = hip.stream(), C.c_void_p(), C.c_void_p()
    try:
        dn.hip_set_stream(st)
        hip.hipStreamBeginCapture(st, C.c_int(2))   # relaxed
        assert call() == 0
        hip.hipStreamEndCapture(st, C.byref(graph))
        hip.hipGraphInstantiate(C.byref(ex), graph, None, None, C.c_size_t(0))
        for rows in (kinds[i] for i in (1, 0, 2, 0, 1, 2)):
            dn.hip_push_array(x.ptr, rows.ctypes.data_as(C.POINTER(C.c_float)), rows.size)
            hip.hipGraphLaunch(ex, st)
            hip.hipStreamSynchronize(st)
            replayed = out.get()
            v = rows.astype(np.float64)
            y = v @ m.w.T
            assert (np.abs(replayed - y) <= close(v, m.w, group, F32, F32, y)).all()
            assert call() == 0
            hip.hipStreamSynchronize(st)
            assert np.array_equal(out.get(), replayed)
    finally:
        dn.hip_set_stream(None)
    hip.hipGraphExecDestroy(ex)
    hip.hipGraphDestroy(graph)
    hip.hipStreamDestroy(st)
