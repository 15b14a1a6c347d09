"""Row operators without a GPU: what they refuse (before anything touches a device), the sizes they ask for, and
the plain forms that their GPU tests compare with."""
import numpy as np
import pytest

from darknet_amd import lib

import row_reference as R

P = 1 << 20     # an address that nothing reads: every call here is refused first


@pytest.fixture(scope="module")
def L():
    return lib.load()


def norm(L, **kw):
    a = dict(input=P, add=P, scales=P, sum=P, output=2 * P, q=None, qs=None, type=R.F32, rows=2, n=8, group=0, eps=1e-5)
    a.update(kw)
    return L.forward_rmsnorm_gpu(*a.values())


@pytest.mark.parametrize("change,word", [
    (dict(type=R.I8), "type"), (dict(type=9), "type"), (dict(rows=-1), "geometry"), (dict(n=0), "geometry"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(input=None), "input"),
    (dict(output=None), "neither"), (dict(q=P), "together"), (dict(qs=P), "together"), (dict(group=48), "q8_group"),
    (dict(add=None), "needs add"), (dict(sum=2 * P), "two buffers"), (dict(input=P + 2), "aligned"),
    (dict(type=R.BF16, output=P + 1), "aligned"), (dict(q=P, qs=P + 2), "aligned"), (dict(scales=P + 1), "aligned")])
def test_norm_refuses(L, capfd, change, word):
    assert norm(L, **change) == -1
    err = capfd.readouterr().err
    assert "forward_rmsnorm_gpu" in err and word in err


def q4(L, **kw):
    a = dict(x=P, tx=R.F32, xs=None, xg=0, packed=P, bias=None, y=P, ty=R.F32, batch=1, k=64, n=16, group=32, act=3, ws=P)
    a.update(kw)
    return L.forward_connected_q4_gpu(*a.values())


@pytest.mark.parametrize("change,word", [
    (dict(tx=4), "input type"), (dict(tx=-1), "input type"), (dict(ty=R.I8), "output type"), (dict(batch=-1), "geometry"), (dict(k=0), "geometry"),
    (dict(n=0), "geometry"), (dict(group=16), "group"), (dict(act=14), "activation"), (dict(act=-1), "activation"),
    (dict(x=None), "missing"), (dict(packed=None), "missing"), (dict(y=None), "missing"), (dict(tx=R.I8), "scales"),
    (dict(tx=R.I8, xs=P, xg=64), "input_group"), (dict(packed=P + 8), "aligned"), (dict(y=P + 2), "aligned"),
    (dict(x=P + 1, tx=R.F16), "aligned"), (dict(bias=P + 1), "aligned")])
def test_q4_refuses(L, capfd, change, word):
    assert q4(L, **change) == -1
    err = capfd.readouterr().err
    assert "forward_connected_q4_gpu" in err and word in err


def test_q4_packing_refuses(L, capfd):
    for call in (lambda **k: L.q4_pack_codes_gpu(k.get("src", P), P, P, k.get("to", P), k.get("k", 8), 8, k.get("g", 32)),
                 lambda **k: L.q4_pack_weights_gpu(k.get("src", P), k.get("to", P), k.get("k", 8), 8, k.get("g", 32)),
                 lambda **k: L.q4_unpack_weights_gpu(k.get("to", P), k.get("src", P), k.get("k", 8), 8, k.get("g", 32))):
        for bad, word in ((dict(src=None), "missing"), (dict(to=None), "missing"), (dict(to=P + 4), "aligned"),
                          (dict(k=0), "geometry"), (dict(g=100), "group")):
            assert call(**bad) == -1
            assert word in capfd.readouterr().err
    assert L.q4_packed_bytes(0, 4, 32) == L.q4_packed_bytes(4, 0, 32) == L.q4_packed_bytes(4, 4, 48) == 0


def test_q4_packed_bytes(L):
    # tiles of 16 outputs x 128 inputs at half a byte, and 5 bytes for each group of each output
    assert L.q4_packed_bytes(128, 16, 128) == 1024 + 16 * 5
    assert L.q4_packed_bytes(129, 17, 32) == 4 * 1024 + 2 * 8 * 16 * 5
    assert L.q4_packed_bytes(1 << 17, 1 << 17, 128) == (1 << 33) + (1 << 27) * 5     # beyond 32 bits


def sample(L, **kw):
    a = dict(x=P, t=R.F32, rows=1, n=8, stride=8, temp=P, k=P, p=P, m=P, u=P, tok=P, prob=P, ws=P)
    a.update(kw)
    return L.sample_rows_gpu(*a.values())


@pytest.mark.parametrize("change,word", [
    (dict(t=R.I8), "type"), (dict(rows=-1), "geometry"), (dict(n=0), "geometry"), (dict(n=(1 << 24) + 1, stride=1 << 25), "geometry"),
    (dict(stride=7), "stride"), (dict(x=None), "missing"), (dict(u=None), "missing"), (dict(tok=None), "missing"),
    (dict(x=P + 2), "aligned"), (dict(tok=P + 1), "aligned"), (dict(k=P + 2), "aligned"), (dict(prob=P + 2), "aligned")])
def test_sample_refuses(L, capfd, change, word):
    assert sample(L, **change) == -1
    err = capfd.readouterr().err
    assert "sample_rows_gpu" in err and word in err


def test_no_rows_is_no_work(L):
    assert norm(L, rows=0) == 0 and q4(L, batch=0) == 0 and sample(L, rows=0) == 0


def test_plain_forms():
    """The plain forms on cases worked by hand."""
    s, y = R.rmsnorm(np.float32([[3, 4]]), np.float32([[0, 0]]), np.float32([1, 2]), 0.0, R.F32)
    assert np.allclose(y, np.float64([[3, 8]]) / np.sqrt(12.5), rtol=1e-15)
    codes, scales = R.q8(np.float64([[127.0, -63.5, 0.4, 0.0]]), 0)
    assert codes.tolist() == [[127, -64, 0, 0]] and scales.tolist() == [[1.0]]
    assert R.from_type(R.to_type(np.float32([1.00390625, 1.01171875]), R.BF16), R.BF16).tolist() == [1.0, 1.015625]
    w = R.q4_weights(np.uint8([[0, 15, 8]]), np.float32([[0.5]]), np.uint8([[3]]), 32)
    assert w.tolist() == [[-1.5, 6.0, 2.5]]
    assert R.q4_bytes(np.uint8([[1, 2, 3]])).tolist() == [[0x21, 0xF3]]
    l = np.log(np.float64([1, 4, 2, 4, np.nan, 0]), where=[1, 1, 1, 1, 0, 0], out=np.full(6, -np.inf)).astype(np.float32)
    l[4] = np.nan
    assert R.sample(l, 1, 0, 1, 0, 0.5)[0] == 2                  # masses 1 4 2 4: half of 11 lies in the third
    assert R.sample(l, 1, 2, 1, 0, 0.6)[0] == 3                  # the two fours
    assert R.sample(l, 1, 0, 0.3, 0, 1.0)[0] == 1                # one four alone is 4/11
    assert R.sample(l, 1, 0, 1, 0.4, 1.0)[0] == 3 and R.sample(l, 0, 0, 1, 0, 0.9)[:2] == (1, 1.0)
    assert R.sample(np.float32([np.nan, -np.inf]), 1, 0, 1, 0, .5)[:2] == (-1, 0.0)


def test_no_rows_need_no_buffers(L):
    assert norm(L, rows=0, input=None, add=None, scales=None, sum=None, output=None) == 0
    assert q4(L, batch=0, x=None, packed=None, y=None, ws=None) == 0
    assert sample(L, rows=0, x=None, u=None, tok=None, ws=None) == 0


def test_sizes_whose_indexes_leave_an_int_are_refused(L, capfd):
    big = 0x7FFFFFFF
    assert norm(L, n=big) == q4(L, k=big) == q4(L, n=big) == q4(L, batch=big, k=64, n=16) == -1
    assert "geometry" in capfd.readouterr().err
    assert L.q4_packed_bytes(big, 16, 32) == L.q4_packed_bytes(16, big, 32) == 0


@pytest.mark.parametrize("batch,k,n", [(5, 64, 16), (64, 64, 16), (1, 40000, 16), (16, 128, 45000)])
def test_q4_workspace(L, capfd, batch, k, n):
    """Asked for and missing, or not aligned."""
    assert L.connected_q4_workspace_bytes(R.F32, batch, k, n, 32) > 0
    assert q4(L, batch=batch, k=k, n=n, ws=None) == -1 and "workspace is missing" in capfd.readouterr().err
    assert q4(L, batch=batch, k=k, n=n, ws=P + 8) == -1 and "workspace" in capfd.readouterr().err


def test_q4_workspace_not_needed(L):
    assert L.connected_q4_workspace_bytes(R.F32, 1, 4096, 4096, 128) == 0
    assert L.connected_q4_workspace_bytes(R.F32, 0, 4096, 4096, 128) == L.connected_q4_workspace_bytes(R.F32, 8, 4096, 4096, 5) == 0


def test_sample_workspace(L, capfd):
    assert L.sample_workspace_bytes(4, 8192) == 0 and L.sample_workspace_bytes(4, 8193) > 0
    assert L.sample_workspace_bytes(0, 9000) == L.sample_workspace_bytes(1, (1 << 24) + 1) == 0
    assert L.sample_workspace_bytes(100000, 1 << 17) > 1 << 32     # sizes are not cut to 32 bits
    assert sample(L, n=9000, stride=9000, ws=None) == -1 and "workspace is missing" in capfd.readouterr().err
    assert sample(L, n=9000, stride=9000, ws=P + 8) == -1 and "workspace" in capfd.readouterr().err
