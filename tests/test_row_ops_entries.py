"""The C entries of the row operators refuse what their kernels do not take: an
error code before any launch (no GPU needed)."""

import pytest
import torch

from zookeeper_amd.ops import _native

BAD = 1  # hipErrorInvalidValue
P = 1 << 20  # stands for a device address; never read


@pytest.fixture
def lib():
    if not _native.available():
        pytest.skip(f"native library not built: {_native.load_error()}")
    return _native.lib()


def test_layer_norm_entries(lib):
    fwd = lib.zk_layer_norm_fwd

    def f(rows=2, cols=8, xs=8, dt=1):
        return fwd(P, P, P, P, None, None, rows, cols, xs, 1e-3, dt, 0)

    assert f(rows=0) == 0
    assert [f(rows=-1), f(cols=0), f(xs=-1), f(dt=3), f(dt=-1), f(rows=1 << 31)] == [BAD] * 6

    def b(rows=2, cols=8, xs=8, dys=8, dt=1, ws=P, n=1 << 20):
        return lib.zk_layer_norm_bwd(P, P, P, P, P, P, P, P, ws, n, rows, cols, xs, dys, dt, 0, 0)

    assert [b(rows=0), b(cols=0), b(xs=-1), b(dys=-1), b(dt=3), b(ws=None), b(n=16)] == [BAD] * 7
    assert lib.zk_layer_norm_bwd_ws_bytes(0, 8) == 0
    for rows in (1, 3, 100, 5000, 10 ** 6):
        for cols in (1, 33, 1000, 2048, 16384, 16385, 100000):
            n = lib.zk_layer_norm_bwd_ws_bytes(rows, cols)
            assert n % (8 * cols) == 0 and 0 < n <= 8 * cols * min(rows, 1024)


def test_token_logprobs_entries(lib):
    def f(rows=2, cols=8, xs=8, k=0, dt=1, ws=None, n=0, top=P):
        return lib.zk_token_logprobs_fwd(P, P, P, P, None, top, top, ws, n, rows, cols, xs, k,
                                         -100, dt, 0)

    assert f(rows=0) == 0
    assert [f(rows=-1), f(cols=0), f(xs=-1), f(k=-1), f(k=9), f(cols=100, k=65), f(dt=3),
            f(k=2, top=None), f(rows=1, cols=100000), f(rows=1, cols=100000, ws=P, n=64),
            f(cols=0x7FFF0000)] == [BAD] * 11

    def b(rows=2, cols=8, xs=8, dt=1):
        return lib.zk_token_logprobs_bwd(P, P, P, P, P, P, rows, cols, xs, -100, dt, 0)

    assert b(rows=0) == 0
    assert [b(rows=-1), b(cols=0), b(xs=-1), b(dt=3)] == [BAD] * 4
    assert lib.zk_token_logprobs_ws_bytes(5000, 100000, 5) == 0
    assert lib.zk_token_logprobs_ws_bytes(1, 2048, 5) == 0
    assert 0 < lib.zk_token_logprobs_ws_bytes(1, 100000, 64) <= 64 * (16 + 4 * 8 * 64)


def test_act8_entries(lib):
    for rows, cols, xs, dt in ((-1, 8, 8, 1), (2, 0, 8, 1), (2, 8, -1, 1), (2, 8, 8, 3)):
        assert lib.zk_pack8(P, P, P, rows, cols, xs, dt, 0) == BAD
        assert lib.zk_gelu8_fwd(P, P, P, P, rows, cols, xs, dt, 0) == BAD
        assert lib.zk_gelu8_bwd(P, P, P, P, rows, cols, xs, dt, 0) == BAD
    assert lib.zk_unpack8(P, P, P, 2, 0, 1, 0) == BAD
    assert lib.zk_pack8(P, P, P, 0, 8, 8, 1, 0) == 0

    def need(rows=128, outs=64, cols=64, dys=64, dt=1, variant=-1):
        return lib.zk_dense8_wgrad_ws_bytes(rows, outs, cols, dys, dt, 1, variant)

    assert need() > 0
    assert [need(rows=0), need(outs=0), need(cols=0), need(dys=-1), need(dys=1 << 24), need(dt=3),
            need(variant=2), need(rows=63, variant=1), need(cols=63, variant=1),
            need(rows=1 << 29), need(outs=1 << 24)] == [-1] * 11

    def w(ws=P, n=1 << 30, **kw):
        a = dict(rows=128, outs=64, cols=64, dys=64, dt=1, variant=-1)
        a.update(kw)
        return lib.zk_dense8_wgrad(P, P, P, P, P, ws, n, a["rows"], a["outs"], a["cols"],
                                   a["dys"], a["dt"], 0, a["variant"], 0)

    assert [w(ws=None), w(n=16), w(rows=0), w(dt=5), w(variant=3), w(ws=P + 4)] == [BAD] * 6


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from zookeeper_amd import ops

    x = torch.randn(3, 40, device="cuda")
    t = torch.zeros(3, dtype=torch.int64, device="cuda")
    for f in (ops.layer_norm, ops.gelu8, ops.pack8, lambda v: ops.token_logprobs(v, t),
              lambda v: ops.dense8(v, torch.ones(2, 40, device="cuda"))):
        for bad in (x.double(), x.to(torch.float8_e4m3fn), x.int()):
            with pytest.raises(ValueError):
                f(bad)
    with pytest.raises(ValueError, match="cpu"):
        ops.layer_norm(x, torch.ones(40))
    with pytest.raises(ValueError, match="cpu"):
        ops.token_logprobs(x, t.cpu())
    with pytest.raises(ValueError, match="cpu"):
        ops.dense8(x, torch.ones(2, 40))
    with pytest.raises(ValueError, match="cpu"):
        ops.dense8_grads(torch.ones(3, 2), ops.pack8(x))
    with pytest.raises(ValueError):
        ops.unpack8(ops.pack8(x), torch.float64)
    with pytest.raises(ValueError):
        ops.dense8_grads(torch.ones(3, 2, device="cuda", dtype=torch.float64), ops.pack8(x))
