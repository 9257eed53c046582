"""8-bit kept activations against their definitions in 64 bits.

The form itself is exact arithmetic (powers of two, one rounding to a whole
number), so packed and unpacked values are compared bit for bit.  Tolerances of
the rest, with ``u = 2^-24`` and half a unit of the output type added:

* Phi: the fitted tail is right to 1e-7 of itself, its eight Horner steps, the
  reciprocal and the products round ~30 times, and the exponent's rounding moves
  it by ``x^2 u`` of itself; ``1 - tail`` rounds once more.
* matrix products: every product is exact, a sum of M of them in any order is off
  by at most ``M`` roundings of its absolute sum (2^-23 each, should the matrix
  unit truncate)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from zookeeper_amd import ops

    assert ops.available(), ops.load_error()


def _held(x):
    """What the 8-bit form of x stands for, fp64, from its definition."""
    n = x.shape[-1]
    v = torch.nn.functional.pad(x.double(), (0, -n % 32)).unflatten(-1, (-1, 32))
    top = v.abs().amax(-1)
    fine = torch.isfinite(top)
    t = torch.where(fine, top, torch.ones_like(top))
    e = torch.where(t > 0, torch.frexp(t).exponent.double() - 1, torch.full_like(t, -120.0))
    e = e.clamp(-120, 127)
    e = e + ((torch.round(t * torch.exp2(6 - e)) >= 128) & (e < 127)).double()
    step = torch.exp2(e - 6).unsqueeze(-1)
    k = torch.round(v / step).clamp(-127, 127) * step
    return k.masked_fill(~fine.unsqueeze(-1), float("nan")).flatten(-2)[..., :n]


def _half(dt):
    return torch.finfo(dt).eps / 2


def _tiny(dt):
    return torch.finfo(dt).tiny * torch.finfo(dt).eps / 2 + 2.0 ** -126


SHAPES = [(1, 1), (1, 32), (3, 31), (2, 33), (7, 64), (5, 8), (33, 100), (1, 4097), (64, 1000),
          (257, 96), (2047, 1111), (4, 3, 40), (1000, 2), (2, 70001)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_pack_and_unpack(shape, dt):
    from zookeeper_amd.ops import pack8, unpack8

    torch.manual_seed(sum(shape))
    scale = torch.exp2(torch.randint(-20, 8, shape, device="cuda").float())
    x = (torch.randn(shape, device="cuda") * scale).to(dt)
    kept = pack8(x)
    held = _held(x)
    assert kept.shape == x.shape and kept.dtype == dt
    assert torch.equal(unpack8(kept, torch.float32).double(), held)
    assert torch.equal(unpack8(kept, torch.bfloat16).double(), held)  # exact in bf16
    assert torch.equal(unpack8(kept), held.to(torch.float32).to(dt))
    n = shape[-1]
    top = torch.nn.functional.pad(x.double(), (0, -n % 32)).unflatten(-1, (-1, 32)).abs().amax(-1)
    err = (held - x.double()).abs()
    # half a step: 2^(E - 7) <= 2^-7 top as top >= 2^E; where the step was doubled, top
    # rounds to 128 steps, so top >= 127.5 * 2^(E - 6) and half of 2^(E - 5) is top / 127.5
    assert (err <= top.repeat_interleave(32, -1)[..., :n] / 127.5).all()
    # the host's form is the same bytes
    host = pack8(x.cpu())
    assert torch.equal(host.codes, kept.codes.cpu()) and torch.equal(host.scales,
                                                                     kept.scales.cpu())


def test_pack_borders():
    from zookeeper_amd.ops import pack8, unpack8

    big = torch.finfo(torch.float32).max
    rows = [[0.0] * 32, [-0.0] * 32, [1.0] + [0.0] * 31, [127.0, 63.5, 0.5, 1.5, 2.5],
            [127.4999, 1.0], [127.5, 1.0], [1.9921875, -1.9921875], [1.9999999],
            [big, -big, 1.0], [big * 2.0 ** -1], [1e-40, -1e-45], [2.0 ** -126, 2.0 ** -127],
            [2.0 ** -120, 2.0 ** -126], [3.0] * 32]
    x = torch.zeros(len(rows), 32, device="cuda")
    for i, r in enumerate(rows):
        x[i, :len(r)] = torch.tensor(r)
    held = unpack8(pack8(x))
    assert torch.equal(held.double(), _held(x))
    assert torch.isfinite(held).all()
    host = pack8(x.cpu())
    assert torch.equal(host.codes, pack8(x).codes.cpu())
    assert torch.equal(host.scales, pack8(x).scales.cpu())


def test_nan_and_infinity_take_their_block_only():
    from zookeeper_amd.ops import pack8, unpack8

    for dt in DTYPES:
        x = torch.randn(3, 100, device="cuda").to(dt)
        x[0, 40], x[1, 99], x[2, 0] = float("nan"), float("inf"), float("-inf")
        h = unpack8(pack8(x))
        bad = torch.zeros(3, 100, dtype=torch.bool, device="cuda")
        bad[0, 32:64], bad[1, 96:], bad[2, :32] = True, True, True
        assert torch.equal(h.isnan(), bad)
        assert torch.equal(pack8(x.cpu()).scales, pack8(x).scales.cpu())


def _phi(x):
    return torch.special.erfc(-x / math.sqrt(2)) / 2


def _gelu_tols(x, dy, k, y, dx, dt):
    tail = _phi(-x.abs())
    ty = (_half(dt) * y.abs() + x.abs() * (tail * (1e-7 + (32 + x * x) * U) + 2 * U) + _tiny(dt))
    tail = _phi(-k.abs())
    dens = torch.exp(-k * k / 2) / math.sqrt(2 * math.pi)
    slope = tail * (1e-7 + (32 + k * k) * U) + 4 * U + (k.abs() * dens) * (8 + k * k) * U
    return ty, _half(dt) * dx.abs() + dy.abs() * slope + _tiny(dt)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_gelu(shape, dt):
    from zookeeper_amd.ops import gelu8

    torch.manual_seed(sum(shape))
    x = (torch.randn(shape, device="cuda") * 3).to(dt).requires_grad_(True)
    dy = torch.randn(shape, device="cuda").to(dt)
    y = gelu8(x)
    dx, = torch.autograd.grad(y, x, dy)
    assert y.dtype == dx.dtype == dt
    xd, kd, dyd = x.detach().double(), _held(x.detach()), dy.double()
    want_y = xd * _phi(xd)
    want = dyd * (_phi(kd) + kd * torch.exp(-kd * kd / 2) / math.sqrt(2 * math.pi))
    ty, tdx = _gelu_tols(xd, dyd, kd, want_y, want, dt)
    assert ((y.detach().double() - want_y).abs() <= ty).all()
    assert ((dx.double() - want).abs() <= tdx).all()
    with torch.no_grad():
        assert torch.equal(gelu8(x), y)


def test_gelu_far_values_and_differences():
    from zookeeper_amd.ops import gelu8

    x = torch.tensor([[-40.0, -14.0, -6.0, 0.0, 6.0, 14.0, 40.0, 1e30, -1e30]], device="cuda")
    y = gelu8(x)
    want = x.double() * _phi(x.double())
    xd = x.double()
    tail = _phi(-xd.abs())
    assert ((y.double() - want).abs() <= xd.abs() * tail * (1e-7 + (32 + xd * xd) * U)
            + 4 * U * want.abs() + 2.0 ** -126).all()
    assert torch.equal(gelu8(torch.tensor([float("inf")], device="cuda")),
                       torch.tensor([float("inf")], device="cuda"))
    assert gelu8(torch.full((3,), float("nan"), device="cuda")).isnan().all()
    # values that the form holds exactly: the gradient is the function's own slope
    x = (torch.randint(-60, 61, (4, 64), device="cuda").float() / 32)
    x[:, ::32] = 127 / 64  # every block's step is 1 / 64
    x.requires_grad_(True)
    g, = torch.autograd.grad(gelu8(x).sum(), x)
    h = 2.0 ** -8
    with torch.no_grad():
        d = (gelu8(x + h).double() - gelu8(x - h).double()) / (2 * h)
    # outputs under 2 are off by under 40 u; a third derivative of at most 1.2
    assert ((g.double() - d).abs() <= 40 * U / h + 1.2 * h * h / 6).all()


def test_gelu_strides():
    from zookeeper_amd.ops import gelu8

    base = torch.randn(6, 5, 150, device="cuda").bfloat16()
    for x in (base[..., 3:103], base.transpose(0, 1)[..., :64], base[:, ::2, :96],
              base.permute(0, 2, 1), base[0, 0, :50].expand(4, 50)):
        x = x.detach().requires_grad_(True)
        y = gelu8(x)
        g, = torch.autograd.grad(y.sum(), x)
        c = x.detach().contiguous().requires_grad_(True)
        yc = gelu8(c)
        gc, = torch.autograd.grad(yc, c, torch.ones_like(c))
        assert torch.equal(y, yc) and torch.equal(g, gc)


GEMMS = [(1, 1, 1), (1, 130, 70), (33, 5, 300), (300, 128, 128), (257, 129, 127), (512, 256, 256),
         (1000, 515, 1001), (5000, 64, 40), (40000, 16, 24), (700, 1, 600), (70, 600, 1),
         (2049, 384, 640), (4096, 1024, 512), (64, 2048, 1536), (1300, 1000, 512)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,outs,cols", GEMMS)
def test_dense_gradients(rows, outs, cols, dt):
    from zookeeper_amd.ops import dense8_grads, pack8

    torch.manual_seed(rows + outs + cols)
    x = torch.randn(rows, cols, device="cuda").to(dt)
    dy = torch.randn(rows, outs, device="cuda").to(dt)
    kept = pack8(x)
    dw, db = dense8_grads(dy, kept)
    assert dw.dtype == db.dtype == torch.float32
    h, d = _held(x), dy.double()
    tol = (rows + 16) * 2.0 ** -23
    assert ((dw.double() - d.t() @ h).abs() <= tol * (d.abs().t() @ h.abs()) + 1e-30).all()
    assert ((db.double() - d.sum(0)).abs() <= tol * d.abs().sum(0) + 1e-30).all()
    # right on average too: a random walk of roundings, not a drift
    rel = (dw.double() - d.t() @ h).norm() / (d.t() @ h).norm().clamp_min(1e-30)
    assert rel <= 64 * U * max(1.0, math.sqrt(rows / 64))
    again = dense8_grads(dy, kept, bias=False)
    assert again[1] is None and torch.equal(again[0], dw)


WIDE = [(64, 1, 64), (65, 5, 70), (130, 300, 100), (257, 257, 257), (700, 1, 600),
        (1000, 515, 1001), (2049, 384, 640), (4096, 1024, 512), (64, 2048, 1536),
        (1300, 1000, 512), (9001, 72, 96), (3333, 260, 67)]


@pytest.mark.parametrize("variant", [0, 1])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,outs,cols", WIDE)
def test_dense_gradients_of_each_kernel(rows, outs, cols, dt, variant):
    from zookeeper_amd.ops import pack8
    from zookeeper_amd.ops.act8 import _dense_grads

    torch.manual_seed(rows + outs + cols)
    x = torch.randn(rows, cols, device="cuda").to(dt)
    dy = torch.randn(rows, outs, device="cuda").to(dt)
    kept = pack8(x)
    h, d = _held(x), dy.double()
    tol = (rows + 16) * 2.0 ** -23
    want, mag = d.t() @ h, d.abs().t() @ h.abs()
    wb, mb = d.sum(0), d.abs().sum(0)
    dw, db = _dense_grads(dy, kept.codes, kept.scales, True, variant=variant)
    assert ((dw.double() - want).abs() <= tol * mag + 1e-30).all()
    assert ((db.double() - wb).abs() <= tol * mb + 1e-30).all()
    # added to buffers, and again: the same bits
    w2, b2 = torch.ones_like(dw), torch.full_like(db, 2.0)
    _dense_grads(dy, kept.codes, kept.scales, True, w2, b2, variant=variant)
    assert torch.equal(w2, dw + 1) and torch.equal(b2, db + 2)


@pytest.mark.parametrize("variant", [0, 1])
def test_dense_gradients_of_extreme_values(variant):
    """Kept values from the smallest step to the largest, dy scaled against them."""
    from zookeeper_amd.ops import pack8
    from zookeeper_amd.ops.act8 import _dense_grads

    torch.manual_seed(7)
    rows, outs, cols = 130, 70, 128
    big = torch.finfo(torch.float32).max
    x = torch.rand(rows, cols, device="cuda") * 2 - 1
    x[:, :32] *= big
    x[::3, 0], x[1::3, 1] = big, -big
    x[:, 32:64] *= 2.0 ** -119
    x[:, 64:96] *= 2.0 ** -127  # subnormal
    kept = pack8(x)
    assert int(kept.scales.max()) == 254 and int(kept.scales.min()) == 7
    h = _held(x)
    for scale, lo, hi in ((2.0 ** -40, 0, 32), (2.0 ** 40, 32, 96), (1.0, 96, 128)):
        dy = torch.randn(rows, outs, device="cuda") * scale
        for dt in (torch.float32, torch.bfloat16):
            d = dy.to(dt).double()
            dw, _ = _dense_grads(dy.to(dt), kept.codes, kept.scales, True, variant=variant)
            mag = d.abs().t() @ h.abs()
            err = (dw.double() - d.t() @ h).abs()[:, lo:hi]
            assert (err <= (rows + 16) * 2.0 ** -23 * mag[:, lo:hi]).all()


def test_dense_rows_with_gaps_and_special_values():
    from zookeeper_amd.ops import dense8_grads, pack8

    torch.manual_seed(0)
    for dt in DTYPES:
        base = torch.randn(200, 3, 70, device="cuda").to(dt)
        x = torch.randn(200, 90, device="cuda").to(dt)
        dy = base[:, 1, 3:68]
        dw, db = dense8_grads(dy, pack8(x))
        cw, cb = dense8_grads(dy.contiguous(), pack8(x))
        assert torch.equal(dw, cw) and torch.equal(db, cb)
        one = base[0, 0, :65].expand(200, 65)  # the gradient of a sum: no rows of its own
        dw, db = dense8_grads(one, pack8(x))
        cw, cb = dense8_grads(one.contiguous(), pack8(x))
        assert torch.equal(dw, cw) and torch.equal(db, cb)
        # a NaN in dy stays in its row of dw, one in x in its block's columns
        dy = torch.randn(200, 65, device="cuda").to(dt)
        dy[5, 7] = float("inf")
        dw, db = dense8_grads(dy, pack8(x))
        assert db[7].isinf() and db[:7].isfinite().all() and db[8:].isfinite().all()
        bad = ~dw.isfinite()
        assert bad[7].all() and not bad[:7].any() and not bad[8:].any()
        dy[5, 7] = 1
        x[9, 40] = float("nan")
        dw, db = dense8_grads(dy, pack8(x))
        assert dw[:, 32:64].isnan().all() and db.isfinite().all()
        assert dw[:, :32].isfinite().all() and dw[:, 64:].isfinite().all()


def test_fp32_gradients_keep_fp32_products():
    from zookeeper_amd.ops import dense8_grads, pack8

    # 24-bit values against one kept value each: the products are exact
    dy = torch.zeros(40, 130, device="cuda")
    dy[0] = torch.randn(130, device="cuda") * torch.exp2(
        torch.randint(-60, 60, (130,), device="cuda").float())
    x = torch.zeros(40, 33, device="cuda")
    x[0, 0], x[0, 32] = 1.0, -0.5
    dw, _ = dense8_grads(dy, pack8(x))
    assert torch.equal(dw[:, 0], dy[0]) and torch.equal(dw[:, 32], dy[0] * -0.5)
    assert (dw[:, 1:32] == 0).all()


def test_dense_layer_and_autograd():
    from zookeeper_amd.ops import dense8

    torch.manual_seed(1)
    for dt in DTYPES:
        x = torch.randn(3, 50, 72, device="cuda").to(dt).requires_grad_(True)
        w = (torch.randn(40, 72, device="cuda") / 8).requires_grad_(True)
        b = torch.randn(40, device="cuda").requires_grad_(True)
        dy = torch.randn(3, 50, 40, device="cuda").to(dt)
        y = dense8(x, w, b)
        assert torch.equal(y, torch.nn.functional.linear(x, w.to(dt), b.to(dt)))
        dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
        d = dy.double().reshape(-1, 40)
        h = _held(x.detach()).reshape(-1, 72)
        tol = 166 * 2.0 ** -23
        assert dw.dtype == torch.float32
        assert ((dw.double() - d.t() @ h).abs() <= tol * (d.abs().t() @ h.abs())).all()
        assert ((db.double() - d.sum(0)).abs() <= tol * d.abs().sum(0)).all()
        assert torch.equal(dx, torch.matmul(dy, w.to(dt)))
        # only the bias wants a gradient: nothing is kept
        y = dense8(x.detach(), w.detach(), b)
        gb, = torch.autograd.grad(y, b, dy)
        assert ((gb.double() - d.sum(0)).abs() <= tol * d.abs().sum(0)).all()
        with pytest.raises(RuntimeError, match="not differentiable"):
            torch.autograd.grad(dense8(x, w, b).sum(), w, create_graph=True)


def test_accumulates_into_the_flat_gradient():
    from zookeeper_amd import nn as znn
    from zookeeper_amd.parallel.flat import FlatParams

    torch.manual_seed(2)
    for rows in (40, 9000):  # one split, several
        m = znn.QuantDense(64, 48, use_bias=True, kept="int8").cuda()
        x = torch.randn(rows, 64, device="cuda")
        dy = torch.randn(rows, 48, device="cuda")
        m(x).backward(dy)
        gw, gb = m.weight.grad.clone(), m.bias.grad.clone()
        FlatParams(m, torch.device("cuda"))
        m.weight.grad.fill_(2.0)
        m.bias.grad.fill_(-1.0)
        m(x).backward(dy)
        assert torch.equal(m.weight.grad, gw + 2.0) and torch.equal(m.bias.grad, gb - 1.0)


def test_no_rows():
    from zookeeper_amd.ops import dense8_grads, gelu8, pack8, unpack8

    x = torch.randn(0, 40, device="cuda", requires_grad=True)
    assert unpack8(pack8(x)).shape == (0, 40)
    assert torch.autograd.grad(gelu8(x).sum(), x)[0].shape == (0, 40)
    dw, db = dense8_grads(torch.randn(0, 30, device="cuda"), pack8(x))
    assert torch.equal(dw, torch.zeros(30, 40, device="cuda"))
    assert torch.equal(db, torch.zeros(30, device="cuda"))


def test_replays_in_a_graph():
    from zookeeper_amd.ops import dense8_grads, gelu8, pack8

    torch.manual_seed(3)
    dy = torch.randn(3000, 72, device="cuda").bfloat16()

    def step(v):
        v = v.detach().requires_grad_(True)
        y = gelu8(v)
        dx, = torch.autograd.grad(y, v, torch.ones_like(y))
        return [y.detach(), dx, *dense8_grads(dy, pack8(y.detach()))]

    static = torch.randn(3000, 90, device="cuda").bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for k in range(3):
        new = torch.randn(3000, 90, device="cuda").bfloat16()
        static.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(out, step(new)):
            assert torch.equal(a, e), k


def test_the_operators_together():
    """norm -> dense -> GELU -> dense -> log probabilities, all gradients, against
    the same network of 64-bit operations on the kept values."""
    from zookeeper_amd import nn as znn
    from zookeeper_amd import ops

    torch.manual_seed(4)
    net = torch.nn.Sequential(
        znn.LayerNorm(64), znn.QuantDense(64, 96, use_bias=True, kept="int8"),
        znn.GELU(kept="int8"), znn.QuantDense(96, 50, use_bias=True, kept="int8")).cuda()
    x = torch.randn(4, 33, 64, device="cuda")
    t = torch.randint(0, 50, (4, 33), device="cuda")
    acts = [x]
    for m in net:
        acts.append(m(acts[-1]))
        acts[-1].retain_grad()
    r = ops.token_logprobs(acts[-1], t)
    loss = -(r.logp + 0.1 * r.entropy).mean()
    loss.backward()

    ln, d1, _, d2 = net
    h0 = torch.nn.functional.layer_norm(x.double(), (64,), ln.weight.double(), ln.bias.double(),
                                        1e-3)
    h1 = torch.nn.functional.linear(h0, d1.weight.double(), d1.bias.double())
    h2 = h1 * _phi(h1)
    z = torch.nn.functional.linear(h2, d2.weight.double(), d2.bias.double()).detach()
    z.requires_grad_(True)
    lp = torch.log_softmax(z, -1)
    ref = -(lp.gather(-1, t[..., None])[..., 0] - 0.1 * (lp.exp() * lp).sum(-1)).mean()
    gz, = torch.autograd.grad(ref, z)
    k2, k1, k0 = (_held(acts[i].detach()) for i in (3, 2, 1))
    gh2 = gz @ d2.weight.double()
    gh1 = gh2 * (_phi(k1) + k1 * torch.exp(-k1 * k1 / 2) / math.sqrt(2 * math.pi))
    gh0 = gh1 @ d1.weight.double()
    n = (x.double() - x.double().mean(-1, keepdim=True))
    n = n / torch.sqrt(n.square().mean(-1, keepdim=True) + 1e-3)

    def dw(g, k):
        return g.reshape(-1, g.shape[-1]).t() @ k.reshape(-1, k.shape[-1])

    pairs = [(loss, ref), (acts[-1].grad, gz), (d2.weight.grad, dw(gz, k2)),
             (d2.bias.grad, gz.sum((0, 1))), (d1.weight.grad, dw(gh1, k0)),
             (d1.bias.grad, gh1.sum((0, 1))), (ln.weight.grad, (gh0 * n).sum((0, 1))),
             (ln.bias.grad, gh0.sum((0, 1)))]
    for got, want in pairs:
        # each value is a sum of at most 132 * 96 terms through five fp32 layers
        assert (got.double() - want).norm() <= 2e-5 * want.norm()


def test_gradients_of_other_layouts():
    """Incoming gradients that are transposed, sliced or broadcast."""
    from zookeeper_amd.ops import dense8, gelu8

    torch.manual_seed(6)
    for shape in ((12, 40), (3, 4, 40)):
        x = torch.randn(shape, device="cuda", requires_grad=True)
        w = torch.randn(40, 40, device="cuda", requires_grad=True)
        flip = torch.randn(*reversed(shape), device="cuda").permute(*reversed(range(len(shape))))
        wide = torch.randn(*shape[:-1], 57, device="cuda")[..., 9:49]
        row = torch.randn(40, device="cuda").expand(shape)
        for dy in (flip, wide, row):
            got, = torch.autograd.grad(gelu8(x), x, dy)
            want, = torch.autograd.grad(gelu8(x), x, dy.contiguous())
            assert torch.equal(got, want)
            got, = torch.autograd.grad(dense8(x, w), w, dy)
            want, = torch.autograd.grad(dense8(x, w), w, dy.contiguous())
            assert torch.equal(got, want)


def _form_of_small_steps(rows, cols):
    """Codes of the whole range under the scale bytes 0 .. 8 (one to a row), which no
    packed tensor has under 7 but other producers' forms do, and what they stand for
    by the form's definition."""
    from zookeeper_amd.ops import Packed8

    g = torch.Generator().manual_seed(3)
    codes = torch.randint(-127, 128, (rows, cols), generator=g, dtype=torch.int32).to(torch.int8)
    scales = (torch.arange(rows).view(-1, 1) % 9).expand(rows, -(-cols // 32)).to(torch.uint8)
    value = codes.double() * torch.exp2(scales[:, :1].double() - 133)
    kept = Packed8(codes.cuda(), scales.contiguous().cuda(), torch.float32)
    return kept, value.cuda()


def test_small_steps_unpacked_and_in_gelu():
    from zookeeper_amd.ops import unpack8
    from zookeeper_amd.ops.act8 import _Gelu8Fn

    kept, value = _form_of_small_steps(18, 100)
    assert torch.equal(unpack8(kept, torch.float32).double(), value)
    assert torch.equal(unpack8(kept, torch.bfloat16).double(), value)  # exact in bf16
    assert torch.equal(unpack8(kept, torch.float16).double(), value.to(torch.float16).double())

    class Ctx:
        rows = 18
        saved_tensors = (torch.cat([kept.codes.view(torch.uint8).reshape(-1),
                                    kept.scales.reshape(-1)]),)

    with torch.no_grad():
        dx = _Gelu8Fn.backward(Ctx, torch.full((18, 100), 3.0, device="cuda"))
    # the slope at |x| < 2^-117 is 1 / 2 + O(x): one rounding of Phi, of the sum and of
    # the product each, the fit's 1e-7
    assert ((dx - 1.5).abs() <= 1.5 * (1e-7 + 4 * 2.0 ** -24)).all()


@pytest.mark.parametrize("variant", [0, 1])
@pytest.mark.parametrize("dt", DTYPES)
def test_small_steps_in_the_weight_gradient(dt, variant):
    """Both kernels decode the same values; dy is scaled up so that the products are
    normal numbers."""
    from zookeeper_amd.ops.act8 import _dense_grads

    rows, outs, cols = 189, 70, 130
    kept, value = _form_of_small_steps(rows, cols)
    torch.manual_seed(4)
    up = 2.0 ** 14 if dt == torch.float16 else 2.0 ** 60
    dy = (torch.randn(rows, outs, device="cuda").clamp(-3.9, 3.9) * up).to(dt)
    dw, db = _dense_grads(dy, kept.codes, kept.scales, True, variant=variant)
    d = dy.double()
    want, mag = d.t() @ value, d.abs().t() @ value.abs()
    # every product exact, a sum of them off by a rounding each (as above); fp16: a step
    # of the subnormals each, where the sums fall under the normal range
    tol = (rows + 16) * (2.0 ** -23 * mag + (2.0 ** -149 if dt == torch.float16 else 0))
    assert ((dw.double() - want).abs() <= tol).all()
    zero = torch.zeros_like(kept.codes)
    dw, _ = _dense_grads(dy, zero, torch.zeros_like(kept.scales), True, variant=variant)
    assert torch.equal(dw, torch.zeros_like(dw))


@pytest.mark.parametrize("flat", [False, True])
@pytest.mark.parametrize("rows,outs,dt", [(1, 5, torch.float32), (5000, 33, torch.float16),
                                          (100000, 7, torch.bfloat16)])
def test_bias_of_a_frozen_weight_replays_in_a_graph(rows, outs, dt, flat):
    from zookeeper_amd.ops import dense8
    from zookeeper_amd.parallel.flat import FlatParams

    torch.manual_seed(rows)
    m = torch.nn.Module()
    m.b = torch.nn.Parameter(torch.randn(outs, device="cuda"))
    w = torch.randn(outs, 20, device="cuda")
    if flat:
        f = FlatParams(m)
    x = torch.zeros(rows, 20, device="cuda", dtype=dt)
    dy = torch.zeros(rows, outs, device="cuda", dtype=dt)

    def step():
        if flat:
            m.b.grad.zero_()
            dense8(x, w, m.b).backward(dy)
            return m.b.grad
        return torch.autograd.grad(dense8(x, w, m.b), m.b, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        dy.copy_(torch.randn(rows, outs, device="cuda").to(dt))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        want, mag = dy.double().sum(0), dy.double().abs().sum(0)
        assert ((got.double() - want).abs() <= (rows + 16) * 2.0 ** -23 * mag).all(), i
        assert torch.equal(step(), got), i
        torch.cuda.synchronize()


@pytest.mark.parametrize("shape", [(0, 40), (3, 0), (0, 0), (0,)])
def test_a_form_of_nothing(shape):
    """What the constructor takes unpacks, as on the host."""
    from zookeeper_amd.ops import Packed8, unpack8

    for device in ("cuda", "cpu"):
        codes = torch.zeros(shape, dtype=torch.int8, device=device)
        scales = torch.zeros((*shape[:-1], -(-shape[-1] // 32)), dtype=torch.uint8, device=device)
        out = unpack8(Packed8(codes, scales, torch.bfloat16))
        assert out.shape == shape and out.dtype == torch.bfloat16
