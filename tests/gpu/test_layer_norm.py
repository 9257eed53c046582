"""Layer norm kernels against the definition in 64 bits.

Tolerances: with ``u`` half a unit of the output type (``finfo.eps / 2``), an
output is one rounding of an fp32 value, ``u * |value|``; the fp32 value itself
is off by a few fp32 units of the row's terms (mean, rstd, product), taken as
``32 * 2^-24`` of the largest magnitude that enters it.  Column sums over R rows
add at most ``R * 2^-24`` of the sum of the terms' magnitudes."""

import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from zookeeper_amd import ops

    assert ops.available(), ops.load_error()


def _half(dt):
    return torch.finfo(dt).eps / 2


def _reference(x, w, b, eps, dy):
    x, dy = x.double(), dy.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + eps)
    h = (x - mean) * rstd
    wd = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.double()
    bd = torch.zeros_like(wd) if b is None else b.double()
    g = dy * wd
    dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    lead = list(range(x.dim() - 1))
    mag = {"y": (h * wd).abs() + bd.abs(), "rstd": rstd,
           "dx": rstd * (g.abs() + g.abs().mean(-1, keepdim=True)
                         + h.abs() * (g * h).abs().mean(-1, keepdim=True)),
           "x": x.abs().amax(-1, keepdim=True), "wd": wd.abs(), "g": g.abs(),
           "dw": (dy * h).abs().sum(lead), "db": dy.abs().sum(lead),
           # an error e of (x - mean) * rstd in every row moves dw by sum |dy| e
           "dw_x": (dy.abs() * rstd * x.abs().amax(-1, keepdim=True)).sum(lead)}
    return h * wd + bd, dx, (dy * h).sum(lead), dy.sum(lead), mag


def _check(x, w, b, eps, y, dx, dw, db, dy):
    ry, rdx, rdw, rdb, m = _reference(x, w, b, eps, dy)
    dt = x.dtype
    # |x - mean| carries the rounding of the mean: U32 * max |x|, scaled by rstd
    off = 32 * U32 * m["rstd"] * m["x"]
    tol = _half(dt) * ry.abs() + 32 * U32 * m["y"] + off * m["wd"] + torch.finfo(dt).tiny
    assert ((y.double() - ry).abs() <= tol).all(), ((y.double() - ry).abs() - tol).max()
    if dx is not None:
        # xhat is off by `off` in each of two factors of the last term
        gmean = m["g"].mean(-1, keepdim=True)
        xhat = (x.double() - x.double().mean(-1, keepdim=True)) * m["rstd"]
        tol = (_half(dt) * rdx.abs() + 64 * U32 * m["dx"] + torch.finfo(dt).tiny
               + m["rstd"] * off * gmean * 4 * (1 + xhat.abs()))
        if dt == torch.float16:
            tol = tol + 2.0 ** -25  # half a step of fp16's subnormals
        assert ((dx.double() - rdx).abs() <= tol).all(), ((dx.double() - rdx).abs() - tol).max()
    rows = x.numel() // x.shape[-1]
    n = (rows + 32) * U32
    if dw is not None:
        tol = n * m["dw"] + 32 * U32 * m["dw_x"] + 1e-30
        assert ((dw.double() - rdw).abs() <= tol).all(), ((dw.double() - rdw).abs() / tol).max()
    if db is not None:
        assert ((db.double() - rdb).abs() <= n * m["db"] + 1e-30).all()


SHAPES = [(1, 1), (1, 4096), (3, 5), (70, 31), (129, 33), (5, 128), (300, 200), (9, 512),
          (33, 777), (17, 1024), (50, 2047), (64, 2048), (1030, 2049), (11, 4096), (7, 5001),
          (5, 8192), (6, 12289), (3, 16384), (4, 16385), (70, 20000), (2, 50001), (5000, 8),
          (4999, 96)]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward_and_gradients(rows, cols, dt):
    from zookeeper_amd.ops import layer_norm

    torch.manual_seed(rows * 31 + cols)
    x = (torch.randn(rows, cols, device="cuda") * 2 + 0.5).to(dt).requires_grad_(True)
    w = (1 + 0.2 * torch.randn(cols, device="cuda")).requires_grad_(True)
    b = (0.2 * torch.randn(cols, device="cuda")).requires_grad_(True)
    dy = torch.randn(rows, cols, device="cuda").to(dt)
    y = layer_norm(x, w, b, 1e-3)
    assert y.dtype == dt and y.shape == x.shape and y.is_contiguous()
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    _check(x.detach(), w.detach(), b.detach(), 1e-3, y.detach(), dx, dw, db, dy)
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, 1e-3), y)


@pytest.mark.parametrize("cols", [64, 1000, 3000, 17000])
def test_without_parameters_and_partial_gradients(cols):
    from zookeeper_amd.ops import layer_norm

    torch.manual_seed(0)
    x = torch.randn(37, cols, device="cuda", requires_grad=True)
    dy = torch.randn(37, cols, device="cuda")
    y = layer_norm(x, eps=1e-5)
    _check(x.detach(), None, None, 1e-5, y.detach(), torch.autograd.grad(y, x, dy)[0], None,
           None, dy)
    w = torch.rand(cols, device="cuda", requires_grad=True)
    y = layer_norm(x.detach(), w, None, 1e-5)
    _check(x.detach(), w.detach(), None, 1e-5, y.detach(), None,
           torch.autograd.grad(y, w, dy)[0], None, dy)
    b = torch.rand(cols, device="cuda", requires_grad=True)
    y = layer_norm(x.detach(), w.detach(), b, 1e-5)
    _check(x.detach(), w.detach(), b.detach(), 1e-5, y.detach(), None, None,
           torch.autograd.grad(y, b, dy)[0], dy)


def test_strides_leading_dims_and_broadcast():
    from zookeeper_amd.ops import layer_norm

    torch.manual_seed(1)
    w, b = torch.rand(96, device="cuda"), torch.rand(96, device="cuda")
    base = torch.randn(5, 7, 131, device="cuda")
    for x in (base[..., 3:99], base[:, ::2, :96], base.transpose(0, 1)[..., 1:97],
              torch.randn(7, 96, 5, device="cuda").transpose(1, 2),  # no unit stride inside a row
              torch.randn(96, device="cuda"), torch.randn(96, device="cuda").expand(4, 96)):
        x = x.detach().requires_grad_(True)
        y = layer_norm(x, w, b)
        dy = torch.randn(y.shape, device="cuda")
        dx, = torch.autograd.grad(y, x, dy)
        _check(x.detach(), w, b, 1e-3, y.detach(), dx, None, None, dy)
        # an incoming gradient without rows of its own (a sum's)
        y = layer_norm(x, w, b)
        dx, = torch.autograd.grad(y.sum(), x)
        _check(x.detach(), w, b, 1e-3, y.detach(), dx, None, None, torch.ones_like(y))


def test_bf16_parameters_and_constant_rows():
    from zookeeper_amd.ops import layer_norm

    x = torch.full((4, 100), 7.25, device="cuda", dtype=torch.bfloat16)
    x[1] = 0
    w = torch.rand(100, device="cuda").bfloat16().requires_grad_(True)
    b = torch.rand(100, device="cuda").bfloat16().requires_grad_(True)
    y = layer_norm(x, w, b)
    assert torch.equal(y, b.expand(4, 100))  # the variance is exactly 0
    gw, gb = torch.autograd.grad(y, [w, b], torch.ones_like(y))
    assert gw.dtype == gb.dtype == torch.bfloat16
    assert torch.equal(gw, torch.zeros_like(gw)) and torch.equal(gb, torch.full_like(gb, 4))


def test_far_from_zero_mean():
    """A mean of 1000 standard deviations: the centred variance keeps its digits."""
    from zookeeper_amd.ops import layer_norm

    torch.manual_seed(2)
    x = torch.randn(8, 1536, device="cuda") + 1000
    y = layer_norm(x, eps=0.0)
    r = torch.nn.functional.layer_norm(x.double(), (1536,), eps=0.0)
    # the mean is rounded to a step of 2^-14 at 1000
    assert (y.double() - r).abs().max() < 2.0 ** -13


def test_nan_and_infinity_stay_in_their_row():
    from zookeeper_amd.ops import layer_norm

    x = torch.randn(6, 300, device="cuda")
    y0 = layer_norm(x)
    x[2, 5], x[4, 7] = float("nan"), float("inf")
    y = layer_norm(x)
    assert y[2].isnan().all() and y[4].isnan().all()
    for r in (0, 1, 3, 5):
        assert torch.equal(y[r], y0[r])


def test_no_rows():
    from zookeeper_amd.ops import layer_norm

    x = torch.randn(0, 64, device="cuda", requires_grad=True)
    w = torch.rand(64, device="cuda", requires_grad=True)
    y = layer_norm(x, w)
    assert y.shape == (0, 64)
    dx, dw = torch.autograd.grad(y.sum(), [x, w])
    assert dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(w))


def test_gradient_matches_differences():
    from zookeeper_amd.ops import layer_norm

    torch.manual_seed(3)
    x = torch.randn(3, 40, device="cuda", requires_grad=True)
    w = torch.rand(40, device="cuda", requires_grad=True)
    b = torch.rand(40, device="cuda", requires_grad=True)
    r = torch.randn(3, 40, device="cuda")
    grads = torch.autograd.grad((layer_norm(x, w, b) * r).sum(), [x, w, b])
    h = 2.0 ** -6
    for t, g in zip((x, w, b), grads):
        d = torch.randn_like(t)

        def f(s):
            args = [(v + s * d if v is t else v).detach() for v in (x, w, b)]
            return (layer_norm(*args).double() * r).sum()

        got = float((f(h) - f(-h)) / (2 * h))
        want = float((g.double() * d).sum())
        # fp32 outputs over 2h, and h^2 / 6 of a third derivative of order 100
        assert abs(got - want) <= 120 * 8 * U32 / h * 4 + 100 * h * h / 6 * 4, (got, want)


def test_accumulates_into_the_flat_gradient():
    from zookeeper_amd import nn as znn
    from zookeeper_amd.parallel.flat import FlatParams

    torch.manual_seed(4)
    m = znn.LayerNorm(48).cuda()
    x = torch.randn(20, 48, device="cuda")
    m(x).square().sum().backward()
    gw, gb = m.weight.grad.clone(), m.bias.grad.clone()
    FlatParams(m, torch.device("cuda"))
    m.weight.grad.fill_(2.0)
    m.bias.grad.fill_(-1.0)
    m(x).square().sum().backward()
    assert torch.equal(m.weight.grad, gw + 2.0) and torch.equal(m.bias.grad, gb - 1.0)


def test_replays_in_a_graph_and_on_another_stream():
    from zookeeper_amd.ops import layer_norm

    torch.manual_seed(5)
    x = torch.randn(40, 1500, device="cuda").bfloat16()
    w = torch.rand(1500, device="cuda")
    dy = torch.randn(40, 1500, device="cuda").bfloat16()

    def step(xin):
        xl, wl = xin.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = layer_norm(xl, wl)
        return [y.detach(), *torch.autograd.grad(y, [xl, wl], dy)]

    static = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(static)
    for k in range(3):
        new = torch.randn(40, 1500, device="cuda").bfloat16()
        static.copy_(new)
        g.replay()
        torch.cuda.synchronize()
        for a, e in zip(out, step(new)):
            assert torch.equal(a, e), k


def test_second_derivative_is_refused():
    from zookeeper_amd.ops import layer_norm

    x = torch.randn(4, 32, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(layer_norm(x).sum(), x, create_graph=True)


def test_gradients_of_other_layouts():
    """Incoming gradients that are transposed, sliced or broadcast, two and three
    dimensions: dx has the input's shape, row by row."""
    from zookeeper_amd.ops import layer_norm

    torch.manual_seed(6)
    for shape in ((12, 40), (3, 4, 40)):
        x = torch.randn(shape, device="cuda", requires_grad=True)
        w = torch.rand(40, device="cuda", requires_grad=True)
        flip = torch.randn(*reversed(shape), device="cuda").permute(*reversed(range(len(shape))))
        wide = torch.randn(*shape[:-1], 57, device="cuda")[..., 9:49]
        row = torch.randn(40, device="cuda").expand(shape)
        for dy in (flip, wide, row):
            got = torch.autograd.grad(layer_norm(x, w), [x, w], dy)
            want = torch.autograd.grad(layer_norm(x, w), [x, w], dy.contiguous())
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("cols", [1, 2, 4, 8, 64, 4096, 32768])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_large_constant_rows(cols, dt):
    """Rows of one large value and a small eps: xhat is 0 and dx the gradient without its
    mean, also where the width does not fill the lanes."""
    from zookeeper_amd.ops import layer_norm

    # powers of two: the sum, the mean and the differences of 0 are exact
    torch.manual_seed(9)
    x = torch.full((3, cols), 2.0 ** 112, device="cuda", dtype=dt)
    x[1] = -x[1]
    x.requires_grad_(True)
    w = torch.rand(cols, device="cuda", requires_grad=True)
    dy = torch.randn(3, cols, device="cuda").to(dt)
    y = layer_norm(x, w, eps=1e-12)  # xhat of a 0 would be 2^112 * 1e6: an infinity
    assert torch.equal(y, torch.zeros_like(y))
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    assert torch.equal(dw, torch.zeros_like(dw))
    g = dy.double() * w.double()
    want = (g - g.mean(-1, keepdim=True)) * 1e6
    mag = (g.abs() + g.abs().mean(-1, keepdim=True)) * 1e6
    # rstd, the products, the sum's n / 256 + 16 additions and two more roundings; the store
    tol = (cols / 256 + 32) * U32 * mag + _half(dt) * want.abs()
    assert ((dx.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("flat", [False, True])
def test_one_parameter_as_weight_and_bias(flat):
    from zookeeper_amd.ops import layer_norm
    from zookeeper_amd.parallel.flat import FlatParams

    torch.manual_seed(10)
    m = torch.nn.Module()
    m.p = torch.nn.Parameter(torch.rand(1000, device="cuda"))
    x, dy = torch.randn(300, 1000, device="cuda"), torch.randn(300, 1000, device="cuda")
    w = m.p.detach().clone().requires_grad_(True)
    b = m.p.detach().clone().requires_grad_(True)
    dw, db = torch.autograd.grad(layer_norm(x, w, b), [w, b], dy)
    if flat:
        FlatParams(m).zero_grad()
    layer_norm(x, m.p, m.p).backward(dy)
    torch.cuda.synchronize()
    assert torch.equal(m.p.grad, dw + db)
