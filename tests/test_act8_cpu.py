"""8-bit kept activations on host tensors, their layers and their refusals."""

import math

import pytest
import torch

from zookeeper_amd import nn as znn
from zookeeper_amd.ops import Packed8, dense8, dense8_grads, gelu8, pack8, unpack8


def test_form():
    x = torch.tensor([[127.0, -64.0, 0.4, 0.5, 1.5, 2.5] + [0.0] * 27, [0.0] * 33])
    k = pack8(x)
    assert k.codes[0, :6].tolist() == [127, -64, 0, 0, 2, 2] and k.scales[0, 0] == 133
    assert k.scales.shape == (2, 2) and k.nbytes == 66 + 4
    assert torch.equal(unpack8(k)[1], torch.zeros(33))
    # 127.5 of the largest step would be code 128: the step doubles
    k = pack8(torch.tensor([127.5, 1.0]))
    assert k.codes.tolist() == [64, 0] and k.scales.tolist() == [134]
    big = torch.finfo(torch.float32).max
    k = pack8(torch.tensor([big, -big]))
    assert k.codes.tolist() == [127, -127] and k.scales.tolist() == [254]
    k = pack8(torch.tensor([1.0, float("nan")]))
    assert k.scales.tolist() == [255] and unpack8(k).isnan().all()


def test_error_bound():
    torch.manual_seed(0)
    x = torch.randn(50, 320) * torch.exp2(torch.randint(-30, 30, (50, 1)).float())
    top = x.unflatten(-1, (-1, 32)).abs().amax(-1).repeat_interleave(32, -1)
    # half a step: at most 2^-7 of the largest value, or 1 / 127.5 of it where the
    # step was doubled because it rounds to 128 steps
    err = (unpack8(pack8(x)).double() - x.double()).abs()
    assert (err <= top.double() / 127.5).all()


def test_gradients_are_those_of_the_kept_input():
    torch.manual_seed(1)
    x = torch.randn(5, 40, requires_grad=True)
    dy = torch.randn(5, 40)
    y = gelu8(x)
    torch.testing.assert_close(y, torch.nn.functional.gelu(x))
    k = unpack8(pack8(x.detach())).requires_grad_(True)
    want, = torch.autograd.grad(torch.nn.functional.gelu(k), k, dy)
    torch.testing.assert_close(torch.autograd.grad(y, x, dy)[0], want)

    w, b = torch.randn(7, 40, requires_grad=True), torch.randn(7, requires_grad=True)
    g = torch.randn(5, 7)
    dx, dw, db = torch.autograd.grad(dense8(x, w, b), [x, w, b], g)
    torch.testing.assert_close(dw, g.t() @ k.detach())
    torch.testing.assert_close(db, g.sum(0))
    torch.testing.assert_close(dx, g @ w.detach())
    gw, gb = dense8_grads(g, pack8(x))
    assert torch.equal(gw, dw) and torch.equal(gb, db)


def test_less_is_kept():
    x = torch.randn(64, 256, requires_grad=True)
    kept = []

    def note(t):
        kept.append(t.numel() * t.element_size())
        return t

    with torch.autograd.graph.saved_tensors_hooks(note, lambda t: t):
        gelu8(x)
    assert sum(kept) == 64 * 256 + 64 * 8


def test_layers():
    m = torch.nn.Sequential(znn.QuantDense(8, 16, use_bias=True, kept="int8"),
                            znn.GELU(kept="int8"), znn.QuantDense(16, 3, kept="int8"))
    x = torch.randn(4, 8)
    m(x).sum().backward()
    assert all(p.grad is not None for p in m.parameters())
    plain = znn.GELU()
    assert torch.equal(plain(x), torch.nn.functional.gelu(x))
    with pytest.raises(ValueError, match="kept"):
        znn.GELU(kept="fp4")
    with pytest.raises(ValueError, match="float layers"):
        znn.QuantDense(8, 8, input_quantizer="ste_sign", kept="int8")


def test_refusals():
    x = torch.randn(3, 40)
    for f in (pack8, gelu8):
        with pytest.raises(ValueError, match="last dimension"):
            f(torch.tensor(1.0))
        with pytest.raises(ValueError, match="last dimension"):
            f(torch.randn(2, 0))
        with pytest.raises(ValueError, match="floating"):
            f(torch.ones(3, dtype=torch.int32))
    k = pack8(x)
    with pytest.raises(ValueError, match="rows differ"):
        dense8_grads(torch.randn(4, 5), k)
    with pytest.raises(ValueError, match="rows differ"):
        dense8_grads(torch.randn(5), k)
    with pytest.raises(ValueError, match="weight"):
        dense8(x, torch.randn(5, 41))
    with pytest.raises(ValueError, match="weight"):
        dense8(x, torch.randn(0, 40))
    with pytest.raises(ValueError, match="bias"):
        dense8(x, torch.randn(5, 40), torch.randn(4))
    with pytest.raises(ValueError, match="floating"):
        dense8(x, torch.ones(5, 40, dtype=torch.int32))
    for codes, scales in ((k.codes.float(), k.scales), (k.codes, k.scales[:, :1]),
                          (k.codes, k.scales.to(torch.int8)), (k.codes[:, ::2], k.scales[:, :1])):
        with pytest.raises(ValueError, match="Packed8"):
            Packed8(codes, scales, torch.float32)
    with pytest.raises(RuntimeError, match="not differentiable"):
        v = x.clone().requires_grad_(True)
        torch.autograd.grad(gelu8(v).sum(), v, create_graph=True)
    assert math.isfinite(float(unpack8(k).sum()))


def test_steps_under_the_smallest_packed_one():
    """Scale bytes that pack8 does not write mean what the form says."""
    scales = torch.arange(10, dtype=torch.uint8).view(10, 1)
    codes = torch.tensor([[-127, -3, 0, 1, 64]] * 10, dtype=torch.int8)
    want = codes.double() * torch.exp2(scales.double() - 133)
    kept = Packed8(codes, scales, torch.float32)
    assert torch.equal(unpack8(kept).double(), want)
    assert torch.equal(unpack8(kept, torch.bfloat16).double(), want)
    dw, _ = dense8_grads(torch.eye(10) * 2.0 ** 100, kept)
    assert torch.equal(dw.double(), want * 2.0 ** 100)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_dense_products_are_no_batched_ones(bias, recorded, dt):
    """Rows that do not merge (permuted, broadcast) are copied to one matrix: torch's
    batched product would take the weight as a transposed view."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Calls(TorchDispatchMode):
        seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen.append(str(func))
            return func(*args, **(kwargs or {}))

    torch.manual_seed(3)
    w = torch.randn(40, 7).t()  # itself a transposed view
    b = torch.randn(7) if bias else None
    base = torch.randn(6, 5, 40).to(dt)
    for x in (base, base.transpose(0, 1), base[:1].expand(4, 5, 40), base[0], base[0, 0],
              base[:0]):
        v = x.detach().requires_grad_(recorded)
        wr = w.detach().requires_grad_(recorded)
        dy = torch.randn(*reversed(x.shape[:-1]), 7)
        dy = dy.permute(*reversed(range(x.dim() - 1)), -1).to(dt)
        with Calls():
            y = dense8(v, wr, b)
            grads = torch.autograd.grad(y, [v, wr], dy) if recorded else ()
        assert y.shape == (*x.shape[:-1], 7) and all(g.shape == u.shape
                                                     for g, u in zip(grads, (x, w)))
        if dt == torch.float32:
            torch.testing.assert_close(y, torch.nn.functional.linear(x, w, b))
            if recorded:
                torch.testing.assert_close(grads[0], dy @ w)
    assert any("mm" in f for f in Calls.seen) and not any("bmm" in f for f in Calls.seen)
