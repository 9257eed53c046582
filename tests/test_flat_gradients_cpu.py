"""When a gradient that an operator adds straight into the flat buffer is complete:
told to the data-parallel bucketer once a pass, behind its last use, whatever uses
the pass has.  On host tensors, with a stand-in for the operators."""

import pytest
import torch
import torch.distributed as dist
from torch.utils.checkpoint import checkpoint

from zookeeper_amd.ops import _rows
from zookeeper_amd.parallel.flat import FlatParams


class _Scale(torch.autograd.Function):
    """x * w with w's gradient added to the flat buffer, as the row operators do it."""

    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x, w)
        ctx.rest = (w, _rows.in_backward())
        return x * w

    @staticmethod
    def backward(ctx, g):
        x, w = ctx.saved_tensors
        p, inner = ctx.rest
        dw = (g * x).sum(0)
        needed, flat = _rows.flat_grad(ctx, p, inner)
        if flat is not None:
            flat += dw
            _rows.written(p)
        return g * w, dw if needed and flat is None else None


class _Layer(torch.nn.Module):
    def __init__(self, n=5):
        super().__init__()
        self.w = torch.nn.Parameter(torch.rand(n) + 0.5)

    def forward(self, x):
        return _Scale.apply(x, self.w)


@pytest.fixture
def layer():
    torch.manual_seed(0)
    m = _Layer()
    flat = FlatParams(m)
    m.seen = []
    m.w._zk_grad_ready = lambda: m.seen.append(flat.grad[:5].clone())
    m.flat = flat
    return m


def _want(f, w):
    """w's gradient by autograd alone."""
    w = w.detach().clone().requires_grad_(True)
    return torch.autograd.grad(f(lambda x: x * w, w), w)[0]


X = torch.randn(3, 5, generator=torch.Generator().manual_seed(1))


def _check(layer, f, passes=1, backward=lambda z: z.backward()):
    layer.flat.zero_grad()
    layer.seen.clear()
    backward(f(layer, layer.w))
    assert len(layer.seen) == passes
    torch.testing.assert_close(layer.w.grad, passes * _want(f, layer.w))
    assert torch.equal(layer.seen[-1], layer.w.grad)  # told when it was complete
    return layer.seen


def test_one_use_and_two(layer):
    _check(layer, lambda m, w: m(X).sum())
    _check(layer, lambda m, w: m(m(X).sin()).sum())
    _check(layer, lambda m, w: (m(X) + m(X.square())).sum())


def test_a_graph_passed_twice(layer):
    def twice(z):
        z.backward(retain_graph=True)
        z.backward()

    seen = _check(layer, lambda m, w: m(m(X).sin()).sum(), 2, twice)
    torch.testing.assert_close(seen[1], 2 * seen[0])


def test_uses_that_a_pass_does_not_have(layer):
    z = layer(X).sum()  # recorded, alive, never passed
    _check(layer, lambda m, w: m(m(X).sin()).sum())
    _check(layer, lambda m, w: m(X).sum())
    del z
    _check(layer, lambda m, w: m(X).sum())


def test_a_parameter_that_autograd_adds_to_as_well(layer):
    """Tied to a use that is no such operator: its gradient counts, wherever it comes."""
    _check(layer, lambda m, w: (m(X).sin() * w).sum())
    _check(layer, lambda m, w: m((X * w).sin()).sum())
    _check(layer, lambda m, w: m(X + w).sum() + (w * w).sum())


def test_outside_of_a_pass(layer):
    class Ctx:
        saved_tensors = (X, layer.w.detach())
        rest = (layer.w, False)

    layer.flat.zero_grad()
    _Scale.backward(Ctx, torch.ones(3, 5))
    assert len(layer.seen) == 1


def test_gradients_that_a_pass_is_not_asked_for(layer):
    """torch.autograd.grad leaves the flat buffer alone and hands out what it names."""
    def f(m, w):
        return m(m(X).sin()).sum()

    want = _want(f, layer.w)
    layer.flat.zero_grad()
    x = X.clone().requires_grad_(True)
    z = layer(layer(x).sin()).sum()
    torch.autograd.grad(z, x, retain_graph=True)
    z.backward(inputs=[x], retain_graph=True)
    assert not layer.flat.grad.any() and not layer.seen
    got, = torch.autograd.grad(z, layer.w, retain_graph=True)
    torch.testing.assert_close(got, want)
    assert not layer.flat.grad.any() and not layer.seen
    z.backward(inputs=[layer.w])
    torch.testing.assert_close(layer.w.grad, want)
    assert len(layer.seen) == 1


class _Fail(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return x.clone()

    @staticmethod
    def backward(ctx, g):
        raise ArithmeticError("on purpose")


def test_a_pass_that_fails_leaves_nothing_behind(layer):
    x = X.clone().requires_grad_(True)
    for _ in range(2):
        with pytest.raises(ArithmeticError):
            layer(_Fail.apply(x)).sum().backward()
    layer.flat.zero_grad()
    _check(layer, lambda m, w: m(X).sum())
    assert not _rows._PASSES and not _rows._FAILED


def test_captured_passes_are_not_waited_for(monkeypatch):
    """Another thread's eager pass beside one that is captured, and the reverse."""
    device = torch.device("cuda", 0)
    state = {"capturing": False}
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    eager = _rows._PASSES[-10] = _rows._Pass(device)
    eager.writers[1] = (device, 17)
    state["capturing"] = True
    captured = _rows._PASSES[-11] = _rows._Pass(device)
    captured.writers[1] = (device, 18)
    assert not captured.left and not _rows._unjoined(device)
    state["capturing"] = False
    assert _rows._unjoined(device) == {(device, 17)}
    assert not _rows._unjoined(torch.device("cuda", 1))
    del captured
    assert not _rows._FAILED
    del eager  # failed
    assert _rows._FAILED == {(device, 17)} and not _rows._PASSES
    _rows._FAILED.clear()


@pytest.fixture
def bucketer(layer, tmp_path):
    from zookeeper_amd.parallel.ddp import GradBucketer

    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    b = GradBucketer(layer.flat, world=1, force=True)
    try:
        yield b
    finally:
        b.remove()
        dist.destroy_process_group()


def _spy(bucketer):
    """What each all-reduce is given."""
    given = []
    issue = bucketer._issue

    def spy(view):
        given.append(view.clone())
        return issue(view)

    bucketer._issue = spy
    return given


def test_the_bucketer_gets_complete_gradients(layer, bucketer):
    given = _spy(bucketer)

    def f(m, w):
        return m(m(X).sin()).sum()

    z = f(layer, layer.w)
    for n in (1, 2):  # two steps over one graph
        layer.flat.zero_grad()
        z.backward(retain_graph=True)
        assert len(given) == n  # within the pass
        torch.testing.assert_close(given[-1][:5], _want(f, layer.w))
        bucketer.finish()
        assert len(given) == n


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointed_segments_of_a_shared_layer(layer, bucketer, reentrant):
    given = _spy(bucketer)

    def f(m, w):
        h = X.clone().requires_grad_(True)
        for _ in range(3):
            h = checkpoint(lambda v: m(v).sin(), h, use_reentrant=reentrant)
        return h.sum()

    for n in (1, 2):
        layer.flat.zero_grad()
        f(layer, layer.w).backward()
        bucketer.finish()
        assert len(given) == n
        want = _want(lambda m, w: m(m(m(X).sin()).sin()).sin().sum(), layer.w)
        torch.testing.assert_close(given[-1][:5], want)


def test_a_write_behind_the_all_reduce_is_refused(layer, bucketer):
    """Outside of a reentrant checkpoint first and then inside, which nothing foretells."""
    h = checkpoint(layer, X.clone().requires_grad_(True), use_reentrant=True)
    with pytest.raises(RuntimeError, match="all-reduce"):
        layer(h.sin()).sum().backward()
    bucketer.finish()
    layer.flat.zero_grad()
    layer(X).sum().backward()  # the next step is as usual
    bucketer.finish()


def test_a_bucketer_that_is_gone(layer, bucketer):
    bucketer.remove()
    layer.flat.zero_grad()
    layer(X).sum().backward()
    torch.testing.assert_close(layer.w.grad, _want(lambda m, w: m(X).sum(), layer.w))
