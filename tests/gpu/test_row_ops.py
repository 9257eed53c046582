"""The row operators (layer norm, log probabilities, 8-bit kept activations) as a
program uses them: rows farther apart than 32-bit offsets reach, two streams and
two threads at a time, a model under the trainer with and without graph replay."""

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from zookeeper_amd import ops

    assert ops.available(), ops.load_error()


def test_rows_far_apart():
    """Row starts past 2^31 elements."""
    from zookeeper_amd import ops

    torch.manual_seed(0)
    step = (1 << 30) + 40
    base = torch.empty(2 * step + 5000, dtype=torch.bfloat16, device="cuda")
    far = torch.as_strided(base, (3, 5000), (step, 1))
    near = torch.randn(3, 5000, device="cuda").bfloat16()
    far.copy_(near)
    t = torch.randint(0, 5000, (3,), device="cuda")
    dy = torch.randn(3, 5000, device="cuda").bfloat16()

    def run(v):
        v = v.detach().requires_grad_(True)
        y = ops.layer_norm(v)
        out = [y, torch.autograd.grad(y, v, dy)[0]]
        r = ops.token_logprobs(v, t, top=7)
        out += [*r, torch.autograd.grad(r.logp.sum() + r.entropy.sum(), v)[0]]
        y = ops.gelu8(v)
        out += [y, torch.autograd.grad(y, v, dy)[0], ops.unpack8(ops.pack8(v.detach()))]
        # ... as the incoming gradient
        n = near.detach().requires_grad_(True)
        g = torch.as_strided(v.detach(), v.shape, v.stride())
        out += [torch.autograd.grad(ops.layer_norm(n), n, g)[0],
                torch.autograd.grad(ops.gelu8(n), n, g)[0],
                *ops.dense8_grads(g, ops.pack8(dy))]
        return out

    for a, b in zip(run(far), run(near)):
        assert torch.equal(a, b)


def test_more_than_2_31_elements():
    from zookeeper_amd import ops

    torch.manual_seed(1)
    rows, cols = 70000, 32768  # 2.3e9 elements
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    last = torch.randn(3, cols, device="cuda").bfloat16()
    x[-3:] = last
    w = torch.rand(cols, device="cuda")
    assert torch.equal(ops.layer_norm(x, w)[-3:], ops.layer_norm(last, w))
    t = torch.full((rows,), cols - 1, device="cuda")
    r, e = ops.token_logprobs(x, t), ops.token_logprobs(last, t[:3])
    # few rows are split, so the sums differ in their order: at most 32768 / 256 + 64
    # roundings of s on either side, 2.3e-5
    torch.testing.assert_close(r.logp[-3:], e.logp, rtol=0, atol=3e-5)
    kept, want = ops.pack8(x), ops.pack8(last)
    assert torch.equal(kept.codes[-3:], want.codes) and torch.equal(kept.scales[-3:], want.scales)
    del kept
    assert torch.equal(ops.gelu8(x)[-3:], ops.gelu8(last))
    assert not ops.gelu8(x)[:-3].any()


def _program(x, t, w):
    from zookeeper_amd import ops

    v = x.detach().requires_grad_(True)
    wl = w.detach().requires_grad_(True)
    h = ops.layer_norm(v, wl)
    z = ops.gelu8(h)
    r = ops.token_logprobs(z, t, top=9)
    dv, dw = torch.autograd.grad((r.logp - 0.1 * r.entropy).sum(), [v, wl])
    return [r.logp.detach(), r.entropy.detach(), r.top_ids, dv, dw,
            *ops.dense8_grads(dv, ops.pack8(z.detach()))]


def _case(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(700, 2500, device="cuda", generator=g)
    return (x, torch.randint(0, 2500, (700,), device="cuda", generator=g),
            torch.rand(2500, device="cuda", generator=g))


def test_two_streams_at_a_time():
    cases = [_case(s) for s in range(4)]
    want = [_program(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = [None] * 4
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = _program(*cases[i])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_two_threads_at_a_time():
    cases = [_case(s) for s in range(3)]
    want = [_program(*c) for c in cases]
    torch.cuda.synchronize()
    got, bad = [None] * 3, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(4):
                    got[i] = _program(*cases[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            bad.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not bad, bad
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def _trainer(graph):
    from zookeeper_amd import nn as znn
    from zookeeper_amd.core import configure
    from zookeeper_amd.ops import token_logprobs
    from zookeeper_amd.train import SGD, Trainer

    torch.manual_seed(3)
    model = torch.nn.Sequential(
        znn.LayerNorm(48), znn.QuantDense(48, 96, use_bias=True, kept="int8"),
        znn.GELU(kept="int8"), znn.QuantDense(96, 10, use_bias=True, kept="int8"))

    def loss(logits, labels):
        r = token_logprobs(logits, labels, top=1)
        return -(r.logp + 0.01 * r.entropy).mean(), (r.top_ids[:, 0] == labels).sum()

    spec = SGD()
    configure(spec, {"learning_rate": 0.1, "momentum": 0.9})
    return Trainer(model, loss, spec, graph=graph, graph_warmup=2)


def test_a_model_under_the_trainer():
    """Gradients go straight into the flat buffer; graph replays follow the eager
    steps bit for bit."""
    eager, graph = _trainer(False), _trainer(True)
    g = torch.Generator(device="cuda").manual_seed(4)
    losses = []
    for step in range(7):
        x = torch.randn(300, 48, device="cuda", generator=g)
        y = torch.randint(0, 10, (300,), device="cuda", generator=g)
        a, hits = eager.train_step(x, y)
        b, ghits = graph.train_step(x, y)
        torch.cuda.synchronize()
        assert float(a) == float(b) and int(hits) == int(ghits), step
        assert torch.equal(eager.flat.grad, graph.flat.grad), step
        assert torch.equal(eager.flat.data, graph.flat.data), step
        losses.append(float(a))
    assert graph._graph is not None
    assert eager.flat.grad.abs().sum() > 0 and len(set(losses)) == 7


def test_saved_tensors_may_change_their_layout():
    """Hooks that keep saved tensors elsewhere give padded rows back contiguous."""
    from zookeeper_amd import ops

    torch.manual_seed(5)
    wide = torch.randn(50, 3000, device="cuda")
    x = wide[:, 7:907].detach().requires_grad_(True)
    w = torch.rand(900, device="cuda", requires_grad=True)
    t = torch.randint(0, 900, (50,), device="cuda")

    def run():
        r = ops.token_logprobs(x, t)
        h = ops.gelu8(ops.dense8(ops.layer_norm(x, w), torch.eye(900, device="cuda")))
        return torch.autograd.grad(r.logp.sum() + r.entropy.sum() + h.sum(), [x, w])

    want = run()
    with torch.autograd.graph.save_on_cpu():
        got = run()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


class _Delay(torch.autograd.Function):
    """Identity whose backward keeps the stream it runs on busy for a moment."""

    @staticmethod
    def forward(ctx, x):
        return x.view_as(x)

    @staticmethod
    def backward(ctx, g):
        torch.cuda._sleep(20_000_000)
        return g


def _shared_model():
    from zookeeper_amd import nn as znn
    from zookeeper_amd.parallel.flat import FlatParams

    torch.manual_seed(6)
    model = torch.nn.Sequential(znn.LayerNorm(64),
                                znn.QuantDense(64, 64, use_bias=True, kept="int8")).cuda()
    return model, FlatParams(model)


@pytest.mark.parametrize("streams", [1, 2])
def test_layers_applied_twice_with_flat_gradients(streams):
    """Two branches through the same layers, each on its own stream: their writes
    into the flat gradients do not overlap, the caller's stream waits for them,
    and each parameter is reported ready once, with both contributions."""
    model, flat = _shared_model()
    xs = [torch.randn(256, 64, device="cuda") for _ in range(2)]
    flat.zero_grad()
    (model(xs[0]).square().sum() + model(xs[1]).square().sum()).backward()
    torch.cuda.synchronize()
    want = flat.grad.clone()
    single = []
    for x in xs:
        flat.zero_grad()
        model(x).square().sum().backward()
        torch.cuda.synchronize()
        single.append(flat.grad.clone())
    # each pass's sums are the same bits, and one addition joins them
    assert torch.equal(want, single[0] + single[1])

    seen = {}
    for slot in flat.slots:
        def ready(slot=slot):
            assert slot.name not in seen
            seen[slot.name] = slot.param.grad.clone()
        slot.param._zk_grad_ready = ready
    main = torch.cuda.current_stream()
    side = [main] + [torch.cuda.Stream() for _ in range(streams - 1)]
    for _ in range(3):
        flat.zero_grad()
        seen.clear()
        sums = []
        for i, x in enumerate(xs):
            s = side[i % streams]
            s.wait_stream(main)
            with torch.cuda.stream(s):
                sums.append(_Delay.apply(model(x).square()).sum())
        for s in side[1:]:
            main.wait_stream(s)
        (sums[0] + sums[1]).backward()
        got = flat.grad.clone()  # on the caller's stream, with no other wait
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        assert sorted(seen) == sorted(s.name for s in flat.slots)
        for slot in flat.slots:
            assert torch.equal(seen[slot.name], slot.param.grad)


def test_a_dropped_graph_does_not_hold_back_a_parameter():
    model, flat = _shared_model()
    count = []
    for slot in flat.slots:
        slot.param._zk_grad_ready = lambda name=slot.name: count.append(name)
    x = torch.randn(8, 64, device="cuda")
    model(x)  # recorded and dropped
    model(x).sum().backward()
    assert sorted(count) == sorted(s.name for s in flat.slots)
    y = model(x).sum()
    y.backward(retain_graph=True)
    y.backward()
    assert len(count) == 3 * len(flat.slots)


def _operators():
    from zookeeper_amd import ops

    t = torch.randint(0, 100, (40,), generator=torch.Generator().manual_seed(1)).cuda()
    w = torch.rand(100, device="cuda")
    return [lambda v: ops.layer_norm(v, w), ops.gelu8,
            lambda v: ops.token_logprobs(v, t, top=3)[:3], lambda v: ops.dense8(v, w[None])]


@pytest.mark.parametrize("recorded", [False, True])
def test_traced_calls_are_run_again(recorded):
    """A trace without gradients holds the operators and not their empty outputs."""
    torch.manual_seed(8)
    x = torch.randn(40, 100, device="cuda", requires_grad=recorded)
    for f in _operators():
        traced = torch.jit.trace(f, (x,), check_trace=False)
        for _ in range(2):
            z = torch.randn(40, 100, device="cuda")
            got, want = traced(z), f(z)
            if isinstance(got, torch.Tensor):
                got, want = (got,), (want,)
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_forms_are_not_traced():
    from zookeeper_amd import ops

    x = torch.randn(8, 64, device="cuda")
    kept = ops.pack8(x)
    for f in (lambda v: ops.pack8(v).codes, lambda v: v + ops.unpack8(kept),
              lambda v: ops.dense8_grads(v, kept)[0]):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(f, (x,), check_trace=False)


def test_forward_mode_is_refused():
    from torch.autograd import forward_ad

    x = torch.randn(40, 100, device="cuda")
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for f in _operators()[:3]:  # dense8 without a recorded weight is torch's product
            with pytest.raises(NotImplementedError, match="jvp"):
                f(dual)
            with pytest.raises(NotImplementedError, match="jvp"), torch.no_grad():
                f(dual)
            f(x)  # no tangent: as always


def test_a_module_is_saved_whole_after_data_parallel_steps(tmp_path):
    model, flat = _shared_model()
    for slot in flat.slots:
        slot.param._zk_grad_ready = _nothing
    x = torch.randn(8, 64, device="cuda")
    z = model(model(x)).sum()
    z.backward()
    for slot in flat.slots:  # as the bucketer does at its end
        del slot.param._zk_grad_ready
    torch.save(model, tmp_path / "model.pt")
    again = torch.load(tmp_path / "model.pt", weights_only=False)
    assert torch.equal(again(again(x)).sum(), z)


def _nothing():
    pass


def test_a_graph_passed_twice_reports_complete_gradients():
    """The same layers twice in one graph, and two passes over it."""
    model, flat = _shared_model()
    x = torch.randn(16, 64, device="cuda")
    z = model(model(x)).square().sum()
    flat.zero_grad()
    z.backward(retain_graph=True)
    torch.cuda.synchronize()
    want = flat.grad.clone()
    seen = []
    for slot in flat.slots:
        slot.param._zk_grad_ready = lambda slot=slot: seen.append((slot,
                                                                   slot.param.grad.clone()))
    for _ in range(2):
        flat.zero_grad()
        seen.clear()
        z.backward(retain_graph=True)
        torch.cuda.synchronize()
        assert torch.equal(flat.grad, want)
        assert sorted(s.name for s, _ in seen) == sorted(s.name for s in flat.slots)
        assert all(torch.equal(g, s.param.grad) for s, g in seen)


def test_gradients_that_a_pass_is_not_asked_for():
    """torch.autograd.grad leaves flat gradients alone and hands out what it names."""
    model, flat = _shared_model()
    params = list(model.parameters())
    x = torch.randn(16, 64, device="cuda", requires_grad=True)
    flat.zero_grad()
    z = model(x).square().sum()
    z.backward(retain_graph=True)
    torch.cuda.synchronize()
    want = [p.grad.clone() for p in params]
    dx = x.grad.clone()
    flat.zero_grad()
    assert torch.equal(torch.autograd.grad(z, x, retain_graph=True)[0], dx)
    z.backward(inputs=[x], retain_graph=True)
    got = torch.autograd.grad(z, params, retain_graph=True)
    torch.cuda.synchronize()
    assert not flat.grad.any()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # one at a time; the dense bias alone has sums of its own, 16 terms each way
    tol = 2 * 16 * 2.0 ** -24 * (2 * model(x).detach()).abs().sum(0)
    for p, a in zip(params, want):
        tol_p = tol if p is params[-1] else torch.zeros_like(a)
        assert ((torch.autograd.grad(z, p, retain_graph=True)[0] - a).abs() <= tol_p).all()
        flat.zero_grad()
        z.backward(inputs=[p], retain_graph=True)
        torch.cuda.synchronize()
        assert ((p.grad - a).abs() <= tol_p).all()
        assert all(q is p or not q.grad.any() for q in params)


class _Fail(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return x.view_as(x)

    @staticmethod
    def backward(ctx, g):
        raise ArithmeticError("on purpose")


def test_clearing_waits_for_a_failed_pass():
    """A pass on a side stream fails behind its writes; zero_grad on the caller's stream
    comes after them all the same."""
    model, flat = _shared_model()
    x = torch.randn(256, 64, device="cuda", requires_grad=True)
    main, side = torch.cuda.current_stream(), torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(main)
        with torch.cuda.stream(side):
            z = _Delay.apply(model(_Fail.apply(x)).square()).sum()
        main.wait_stream(side)
        with pytest.raises(ArithmeticError):
            z.backward()
        flat.zero_grad()
        got = flat.grad.clone()
        torch.cuda.synchronize()
        assert not got.any() and not flat.grad.any()
    model(x).sum().backward()
    torch.cuda.synchronize()
    assert flat.grad.any()


def test_a_bucket_waits_for_every_stream_that_wrote_it(tmp_path):
    """Two layers in one bucket, their backwards on two streams: the slow one's gradients
    are reported first."""
    import torch.distributed as dist

    from zookeeper_amd import nn as znn
    from zookeeper_amd.parallel.ddp import GradBucketer
    from zookeeper_amd.parallel.flat import FlatParams

    torch.manual_seed(11)
    model = torch.nn.ModuleList([znn.LayerNorm(64), znn.LayerNorm(64)]).cuda()
    flat = FlatParams(model)
    x = torch.randn(256, 64, device="cuda")
    main, side = torch.cuda.current_stream(), torch.cuda.Stream()

    def step():
        flat.zero_grad()
        fast = model[0](x).square().sum()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            slow = _Delay.apply(model[1](x).square()).sum()
        main.wait_stream(side)
        (fast + slow).backward()

    step()
    torch.cuda.synchronize()
    want = flat.grad.clone()
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    bucketer = GradBucketer(flat, world=1, force=True)
    try:
        assert bucketer.num_buckets == 1
        for _ in range(3):
            step()
            bucketer.finish()
            torch.cuda.synchronize()
            assert torch.equal(flat.grad, want)
    finally:
        bucketer.remove()
        dist.destroy_process_group()


@pytest.mark.parametrize("device", ["cuda", "cpu"])
def test_saved_tensors_may_come_back_with_gaps(device):
    from zookeeper_amd import ops

    torch.manual_seed(12)
    x = torch.randn(40, 100, device=device, requires_grad=True)
    w = torch.randn(30, 100, device=device, requires_grad=True)
    b = torch.randn(30, device=device, requires_grad=True)
    t = torch.randint(0, 100, (40,), device=device)

    def run():
        z = ops.dense8(x, w, b).square().sum()
        r = ops.token_logprobs(ops.gelu8(ops.layer_norm(x)), t)
        return (torch.autograd.grad(z, [w, b])
                + torch.autograd.grad((r.logp + r.entropy).sum(), [x]))

    def gaps(v):
        return torch.stack([v, torch.ones_like(v)], -1)[..., 0]

    want = run()
    with torch.autograd.graph.saved_tensors_hooks(lambda v: v, gaps):
        got = run()
    for p, q in zip(got, want):  # the host's reductions may round otherwise by layout
        assert torch.equal(p, q) if device == "cuda" else torch.allclose(p, q, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("segments", [None, False, True])
def test_steps_under_the_bucketer(tmp_path, segments):
    """Plain and checkpointed (not reentrant, reentrant) layers, one of them shared: the
    reduced gradients of several steps are those without data parallelism."""
    import torch.distributed as dist
    from torch.utils.checkpoint import checkpoint

    from zookeeper_amd import nn as znn
    from zookeeper_amd.parallel.ddp import GradBucketer
    from zookeeper_amd.parallel.flat import FlatParams

    torch.manual_seed(13)
    layer = torch.nn.Sequential(znn.LayerNorm(64), znn.GELU(kept="int8"),
                                znn.QuantDense(64, 64, use_bias=True, kept="int8"))
    head = znn.QuantDense(64, 10, use_bias=True, kept="int8")
    flat = FlatParams(torch.nn.ModuleList([layer, head]).cuda())
    batches = [torch.randn(200, 64, device="cuda") for _ in range(3)]

    def step(x, bucketer=None):
        flat.zero_grad()
        h = x.clone().requires_grad_(True)
        for _ in range(3):
            h = h + (layer(h) if segments is None else checkpoint(layer, h, use_reentrant=segments))
        head(h).square().sum().backward()
        if bucketer is not None:
            bucketer.finish()
        torch.cuda.synchronize()
        return flat.grad.clone()

    want = [step(x) for x in batches]
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    bucketer = GradBucketer(flat, world=1, force=True, bucket_mb=0.001, first_bucket_mb=0.001)
    try:
        assert bucketer.num_buckets > 1
        for x, w in zip(batches, want):
            assert torch.equal(step(x, bucketer), w)
    finally:
        bucketer.remove()
        dist.destroy_process_group()
