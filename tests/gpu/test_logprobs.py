"""Log probability kernels against the definition in 64 bits.

Tolerances, in units of ``u = 2^-24``.  A thread adds at most ``V / 256 + 32``
terms one after the other and a handful of joins follow, so the positive sums
s and -q are right to ``n u`` with ``n = V / 256 + 64``; a term e^d adds
``(1.5 |d| + 4) u`` of itself (d is rounded, scaled to base 2 and rounded
again), on average ``1.5 E|d| + 4`` under the distribution.  ln s, x_t - m and
the two subtractions are rounded once each.  16-bit gradients add half a unit
of their type."""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from zookeeper_amd import ops

    assert ops.available(), ops.load_error()


def _reference(x, tokens):
    x = x.double()
    gone = torch.isneginf(x).all(-1, keepdim=True)
    lp = torch.log_softmax(x, -1).masked_fill(gone, float("-inf"))
    p = lp.exp()
    ent = torch.special.entr(p).sum(-1)
    m = x.amax(-1, keepdim=True)
    d = torch.where(p > 0, m - x, torch.zeros_like(x))
    mean_d = (p * d).sum(-1)
    return lp, p, ent, mean_d


def _check(x, tokens, top, r, grad=None, g=None):
    V = x.shape[-1]
    lp, p, ent, mean_d = _reference(x, tokens)
    n = V / 256 + 64 + 1.5 * mean_d + 4  # relative error of s and q, in u
    some = ~torch.isneginf(x.double()).all(-1)
    rlp = lp.gather(-1, tokens.unsqueeze(-1))[..., 0]
    fin = torch.isfinite(rlp)
    ln_s = (ent - mean_d).abs() + mean_d  # |ln s| at most
    tol = U * (n + 4 * ln_s + 4 * rlp.abs())
    assert torch.equal(torch.isneginf(r.logp), ~fin)
    assert ((r.logp.double() - rlp)[fin].abs() <= tol[fin]).all(), (
        ((r.logp.double() - rlp).abs() / tol)[fin].max())
    tol = U * (n * (1 + 2 * mean_d) + 8 * (ln_s + mean_d))
    assert ((r.entropy.double() - ent)[some].abs() <= tol[some]).all(), (
        ((r.entropy.double() - ent).abs() / tol)[some].max())
    assert (r.entropy[~some] == 0).all()
    if top:
        ids = x.double().sort(stable=True, dim=-1, descending=True).indices[..., :top]
        assert torch.equal(r.top_ids, ids)
        rt = lp.gather(-1, ids)
        fin = torch.isfinite(rt)
        tol = (U * (n + 4 * ln_s)).unsqueeze(-1) + 4 * U * rt.abs()
        assert torch.equal(torch.isneginf(r.top_logp), ~fin)
        assert ((r.top_logp.double() - rt)[fin].abs() <= tol[fin]).all()
    if grad is not None:
        gl, gh = (t.double().unsqueeze(-1) for t in g)
        lps = torch.where(p > 0, lp, torch.zeros_like(lp))
        h = ent.unsqueeze(-1)
        soft = -p * (gl + gh * (lps + h))
        hot = torch.zeros_like(lp).scatter_(-1, tokens.unsqueeze(-1), 1.0)
        want = soft + gl * hot
        want[~some] = 0
        mag = p * (gl.abs() + gh.abs() * (lps.abs() + h))
        dt = grad.dtype
        rel = n.unsqueeze(-1) * 3 + 4 * ln_s.unsqueeze(-1) + 4 * lps.abs() + 16
        tol = U * (mag * rel + 4 * (gl * hot).abs()) + torch.finfo(dt).eps / 2 * want.abs()
        # gradients under the normal range: half a step of the subnormals
        tol = tol + torch.finfo(dt).tiny * torch.finfo(dt).eps / 2 + 2.0 ** -126
        assert ((grad.double() - want).abs() <= tol).all(), (
            (grad.double() - want).abs() - tol).max()


def _inputs(rows, V, dt, seed, scale=3.0):
    torch.manual_seed(seed)
    x = (torch.randn(rows, V, device="cuda") * scale).to(dt)
    return x, torch.randint(0, V, (rows,), device="cuda")


SHAPES = [(1, 1, 1), (1, 2, 2), (3, 7, 0), (5, 64, 64), (1536, 10, 5), (37, 1000, 5),
          (9, 2047, 20), (6, 2048, 1), (4, 2049, 64), (1, 4097, 3), (3, 50001, 20),
          (1, 129000, 20), (2, 131072, 64), (1100, 5000, 7), (300, 2050, 33), (1, 200000, 0)]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,V,top", SHAPES)
def test_values_alternatives_and_gradient(rows, V, top, dt):
    from zookeeper_amd.ops import token_logprobs

    x, t = _inputs(rows, V, dt, rows + V)
    x.requires_grad_(True)
    r = token_logprobs(x, t, top=top)
    assert r.logp.dtype == r.entropy.dtype == torch.float32
    g = (torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda"))
    dx, = torch.autograd.grad([r.logp, r.entropy], [x], list(g))
    assert dx.dtype == dt and dx.shape == x.shape
    _check(x.detach(), t, top, r, dx, g)
    q = token_logprobs(x.detach(), t, top=top)
    for a, b in zip(q, r):
        assert (a is None and b is None) or torch.equal(a, b)


@pytest.mark.parametrize("V,top", [(100, 10), (2048, 64), (9000, 64), (70000, 20)])
@pytest.mark.parametrize("kind", ["constant", "rising", "falling", "two values", "blocks",
                                  "minus zero"])
def test_alternatives_of_unkind_rows(V, top, kind):
    from zookeeper_amd.ops import token_logprobs

    i = torch.arange(V, device="cuda", dtype=torch.float32)
    x = {"constant": torch.full_like(i, -2.5), "rising": i / V * 20, "falling": -i / V * 20,
         "two values": (i % 2), "blocks": (i // 512 % 7) - 3.0,
         "minus zero": torch.where(i % 2 == 0, -0.0, 0.0)}[kind]
    x = torch.stack([x, x.flip(0), x.roll(V // 3)])
    t = torch.tensor([0, V - 1, V // 2], device="cuda")
    for dt in (torch.float32, torch.bfloat16):
        _check(x.to(dt), t, top, token_logprobs(x.to(dt), t, top=top))


@pytest.mark.parametrize("V", [30, 1000, 3000, 66000])
def test_masks(V):
    from zookeeper_amd.ops import token_logprobs

    x, t = _inputs(8, V, torch.float32, V)
    lowest = torch.finfo(torch.float32).min
    x[0] = float("-inf")                      # nothing left
    x[1, 1:] = float("-inf")                  # one left
    t[1] = 0
    x[2, ::2] = float("-inf")
    t[2] = 0                                  # the given token is masked
    x[3, :V // 2] = lowest                    # masked with the lowest value
    x[4] = lowest                             # ... everywhere: a uniform row
    x[5, :-1] = float("-inf")                 # the last one left
    t[5] = V - 1
    x.requires_grad_(True)
    top = min(V, 64)
    r = token_logprobs(x, t, top=top)
    g = (torch.rand(8, device="cuda"), torch.rand(8, device="cuda"))
    dx, = torch.autograd.grad([r.logp, r.entropy], [x], list(g))
    _check(x.detach(), t, top, r, dx, g)
    assert r.logp[1] == 0 and r.entropy[1] == 0 and torch.isneginf(r.logp[2])
    assert (dx[0] == 0).all()


def test_ignored_and_out_of_range_tokens():
    from zookeeper_amd.ops import token_logprobs

    for V in (50, 5000):
        x, t = _inputs(6, V, torch.float32, 1)
        t[1], t[2], t[3], t[4] = -100, -1, V, 7
        x.requires_grad_(True)
        r = token_logprobs(x, t)
        assert r.logp[1] == 0 and r.logp[2].isnan() and r.logp[3].isnan()
        dx, = torch.autograd.grad(r.logp.sum(), x)
        assert (dx[1] == 0).all() and dx[2].isnan().all() and dx[3].isnan().all()
        assert dx[0].isfinite().all()
        r = token_logprobs(x, t, ignore_index=7)  # inside the vocabulary
        assert r.logp[4] == 0 and r.logp[1].isnan()
        dx, = torch.autograd.grad(r.logp[4:].sum(), x)
        assert (dx[4] == 0).all() and dx[5].abs().sum() > 0


def test_nan_and_infinity():
    from zookeeper_amd.ops import token_logprobs

    for V in (40, 3000, 70000):
        x, t = _inputs(5, V, torch.float32, 2)
        x[1, V // 2] = float("nan")
        x[2, 3] = float("inf")
        x[3] = float("nan")
        x[4, 1:] = float("-inf")
        x[4, 0] = -float("nan")
        r = token_logprobs(x, t, top=5)
        assert r.logp[1:].isnan().all() and r.entropy[1:].isnan().all()
        assert r.logp[0].isfinite()
        assert r.top_ids[1, 0] == V // 2 and r.top_ids[2, 0] == 3
        assert torch.equal(r.top_ids[3], torch.arange(5, device="cuda"))
        assert torch.equal(r.top_ids[4], torch.arange(5, device="cuda"))


def test_large_offsets_of_the_logits():
    """Adding 10000 to a row changes nothing beyond the rounding of the sum."""
    from zookeeper_amd.ops import token_logprobs

    x, t = _inputs(4, 3000, torch.float32, 3)
    x = (x * 8).round() / 8  # exact after the shift
    a, b = token_logprobs(x, t), token_logprobs(x + 8192.0, t)
    assert torch.equal(a.logp, b.logp) and torch.equal(a.entropy, b.entropy)


@pytest.mark.parametrize("V", [33, 2500, 90000])
def test_strides_and_leading_dims(V):
    from zookeeper_amd.ops import token_logprobs

    torch.manual_seed(4)
    base = torch.randn(3, 4, V + 13, device="cuda").bfloat16()
    for x in (base[..., :V], base[:, 1:3, 5:5 + V], base.transpose(0, 1)[..., :V],
              base[0, 0, :V], base[0, 0, :V].expand(6, V)):
        t = torch.randint(0, V, x.shape[:-1], device="cuda", dtype=torch.int32)
        xr = x.detach().requires_grad_(True)
        r = token_logprobs(xr, t, top=3)
        assert r.logp.shape == t.shape and r.top_ids.shape == (*t.shape, 3)
        g = (torch.randn(t.shape, device="cuda"), torch.randn(t.shape, device="cuda"))
        dx, = torch.autograd.grad([r.logp, r.entropy], [xr], list(g))
        _check(x, t.long(), 3, r, dx, g)


def test_one_gradient_at_a_time_and_none():
    from zookeeper_amd.ops import token_logprobs

    x, t = _inputs(5, 700, torch.float32, 5)
    x.requires_grad_(True)
    z = torch.zeros(5, device="cuda")
    o = torch.ones(5, device="cuda")
    for pick, g in ((0, (o, z)), (1, (z, o))):
        r = token_logprobs(x, t)
        dx, = torch.autograd.grad(r[pick].sum(), x)
        _check(x.detach(), t, 0, r, dx, g)
    r = token_logprobs(x, t, top=4)
    assert not r.top_logp.requires_grad
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(token_logprobs(x, t).logp.sum(), x, create_graph=True)


def test_no_rows():
    from zookeeper_amd.ops import token_logprobs

    x = torch.randn(0, 30, device="cuda", requires_grad=True)
    r = token_logprobs(x, torch.zeros(0, dtype=torch.int64, device="cuda"), top=2)
    assert r.logp.shape == (0,) and r.top_ids.shape == (0, 2)
    assert torch.autograd.grad(r.logp.sum(), x)[0].shape == (0, 30)


def test_gradient_matches_differences():
    from zookeeper_amd.ops import token_logprobs

    x, t = _inputs(3, 50, torch.float32, 6, scale=1.0)
    x.requires_grad_(True)

    def f(v):
        r = token_logprobs(v, t)
        return (r.logp.double() * 2 + r.entropy.double()).sum()

    g, = torch.autograd.grad(f(x), x)
    d = torch.randn_like(x)
    h = 2.0 ** -6
    got = float((f((x + h * d).detach()) - f((x - h * d).detach())) / (2 * h))
    # three rows of values under 10 with errors of ~100 u, and h^2 / 6 of a third
    # derivative of order |d|^3 ~ 30 a row
    assert abs(got - float((g.double() * d).sum())) <= 3 * 3 * 10 * 100 * U / h + h * h / 6 * 600


def test_agrees_with_the_training_loss():
    from zookeeper_amd.ops import softmax_xent, token_logprobs

    x, t = _inputs(256, 1000, torch.float32, 7)
    loss, hits = softmax_xent(x, t)
    r = token_logprobs(x, t, top=1)
    assert abs(float(loss) + float(r.logp.double().mean())) < 1e-4
    assert int(hits) == int((r.top_ids[:, 0] == t).sum())


def test_replays_in_a_graph():
    from zookeeper_amd.ops import token_logprobs

    x, t = _inputs(3, 70000, torch.bfloat16, 8)

    def step(v):
        v = v.detach().requires_grad_(True)
        r = token_logprobs(v, t, top=8)
        return [*(o.detach() for o in r), *torch.autograd.grad(r.logp.sum() + r.entropy.sum(), v)]

    static = x.clone()
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
        new = _inputs(3, 70000, torch.bfloat16, 20 + k)[0]
        static.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(out, step(new)):
            assert torch.equal(a, e), k


def test_the_longest_rows():
    """The last split of a row of almost 2^31 logits ends past 2^31 - 1 when rounded up."""
    from zookeeper_amd.ops import token_logprobs

    V = 0x7FFF0000 - 1
    x = torch.zeros(1, V, device="cuda", dtype=torch.bfloat16)
    x[0, V - 1], x[0, V - 2], x[0, 5] = 25.0, 24.0, 23.0
    r = token_logprobs(x, torch.tensor([V - 1], device="cuda"), top=4)
    assert r.top_ids.tolist() == [[V - 1, V - 2, 5, 0]]
    d = torch.tensor([0.0, -1.0, -2.0, -25.0], dtype=torch.float64)
    n = torch.tensor([1.0, 1.0, 1.0, V - 3], dtype=torch.float64)
    z = (n * d.exp()).sum()
    lp = d - z.log()
    # a thread adds V / (64 * 256) zeros' terms one after the other, each sum rounded; they
    # are `share` of z.  The few other terms and joins: 200 u as above
    share = float(n[3] * d[3].exp() / z)
    tol = V / (64 * 256) * U * share + 200 * U
    assert abs(float(r.logp[0]) - float(lp[0])) <= tol
    assert ((r.top_logp[0].double().cpu() - lp).abs() <= tol + 4 * U * lp.abs()).all()


@pytest.mark.parametrize("V", [50, 5000])
def test_the_entropy_does_not_depend_on_the_token(V):
    """... nor does its gradient, on the host either."""
    from zookeeper_amd.ops import token_logprobs

    x, t = _inputs(6, V, torch.float32, 1)
    x.requires_grad_(True)
    want, = torch.autograd.grad(token_logprobs(x, t).entropy.sum(), x)
    t[1], t[2], t[3] = -100, -1, V
    r = token_logprobs(x, t)
    assert r.logp[2:4].isnan().all()
    assert torch.equal(torch.autograd.grad(r.entropy.sum(), x)[0], want)
    host = x.detach().cpu().requires_grad_(True)
    dx, = torch.autograd.grad(token_logprobs(host, t.cpu()).entropy.sum(), host)
    assert torch.isfinite(dx).all()
    # with the log probability's too, the NaN is in its own rows only
    r = token_logprobs(x, t)
    dx, = torch.autograd.grad((r.logp + r.entropy).sum(), x)
    assert dx[2:4].isnan().all() and torch.isfinite(dx[[0, 1, 4, 5]]).all()
