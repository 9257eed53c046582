"""The token-row operators, as they are timed: layer norm, log probabilities of
given tokens, GELU and dense gradients whose saved input is kept in 8 bits.

``run`` computes a case either in its plain form (elementary torch operations
in 32 bits, ``own`` false) or through ``zookeeper_amd.ops`` (``own`` true);
``exact`` gives the same results from the definitions in 64 bits.

8-bit form of a row: blocks of 32 values share one power-of-two step; with
``E = floor(log2(max |x|))`` the step is ``2^(E - 6)``, one power of two more
where the largest value would round to 128 steps, and never under ``2^-126``.
A value is held as its nearest whole number of steps (ties to even), at most
127 either way; a block with an infinity or a NaN in it is held as NaN.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-3  # the framework's normalisation layers' default


def listed():
    return [
        # --- layer norm -----------------------------------------------------
        # one token at a time through a wide model: latency
        dict(name="norm, one token", op="norm", rows=1, cols=4096, dtype="bf16", affine=2,
             train=False),
        # a training step's rows, forward and backward with the weight's gradient
        dict(name="norm, training rows", op="norm", rows=32768, cols=2048, dtype="bf16",
             affine=2, train=True),
        # odd row count, odd width, full precision
        dict(name="norm, odd width", op="norm", rows=4999, cols=1003, dtype="fp32", affine=2,
             train=True),
        # --- log probabilities ----------------------------------------------
        # sampling or scoring one position of a large vocabulary, 20 alternatives
        dict(name="logprobs, one position", op="logprobs", rows=1, cols=129000, dtype="bf16",
             top=20, pad=0, masked=False, train=False),
        # an ImageNet head at the benchmark's batch: loss, entropy and the top 5
        dict(name="logprobs, classes", op="logprobs", rows=1536, cols=1000, dtype="fp32",
             top=5, pad=0, masked=False, train=True),
        # training on a vocabulary of odd size held in padded rows
        dict(name="logprobs, padded rows", op="logprobs", rows=4095, cols=50001, dtype="bf16",
             top=0, pad=47, masked=False, train=True),
        # a long batch on a large vocabulary, loss and entropy with their gradient
        dict(name="logprobs, large", op="logprobs", rows=8192, cols=131072, dtype="bf16",
             top=0, pad=0, masked=False, train=True),
        # --- GELU, its input kept in 8 bits ---------------------------------
        # a small layer: latency of the two passes
        dict(name="gelu, small", op="gelu", rows=256, cols=1024, dtype="bf16"),
        # the hidden rows of a large multi-layer perceptron
        dict(name="gelu, large", op="gelu", rows=16384, cols=8192, dtype="bf16"),
        # a width that no vector load divides and a last block that is not full
        dict(name="gelu, odd width", op="gelu", rows=2047, cols=1111, dtype="fp16"),
        # --- weight and bias gradient of a dense layer, input kept in 8 bits --
        # a large layer's backward: the matrix product counts
        dict(name="dense, large", op="dense", rows=16384, outs=4096, cols=4096, dtype="bf16"),
        # few outputs, odd sizes: the long axis has to be split
        dict(name="dense, odd sizes", op="dense", rows=7999, outs=515, cols=1001, dtype="fp16"),
    ]


def _spread(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["norm", "logprobs", "gelu", "dense"])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    if op == "norm":
        cols = _spread(rng, 1, 16384)
        rows = _spread(rng, 1, min(32768, (1 << 25) // cols))
        return dict(op=op, rows=rows, cols=cols, dtype=dtype, affine=rng.choice([0, 1, 2, 2]),
                    train=rng.random() < 0.7)
    if op == "logprobs":
        top = rng.choice([0, 0, 1, 5, 20, 64])
        cols = _spread(rng, max(2, top), 200000)
        rows = _spread(rng, 1, min(8192, (1 << (29 if top == 0 else 25)) // cols))
        return dict(op=op, rows=rows, cols=cols, dtype=dtype, top=top,
                    pad=rng.choice([0, 0, 1, 24]), masked=rng.random() < 0.3,
                    train=rng.random() < 0.6)
    if op == "gelu":
        cols = _spread(rng, 1, 16384)
        return dict(op=op, rows=_spread(rng, 1, min(16384, (1 << 26) // cols)), cols=cols,
                    dtype=dtype)
    outs, cols = _spread(rng, 1, 8192), _spread(rng, 1, 8192)
    return dict(op=op, rows=_spread(rng, 1, min(16384, (1 << 37) // (outs * cols))), outs=outs,
                cols=cols, dtype=dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    rows, cols = case["rows"], case["cols"]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    state = dict(case)
    if case["op"] == "norm":
        # columns of unlike spread around a small offset, as residual rows have them
        x = randn(rows, cols).mul_(1 + 0.5 * randn(cols).abs()).add_(0.3 * randn(cols))
        state["x"] = x.to(dt).requires_grad_(case["train"])
        state["w"] = state["b"] = None
        if case["affine"] >= 1:
            state["w"] = (1 + 0.1 * randn(cols)).requires_grad_(case["train"])
        if case["affine"] >= 2:
            state["b"] = (0.1 * randn(cols)).requires_grad_(case["train"])
        if case["train"]:
            state["dy"] = randn(rows, cols).to(dt)
    elif case["op"] == "logprobs":
        width = cols + case["pad"]
        buf = torch.empty(rows, width, dtype=dt, device="cuda")
        for lo in range(0, rows, 1024):
            buf[lo:lo + 1024] = (2.5 * randn(min(1024, rows - lo), width)).to(dt)
        logits = buf[:, :cols]
        tokens = torch.randint(0, cols, (rows,), device="cuda", generator=g)
        if case["masked"]:
            # a sampling mask: half of the tokens are out, in the first row all
            keep = torch.rand(rows, cols, device="cuda", generator=g) < 0.5
            keep.scatter_(1, tokens[:, None], True)
            keep[0] = False
            logits.masked_fill_(~keep, float("-inf"))
        logits.scatter_add_(1, tokens[:, None], torch.full((rows, 1), 6.0, dtype=dt,
                                                           device="cuda"))
        state["logits"] = logits.requires_grad_(case["train"])
        state["tokens"] = tokens
        if case["train"]:
            state["g_logp"] = -(1 + 0.25 * randn(rows))  # per-token advantages
            state["g_entropy"] = -0.01 * (1 + 0.25 * randn(rows))  # entropy bonus
    elif case["op"] == "gelu":
        state["x"] = (1.5 * randn(rows, cols) - 0.25).to(dt).requires_grad_(True)
        state["dy"] = randn(rows, cols).to(dt)
    else:
        h = randn(rows, cols)
        state["x"] = (h * torch.sigmoid(1.7 * h)).to(dt)  # what an activation hands on
        state["dy"] = (0.1 * randn(rows, case["outs"])).to(dt)
    return state


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _PLAIN[state["op"]](state)


# --- the framework's operators ----------------------------------------------

def _own(s):
    from zookeeper_amd import ops

    op = s["op"]
    if op == "norm":
        y = ops.layer_norm(s["x"], s["w"], s["b"], _EPS)
        if not s["train"]:
            return {"y": y}
        leaves = [t for t in (s["x"], s["w"], s["b"]) if t is not None]
        return {"y": y.detach(), "grads": torch.autograd.grad(y, leaves, s["dy"])}
    if op == "logprobs":
        r = ops.token_logprobs(s["logits"], s["tokens"], top=s["top"])
        out = {"logp": r.logp.detach(), "entropy": r.entropy.detach()}
        if s["top"]:
            out["top_logp"], out["top_ids"] = r.top_logp, r.top_ids
        if s["train"]:
            out["grad"], = torch.autograd.grad([r.logp, r.entropy], [s["logits"]],
                                               [s["g_logp"], s["g_entropy"]])
        return out
    if op == "gelu":
        y = ops.gelu8(s["x"])
        return {"y": y.detach(), "grad": torch.autograd.grad(y, [s["x"]], s["dy"])[0]}
    kept = ops.pack8(s["x"])
    dw, db = ops.dense8_grads(s["dy"], kept)
    return {"dw": dw, "db": db}


# --- plain forms ------------------------------------------------------------

def _plain_norm(s):
    x = s["x"].float()
    xc = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt(xc.square().mean(1, keepdim=True) + _EPS)
    xhat = xc * rstd
    y = xhat
    if s["w"] is not None:
        y = y * s["w"]
    if s["b"] is not None:
        y = y + s["b"]
    y = y.to(s["x"].dtype)
    if not s["train"]:
        return {"y": y}
    dy = s["dy"].float()
    g = dy if s["w"] is None else dy * s["w"]
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    grads = [dx.to(s["x"].dtype)]
    if s["w"] is not None:
        grads.append((dy * xhat).sum(0))
    if s["b"] is not None:
        grads.append(dy.sum(0))
    return {"y": y, "grads": grads}


def _plain_logprobs(s):
    x = s["logits"].float()
    t = s["tokens"][:, None]
    m = x.amax(1, keepdim=True)
    # a row without a single token left: probabilities 0, log probabilities -inf
    some = m > float("-inf")
    c = torch.where(some, x - m, x)
    e = torch.exp(c)
    z = e.sum(1, keepdim=True)
    lz = torch.where(some, torch.log(z), torch.zeros_like(z))
    p = torch.where(some, e / z, torch.zeros_like(e))
    logp = c.gather(1, t) - lz
    # 0 log 0 = 0
    ent = lz - (p * torch.where(p > 0, c, torch.zeros_like(c))).sum(1, keepdim=True)
    out = {"logp": logp[:, 0], "entropy": ent[:, 0]}
    if s["top"]:
        # one whole number for value and place: larger values first, then lower places
        bits = (x + 0.0).view(torch.int32)
        order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).to(torch.int64)
        place = torch.arange(x.shape[1], device=x.device)
        key = (order << 32) | (0xFFFFFFFF - place)
        ids = 0xFFFFFFFF - (key.topk(s["top"], dim=1).values & 0xFFFFFFFF)
        out["top_ids"] = ids
        out["top_logp"] = c.gather(1, ids) - lz
    if s["train"]:
        glp, gen = s["g_logp"][:, None], s["g_entropy"][:, None]
        lp = torch.where(p > 0, c - lz, torch.zeros_like(c))
        d = -p * (glp + gen * (lp + ent))
        d.scatter_add_(1, t, torch.where(some, glp, torch.zeros_like(glp)))
        out["grad"] = d.to(s["logits"].dtype)
    return out


def _power(e):
    """2^e in 32 bits for whole e in [-126, 127]."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _plain_kept(x):
    """What the 8-bit form of ``x`` stands for, in 32 bits."""
    rows, cols = x.shape
    blocks = -(-cols // 32)
    v = torch.zeros(rows, blocks * 32, device=x.device)
    v[:, :cols] = x.float()
    v = v.view(rows, blocks, 32)
    top = v.abs().amax(2, keepdim=True)
    fine = torch.isfinite(top)
    e = torch.frexp(torch.where(fine, top, torch.ones_like(top))).exponent - 1
    e = torch.where(top == 0, torch.full_like(e, -120), e.clamp(-120, 127))
    e = e + ((top / _power(e - 6)).round() >= 128).to(e.dtype) * (e < 127).to(e.dtype)
    step = _power(e - 6)
    held = (v / step).round().clamp(-127, 127) * step
    held = torch.where(fine, held, torch.full_like(held, float("nan")))
    return held.view(rows, blocks * 32)[:, :cols]


def _plain_gelu(s):
    x = s["x"].float()
    y = 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    k = _plain_kept(s["x"])
    slope = (0.5 * (1 + torch.erf(k * math.sqrt(0.5)))
             + k * torch.exp(-0.5 * k * k) / math.sqrt(2 * math.pi))
    return {"y": y.to(s["x"].dtype), "grad": (s["dy"].float() * slope).to(s["x"].dtype)}


def _plain_dense(s):
    dy = s["dy"].float()
    return {"dw": dy.t() @ _plain_kept(s["x"]), "db": dy.sum(0)}


_PLAIN = {"norm": _plain_norm, "logprobs": _plain_logprobs, "gelu": _plain_gelu,
          "dense": _plain_dense}


# --- what a pass cannot do without -------------------------------------------

def work(case):
    e, n = _BYTES[case["dtype"]], case["rows"] * case["cols"]
    if case["op"] == "norm":
        params = 4 * case["cols"] * case["affine"]
        if not case["train"]:
            return {"bytes": 2 * n * e + params, "flops": 8 * n}
        return {"bytes": 4 * n * e + 2 * params, "flops": 22 * n}
    if case["op"] == "logprobs":
        out = case["rows"] * (16 + 12 * case["top"])
        if not case["train"]:
            return {"bytes": n * e + out, "flops": 6 * n}
        return {"bytes": 2 * n * e + out + 8 * case["rows"], "flops": 14 * n}
    if case["op"] == "gelu":
        return {"bytes": 4 * n * e, "flops": 60 * n}
    m = case["rows"] * case["outs"]
    return {"bytes": (n + m) * e + 4 * case["outs"] * (case["cols"] + 1),
            "flops": 2 * m * case["cols"]}


# --- the definitions in 64 bits ------------------------------------------------

def exact(case, seed):
    with torch.no_grad():
        return _EXACT[case["op"]](prepare(case, seed))


def _exact_norm(s):
    x = s["x"].double()
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    std = torch.sqrt(var + _EPS)
    n = (x - mean) / std
    w = torch.ones((), dtype=torch.float64, device=x.device) if s["w"] is None \
        else s["w"].double()
    b = torch.zeros((), dtype=torch.float64, device=x.device) if s["b"] is None \
        else s["b"].double()
    if not s["train"]:
        return {"y": n * w + b}
    dy = s["dy"].double()
    dn = dy * w
    cols = x.shape[1]
    # d/dx of (x - mean) / std, written out
    dx = (cols * dn - dn.sum(1, keepdim=True) - n * (dn * n).sum(1, keepdim=True)) / (cols * std)
    grads = [dx]
    if s["w"] is not None:
        grads.append(torch.einsum("rc,rc->c", dy, n))
    if s["b"] is not None:
        grads.append(dy.sum(0))
    return {"y": n * w + b, "grads": grads}


def _exact_logprobs(s):
    parts = []
    for lo in range(0, s["rows"], 512):
        x = s["logits"][lo:lo + 512].double()
        t = s["tokens"][lo:lo + 512]
        gone = torch.isneginf(x).all(1)
        lp = torch.log_softmax(x, 1)
        lp[gone] = float("-inf")
        p = lp.exp()
        h = torch.special.entr(p).sum(1)
        part = {"logp": lp[torch.arange(len(t), device=t.device), t], "entropy": h}
        if s["top"]:
            part["top_logp"] = lp.sort(1, descending=True).values[:, :s["top"]]
        if s["train"]:
            glp = s["g_logp"][lo:lo + 512].double().masked_fill(gone, 0)
            gen = s["g_entropy"][lo:lo + 512].double().masked_fill(gone, 0)
            hot = torch.zeros_like(x)
            hot[torch.arange(len(t), device=t.device), t] = 1
            # d logp_t = hot - p,  d entropy = -p log p - p entropy
            part["grad"] = (hot - p) * glp[:, None] \
                + (torch.special.entr(p) - p * h[:, None]) * gen[:, None]
            if s["logits"].numel() > 1 << 28:
                part["grad"] = part["grad"].float()  # memory: rounded far below the outputs' type
        parts.append(part)
    out = {k: torch.cat([q[k] for q in parts]) for k in parts[0]}
    if s["top"]:
        out["top_ids"] = None
    return out


def _exact_kept(x):
    """Values of the 8-bit form, block by block from its definition."""
    rows, cols = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -cols % 32)).view(rows, -1, 32)
    top = v.abs().amax(2)
    e = torch.floor(torch.log2(top)).clamp(-120, 127)
    # log2 may fall on the wrong side of a power of two: put right
    e = e - (torch.exp2(e) > top).double() * (e > -120)
    e = e + (torch.exp2(e + 1) <= top).double() * (e < 127)
    up = (torch.round(top * torch.exp2(6 - e)) >= 128) & (e < 127)
    step = torch.exp2(e + up.double() - 6)[:, :, None]
    k = torch.clamp(torch.round(v / step), -127, 127) * step
    k[~torch.isfinite(top)] = float("nan")
    return k.view(rows, -1)[:, :cols]


def _exact_gelu(s):
    x = s["x"].double()
    k = _exact_kept(s["x"])
    normal = torch.special.erfc(-k / math.sqrt(2)) / 2
    density = torch.exp(-k.square() / 2) / math.sqrt(2 * math.pi)
    return {"y": x * torch.special.erfc(-x / math.sqrt(2)) / 2,
            "grad": s["dy"].double() * (normal + k * density)}


def _exact_dense(s):
    dy = s["dy"].double()
    return {"dw": torch.mm(dy.t(), _exact_kept(s["x"])), "db": dy.sum(0)}


_EXACT = {"norm": _exact_norm, "logprobs": _exact_logprobs, "gelu": _exact_gelu,
          "dense": _exact_dense}
