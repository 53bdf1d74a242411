"""Row operators: log probabilities with entropy and top alternatives, distillation from a teacher's top
logits (forward and backward), layer norm (forward and backward).

``run`` computes them in their plain form, elementary torch operations in 32 bits, or, where ``own`` is true,
through the array language's own operators on device arrays that share the tensors' memory."""
import functools
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "f32": torch.float32}
BYTES = {"f16": 2, "f32": 4}


def listed():
    return [
        # a sampler's step: four requests' logits, 20 alternatives reported; a call of microseconds
        {"name": "logprobs step", "op": "logprobs", "rows": 4, "n": 131072, "k": 20, "dtype": "f16"},
        # scoring short texts with an odd vocabulary: no row starts on a 16-byte boundary
        {"name": "logprobs odd", "op": "logprobs", "rows": 500, "n": 50257, "k": 5, "dtype": "f32"},
        # log probabilities of whole prompts, the largest reading
        {"name": "logprobs prompts", "op": "logprobs", "rows": 4096, "n": 131072, "k": 20, "dtype": "f16"},
        # distillation loss of one short sequence
        {"name": "distill short", "op": "distill", "rows": 64, "n": 32000, "k": 16, "dtype": "f32", "tau": 2.0},
        # distillation loss of a training batch
        {"name": "distill batch", "op": "distill", "rows": 4096, "n": 131072, "k": 64, "dtype": "f16", "tau": 2.0},
        # its gradient, odd vocabulary, more alternatives than a warp has lanes
        {"name": "distill grad odd", "op": "distill_grad", "rows": 333, "n": 50257, "k": 100, "dtype": "f32", "tau": 1.0},
        # the gradient of the training batch: reads and writes a gigabyte
        {"name": "distill grad batch", "op": "distill_grad", "rows": 4096, "n": 131072, "k": 64, "dtype": "f16", "tau": 2.0},
        # the normalisation in front of one decoding step
        {"name": "norm step", "op": "norm", "rows": 8, "n": 4096, "dtype": "f16", "params": "f16"},
        # a training batch with a width that is no power of two
        {"name": "norm odd", "op": "norm", "rows": 10007, "n": 1000, "dtype": "f32", "params": "f32"},
        # the normalisation of long prompts
        {"name": "norm prompts", "op": "norm", "rows": 65536, "n": 2048, "dtype": "f16", "params": "f16"},
        # backward pass of a small model in full precision
        {"name": "norm grad small", "op": "norm_grad", "rows": 2048, "n": 768, "dtype": "f32", "params": "f32"},
        # backward pass of a large batch, weights kept in 32 bits
        {"name": "norm grad batch", "op": "norm_grad", "rows": 32768, "n": 4096, "dtype": "f16", "params": "f32"},
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logprobs", "distill", "distill_grad", "norm", "norm_grad"])
    dtype = rng.choice(["f16", "f32"])
    if op in ("norm", "norm_grad"):
        n = _spread(rng, 64, 16384)
        if rng.random() < 0.5:
            n = n // 8 * 8
        return {"op": op, "rows": _spread(rng, 1, max(1, min(65536, (1 << 26) // n))), "n": n, "dtype": dtype, "params": rng.choice([dtype, "f32"])}
    n = _spread(rng, 1000, 160000)
    if rng.random() < 0.5:
        n = n // 8 * 8
    case = {"op": op, "rows": _spread(rng, 1, max(1, min(8192, (1 << 28) // n))), "n": n, "dtype": dtype}
    if op == "logprobs":
        return case | {"k": rng.choice([1, 3, 5, 8, 10, 20, 32, 50, 64])}
    return case | {"k": rng.choice([1, 5, 16, 20, 50, 64, 100, 128]), "tau": rng.choice([1.0, 1.5, 2.0, 4.0])}


def _logits(gen, rows, n, dtype):
    """Logits with a part that all rows share (frequent tokens) and rows of different sharpness; stored in the
    model's type, so that the 16-bit ones hold equal values."""
    common = torch.randn(n, device="cuda", generator=gen) * 2
    sharp = 0.5 + 2.5 * torch.rand(rows, 1, device="cuda", generator=gen)
    out = torch.empty(rows, n, device="cuda", dtype=DTYPES[dtype])
    for r in range(0, rows, 1024):
        part = torch.randn(min(1024, rows - r), n, device="cuda", generator=gen)
        out[r : r + 1024] = part * sharp[r : r + 1024] + common
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, rows, n, dt = case["op"], case["rows"], case["n"], DTYPES[case["dtype"]]
    s = {"case": case}
    if op in ("norm", "norm_grad"):
        pt = DTYPES[case["params"]]
        s["x"] = (torch.randn(rows, n, device="cuda", generator=gen) * (0.5 + torch.rand(rows, 1, device="cuda", generator=gen)) + 0.3).to(dt)
        s["gamma"] = (1 + 0.2 * torch.randn(n, device="cuda", generator=gen)).to(pt)
        if op == "norm":
            s["beta"] = (0.1 * torch.randn(n, device="cuda", generator=gen)).to(pt)
        else:
            # what the forward pass left, and the gradient from above
            x = s["x"].float()
            s["mean"] = x.mean(-1)
            s["rstd"] = (x.var(-1, unbiased=False) + 1e-5).rsqrt()
            s["dy"] = (0.1 * torch.randn(rows, n, device="cuda", generator=gen)).to(dt)
        return s
    s["x"] = _logits(gen, rows, n, case["dtype"])
    if op == "logprobs":
        # some words are forbidden in every third row, and some rows are padding without a given token
        forbidden = torch.rand(n, device="cuda", generator=gen) < 0.02
        s["x"][::3].masked_fill_(forbidden, -math.inf)
        tok = torch.randint(0, n, (rows,), device="cuda", generator=gen, dtype=torch.int32)
        s["tokens"] = torch.where(torch.rand(rows, device="cuda", generator=gen) < 0.05, -1, tok).to(torch.int32)
        return s
    # the teacher's top entries: distinct tokens, falling logits; short rows end in absent entries (-1)
    k = case["k"]
    first = torch.randint(0, n, (rows, 1), device="cuda", generator=gen)
    step = 1 + torch.randint(0, max(1, n // k - 1), (rows, 1), device="cuda", generator=gen)
    ids = ((first + step * torch.arange(k, device="cuda")) % n).to(torch.int32)
    length = torch.where(torch.rand(rows, 1, device="cuda", generator=gen) < 0.9, k, torch.randint(0, k + 1, (rows, 1), device="cuda", generator=gen))
    s["ids"] = torch.where(torch.arange(k, device="cuda") < length, ids, -1).contiguous()
    s["teacher"] = (8 - 0.15 * torch.arange(k, device="cuda") - torch.rand(rows, k, device="cuda", generator=gen)).to(dt)
    if op == "distill_grad":
        x, lse = s["x"], torch.empty(rows, device="cuda")
        for r in range(0, rows, 1024):
            lse[r : r + 1024] = torch.logsumexp(x[r : r + 1024].float() / case["tau"], -1)
        s["lse"] = lse
        # the loss is scaled up for 16-bit gradients, and weighs rows differently
        s["g"] = (4096.0 if case["dtype"] == "f16" else 1.0 / rows) * (0.5 + torch.rand(rows, device="cuda", generator=gen))
    return s


# ---- plain form ---------------------------------------------------------------------------------
def _plain_logprobs(s):
    k = s["case"]["k"]
    x = s["x"].float()
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = d.exp()
    z = e.sum(-1)
    lse = m[:, 0] + z.log()
    entropy = z.log() - (e * torch.where(e > 0, d, 0.0)).sum(-1) / z
    tok = s["tokens"].long()
    given = x.gather(-1, tok.clamp(min=0)[:, None])[:, 0]
    logp = torch.where(tok < 0, 0.0, given - lse)
    del d, e
    top, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    return {"logp": logp, "lse": lse, "entropy": entropy, "top": ids[:, :k].to(torch.int32), "top_logp": top[:, :k] - lse[:, None]}


def _teacher_probabilities(s):
    """The teacher's distribution over its present entries, 0 for the absent ones, and the tokens with 0 in their place."""
    there = s["ids"] >= 0
    t = torch.where(there, s["teacher"].float() / s["case"]["tau"], -math.inf)
    m = t.amax(-1, keepdim=True)
    e = (t - torch.where(m == -math.inf, 0.0, m)).exp()
    z = e.sum(-1, keepdim=True)
    return torch.where(z > 0, e / z, 0.0), torch.where(there, s["ids"], 0).long()


def _plain_distill(s):
    tau = s["case"]["tau"]
    x = s["x"].float() / tau
    m = x.amax(-1, keepdim=True)
    lse = m[:, 0] + (x - m).exp().sum(-1).log()
    q, ids = _teacher_probabilities(s)
    logp = x.gather(-1, ids) - lse[:, None]
    loss = tau * tau * torch.where(q > 0, q * (torch.where(q > 0, q, 1.0).log() - logp), 0.0).sum(-1)
    return {"loss": loss, "lse": lse}


def _plain_distill_grad(s):
    tau = s["case"]["tau"]
    q, ids = _teacher_probabilities(s)
    scale = (s["g"] * tau)[:, None]
    p = (s["x"].float() / tau - s["lse"][:, None]).exp()
    d = torch.where((s["ids"] >= 0).any(-1, keepdim=True), scale * p, 0.0)
    return {"dx": d.scatter_add_(-1, ids, -scale * q).to(s["x"].dtype)}


def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    rstd = 1.0 / ((d * d).mean(-1, keepdim=True) + 1e-5).sqrt()
    y = d * rstd * s["gamma"].float() + s["beta"].float()
    return {"y": y.to(s["x"].dtype), "mean": mean[:, 0], "rstd": rstd[:, 0]}


def _plain_norm_grad(s):
    rstd = s["rstd"][:, None]
    xh = (s["x"].float() - s["mean"][:, None]) * rstd
    dy = s["dy"].float()
    a = dy * s["gamma"].float()
    dx = rstd * (a - a.mean(-1, keepdim=True) - xh * (a * xh).mean(-1, keepdim=True))
    pt = s["gamma"].dtype
    return {"dx": dx.to(s["x"].dtype), "dgamma": (dy * xh).sum(0).to(pt), "dbeta": dy.sum(0).to(pt)}


# ---- the framework's operators --------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _executor():
    from accelerate_b200 import backend, sharded

    return sharded.GpuExecutor(backend.default_context())


@functools.lru_cache(maxsize=None)
def _program(op, dtype, params, k, tau):
    """The array program of one operator, built once as a user's program keeps it."""
    import accelerate_b200 as A

    x = A.param(2, dtype)
    if op == "logprobs":
        args = [A.param(1, "i32"), x]
        out = A.logProbs(k, *args)
    elif op == "distill":
        args = [A.param(2, "i32"), A.param(2, dtype), x]
        out = A.distill(tau, *args)
    elif op == "distill_grad":
        args = [A.param(2, "i32"), A.param(2, dtype), x, A.param(1, "f32"), A.param(1, "f32")]
        out = [A.distillGrad(tau, *args)]
    elif op == "norm":
        args = [A.param(1, params), A.param(1, params), x]
        out = A.layerNorm(1e-5, *args)
    else:
        args = [A.param(1, params), x, A.param(1, ("f32", "f32")), A.param(2, dtype)]
        out = A.layerNormGrad(*args)
    program = A.build_program(list(out))
    return program.text, len(program.outputs), [next(i for i, a in enumerate(args) if a.node is node) for node in program.inputs]


def _own(s):
    case = s["case"]
    op, dt = case["op"], case["dtype"]
    ex = _executor()
    text, n_out, order = _program(op, dt, case.get("params"), case.get("k"), case.get("tau"))
    rows = case["rows"]
    if op == "logprobs":
        args = [("i32", s["tokens"]), (dt, s["x"])]
    elif op == "distill":
        args = [("i32", s["ids"]), (dt, s["teacher"]), (dt, s["x"])]
    elif op == "distill_grad":
        args = [("i32", s["ids"]), (dt, s["teacher"]), (dt, s["x"]), ("f32", s["lse"]), ("f32", s["g"])]
    elif op == "norm":
        args = [(case["params"], s["gamma"]), (case["params"], s["beta"]), (dt, s["x"])]
    else:
        args = [(case["params"], s["gamma"]), (dt, s["x"]), None, (dt, s["dy"])]
    arrays = [ex.ctx.wrap(("f32", "f32"), (rows,), [s["mean"].data_ptr(), s["rstd"].data_ptr()]) if a is None else ex.wrap(a[1], a[0]) for a in args]
    # the tensors belong to torch's current stream, the program runs on its own
    current = torch.cuda.current_stream()
    ex.stream.wait_stream(current)
    outs = ex.ctx.execute(text, [arrays[i] for i in order], n_out)
    current.wait_stream(ex.stream)
    leaves = [ex.tensor(o, leaf) for o in outs for leaf in range(len(o.leaf_types))]
    names = {"logprobs": ["logp", "lse", "entropy", "top", "top_logp"], "distill": ["loss", "lse"], "distill_grad": ["dx"],
             "norm": ["y", "mean", "rstd"], "norm_grad": ["dx", "dgamma", "dbeta"]}[op]
    return dict(zip(names, leaves))


def run(state):
    if own:
        return _own(state)
    return {"logprobs": _plain_logprobs, "distill": _plain_distill, "distill_grad": _plain_distill_grad, "norm": _plain_norm, "norm_grad": _plain_norm_grad}[state["case"]["op"]](state)


def work(case):
    rows, n, b = case["rows"], case["n"], BYTES[case["dtype"]]
    if case["op"] in ("norm", "norm_grad"):
        pb = BYTES[case["params"]]
        if case["op"] == "norm":
            return {"bytes": 2 * rows * n * b + 2 * n * pb + 8 * rows, "flops": 8 * rows * n}
        return {"bytes": 3 * rows * n * b + 3 * n * pb + 8 * rows, "flops": 14 * rows * n}
    k = case["k"]
    if case["op"] == "logprobs":
        return {"bytes": rows * (n * b + 4 + 12 + 8 * k), "flops": 7 * rows * n}
    if case["op"] == "distill":
        return {"bytes": rows * (n * b + k * (4 + b) + 8), "flops": 5 * rows * n}
    return {"bytes": rows * (2 * n * b + k * (4 + b) + 8), "flops": 5 * rows * n}


# ---- definitions in 64 bits -------------------------------------------------------------------------
def _exact_rows(case, s, r):
    """Rows `r` (a slice) of everything but the weights' gradients, in double precision."""
    op, tau = case["op"], case.get("tau", 1.0)
    x = s["x"][r].to(torch.float64)
    n = case["n"]
    if op == "norm":
        mean = x.sum(-1) / n
        var = (x - mean[:, None]).pow(2).sum(-1) / n
        rstd = torch.rsqrt(var + 1e-5)
        return {"y": torch.addcmul(s["beta"].double(), (x - mean[:, None]) * rstd[:, None], s["gamma"].double()), "mean": mean, "rstd": rstd}
    if op == "norm_grad":
        dy, mean, rstd = s["dy"][r].double(), s["mean"][r].double()[:, None], s["rstd"][r].double()[:, None]
        u = (x - mean) * rstd
        w = dy * s["gamma"].double()
        both = torch.stack((w.sum(-1), torch.einsum("rn,rn->r", w, u))) / n
        return {"dx": (w - both[0][:, None] - u * both[1][:, None]) * rstd, "dgamma": torch.einsum("rn,rn->n", dy, u), "dbeta": dy.sum(0)}
    logits = x / tau
    lse = torch.logsumexp(logits, -1)
    if op == "logprobs":
        logp = logits - lse[:, None]
        p = torch.exp(logp)
        entropy = -torch.special.xlogy(p, p).sum(-1)
        tok = s["tokens"][r].long()
        given = logp[torch.arange(x.shape[0], device=x.device), tok.clamp(min=0)]
        # order by value, then by falling index: both packed into one whole number
        bits = (s["x"][r].float() + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20) + (n - 1 - torch.arange(n, device=x.device))
        ids = (n - 1) - (torch.topk(order, case["k"], dim=-1, sorted=True).values & ((1 << 20) - 1))
        return {"logp": given.masked_fill(tok < 0, 0.0), "lse": lse, "entropy": entropy, "top": ids.to(torch.int32), "top_logp": logp.gather(-1, ids)}
    ids = s["ids"][r].long()
    t = (s["teacher"][r].double() / tau).masked_fill(ids < 0, -math.inf)
    q = torch.nan_to_num(torch.softmax(t, -1), nan=0.0)
    at = ids.clamp(min=0)
    if op == "distill":
        return {"loss": tau**2 * (torch.special.xlogy(q, q).sum(-1) - (q * (logits.gather(-1, at) - lse[:, None])).sum(-1)), "lse": lse}
    there = (ids >= 0).any(-1, keepdim=True).double()
    d = torch.exp(logits - s["lse"][r].double()[:, None]) * there
    for j in range(case["k"]):
        row = torch.arange(d.shape[0], device=d.device)
        d[row, at[:, j]] -= q[:, j]
    return {"dx": d * (tau * s["g"][r].double())[:, None]}


def exact(case, seed):
    s = prepare(case, seed)
    step = max(1, (1 << 25) // case["n"])
    parts = [_exact_rows(case, s, slice(r, r + step)) for r in range(0, case["rows"], step)]
    # the weights' gradients are sums over all rows, everything else belongs to a row
    return {key: sum(p[key] for p in parts) if key in ("dgamma", "dbeta") else torch.cat([p[key] for p in parts]) for key in parts[0]}
