"""The row operators' kernels against the formulas in 64 bits (rows_cases.py derives the bounds)."""
import numpy as np
import pytest

import accelerate_b200 as A
import rows_cases as R
from accelerate_b200 import backend
from oracle import oracle
from test_rows import teacher

pytestmark = pytest.mark.gpu
G = np.random.default_rng
RUN = lambda term: backend.run(list(term))  # noqa: E731


def adds(n):
    """Additions one thread makes for a row's normaliser: 256 threads, two sums each, 32 elements at a time."""
    return n // 512 + 48


def norm_adds(n):
    """Elements per lane (at most 32 in registers, n / 512 for long rows)."""
    return max(32, n // 512 + 1)


# Lengths around blocks, tiles (4096 Floats, 8192 Halves) and the split over a cluster; odd ones start rows anywhere.
LENGTHS = [(1, 1), (2, 3), (5, 8), (3, 100), (7, 1023), (4, 1024), (3, 4097), (2, 8192), (600, 257), (1, 50257), (2, 131072), (1300, 33)]


@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("k", [0, 1, 20, 128])
@pytest.mark.parametrize("rows,n", LENGTHS)
def test_log_probs(gpu_ctx, t, k, rows, n):
    g = G(rows * n + k)
    x = R.logits(g, (rows, n), t)
    tok = g.integers(-1, n, rows).astype(np.int32 if k else np.int64)
    R.check_log_probs(k, tok, x, RUN(A.logProbs(k, tok, x)), adds(n))


@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("n", [5, 300, 9000, 70001])
@pytest.mark.parametrize("kind", ["all masked", "few left", "lowest", "few above lowest", "constant", "rising", "falling", "ties", "late", "large"])
def test_log_probs_of_unusual_rows(gpu_ctx, t, n, kind):
    g = G(n)
    low = np.float32(-65504) if t == "f16" else np.finfo(np.float32).min
    rows = 3
    x = R.logits(g, (rows, n), "f32")
    some = np.zeros((rows, n), bool)
    some[0, g.integers(0, n, 7)] = True
    some[1, n - 1] = True
    if kind == "all masked":
        x[:] = -np.inf
    elif kind == "few left":
        x[~some] = -np.inf
    elif kind == "lowest":
        x[:] = low
    elif kind == "few above lowest":
        x[~some] = low
    elif kind == "constant":
        x[:] = 0.0
    elif kind == "rising":
        x[:] = np.linspace(-20, 20, n)
    elif kind == "falling":
        x[:] = np.linspace(20, -20, n)
    elif kind == "ties":
        x[:] = g.integers(-3, 3, (rows, n))
    elif kind == "late":                  # the largest elements in the last tile
        x[:, -min(n, 200):] += 40
    else:
        x *= 3000 if t == "f16" else 1e30
    x = np.clip(x, -65504, 65504).astype(np.float16) if t == "f16" and kind not in ("all masked", "few left") else x.astype(R.NP[t])
    tok = g.integers(0, n, rows).astype(np.int32)
    for k in (1, 20, 128):
        R.check_log_probs(k, tok, x, RUN(A.logProbs(k, tok, x)), adds(n))


@pytest.mark.parametrize("t", ["f16", "f32"])
def test_log_probs_with_nan_and_infinity(gpu_ctx, t):
    g = G(9)
    x = R.logits(g, (4, 9001), t)
    x[0, 17] = np.nan
    x[1, 8999] = np.inf
    x[2, 100:200] = np.nan
    x[3, :] = np.nan
    tok = np.zeros(4, np.int32)
    (logp, lse, ent), (ids, top) = RUN(A.logProbs(20, tok, x))
    assert np.all(np.isnan(logp)) and np.all(np.isnan(lse)) and np.all(np.isnan(ent)) and np.all(np.isnan(top))
    key = np.where(np.isnan(x), np.inf, x.astype(np.float64))
    key[1, 8999] = 1e300
    assert np.array_equal(ids, np.argsort(-key, axis=-1, kind="stable")[:, :20])


def test_rows_agree_with_the_definitions(gpu_ctx):
    """Kernel against the array code it stands for, through the oracle: rank 1 and 3, empty arrays."""
    g = G(10)
    for shape, k in (((37,), 4), ((2, 3, 19), 3), ((0, 5), 2), ((2, 0, 5), 2), ((3, 0), 2)):
        x = R.logits(g, shape, "f16")
        tok = np.where(g.random(shape[:-1]) < 0.3, -1, g.integers(0, max(shape[-1], 1), shape[:-1])).astype(np.int32)
        tok = np.full(shape[:-1], -1, np.int32) if shape[-1] == 0 else tok
        a, b = RUN(A.logProbs(k, tok, x)), oracle.run(list(A.logProbs(k, tok, x)))
        assert np.array_equal(a[1][0], b[1][0])
        for u, v in zip(a[0] + a[1][1:], b[0] + b[1][1:]):
            assert u.shape == v.shape and np.allclose(u, v, rtol=1e-5, atol=1e-5, equal_nan=True)
    for shape in ((0, 5), (2, 3, 0)):
        x, v = np.ones(shape, np.float32), np.ones(shape[-1], np.float32)
        y, st = RUN(A.layerNorm(1e-5, v, v, x))
        assert y.shape == shape and np.all(np.isnan(st[0])) and np.all(np.isnan(st[1]))
        dx, dg, db = RUN(A.layerNormGrad(v, x, st, x))
        assert dx.shape == shape and np.all(dg == 0) and np.all(db == 0)
        ids, te = np.zeros(shape[:-1] + (0,), np.int32), np.zeros(shape[:-1] + (0,), np.float32)
        loss, lse = RUN(A.distill(1.0, ids, te, x))
        assert np.all(loss == 0) and np.all(lse == -np.inf)
        assert RUN([A.distillGrad(1.0, ids, te, x, lse, loss)])[0].shape == shape


@pytest.mark.parametrize("t,tt", [("f16", "f32"), ("f16", "f16"), ("f32", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("rows,n,k,tau", [(1, 1, 1, 1.0), (3, 50, 7, 2.0), (5, 1000, 1, 0.5), (2, 4097, 33, 1.0), (700, 300, 20, 4.0), (1, 131072, 64, 2.0), (4, 50257, 100, 1.0),
                                          (2, 2000, 600, 1.5), (2, 9000, 4096, 1.0)])
def test_distill_and_its_gradient(gpu_ctx, t, tt, rows, n, k, tau):
    g = G(rows + n + k)
    x = R.logits(g, (rows, n), t)
    ids, te = teacher(g, rows, n, k, tt)
    if rows > 1:
        ids[0, k // 2:] = -1
        ids[1, :] = -1
    if rows > 2 and k > 3:
        ids[2, 3] = ids[2, 1]            # the same token twice, and one more time
        ids[2, k - 1] = ids[2, 1]
        te[2, 0] = -np.inf
    got = RUN(A.distill(tau, ids, te, x))
    R.check_distill(tau, ids, te, x, got, adds(n))
    up = g.uniform(0.5, 2, rows).astype(np.float32) * (1000 if t == "f16" else 1)
    R.check_distill_grad(tau, ids, te, x, got[1], up, RUN([A.distillGrad(tau, ids, te, x, got[1], up)])[0])


@pytest.mark.parametrize("t", ["f16", "f32"])
def test_distill_of_masked_and_large_rows(gpu_ctx, t):
    g = G(12)
    n, k = 5000, 8
    x = R.logits(g, (5, n), t)
    ids, te = teacher(g, 5, n, k)
    x[0, :] = -np.inf                    # no distribution: the loss is +inf, the gradient -q
    x[1, ids[1, 2]] = -np.inf            # no probability where the teacher has some
    x[2, 10:] = -np.inf
    ids[2] = np.arange(8)
    x[3] *= 2000                         # exponents far apart
    got = RUN(A.distill(2.0, ids, te, x))
    assert got[0][0] == np.inf and got[0][1] == np.inf
    R.check_distill(2.0, ids[2:], te[2:], x[2:], (got[0][2:], got[1][2:]), adds(n))
    up = np.full(5, 3.0, np.float32)
    R.check_distill_grad(2.0, ids, te, x, got[1], up, RUN([A.distillGrad(2.0, ids, te, x, got[1], up)])[0])


@pytest.mark.parametrize("t,pt", [("f16", "f16"), ("f16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 5), (2, 8), (1000, 33), (37, 768), (5, 1000), (300, 1001), (300, 1002), (300, 1004), (9, 4096), (700, 2048), (3, 8192), (2, 8194), (2, 8200), (2, 12296), (2, 16384), (2, 20001), (1, 40000), (3, 140000)])
def test_layer_norm_and_its_gradient(gpu_ctx, t, pt, rows, n):
    g = G(rows + n)
    x = (g.normal(size=(rows, n)) * g.uniform(0.5, 2, (rows, 1)) + 0.4).astype(R.NP[t])
    ga, be = (1 + 0.1 * g.normal(size=n)).astype(R.NP[pt]), g.normal(size=n).astype(R.NP[pt])
    y, st = RUN(A.layerNorm(1e-5, ga, be, x))
    R.check_norm(1e-5, ga, be, x, (y, st), norm_adds(n))
    dy = g.normal(size=(rows, n)).astype(R.NP[t])
    got = RUN(A.layerNormGrad(ga, x, st, dy))
    R.check_norm_grad(ga, x, st, dy, got, norm_adds(n), rows)
    again = RUN(A.layerNormGrad(ga, x, st, dy))
    assert all(np.array_equal(a, b) for a, b in zip(got, again)), "the sums over rows have one order"


@pytest.mark.parametrize("off", [1, 3, 8])
@pytest.mark.parametrize("t", ["f16", "f32"])
def test_rows_that_start_anywhere(gpu_ctx, t, off):
    """Views into larger arrays: bases off a 16-byte boundary, and nothing written outside the results."""
    g = G(off)
    ctx = gpu_ctx
    rows, n = 5, 1232
    size = np.dtype(R.NP[t]).itemsize

    def view(host, where=off):
        """`host` at `where` elements inside a larger device array."""
        flat = np.zeros(host.size + 64, host.dtype)
        flat[where:where + host.size] = host.reshape(-1)
        whole = ctx.from_host(flat)
        ty = {"float16": "f16", "float32": "f32", "int32": "i32"}[host.dtype.name]
        v = ctx.wrap(ty, host.shape, [whole.devptr() + where * host.itemsize])
        v._keepalive = whole
        return v
    x, dy = R.logits(g, (rows, n), t), R.logits(g, (rows, n), t, 1.0)
    tok = g.integers(0, n, rows).astype(np.int32)
    ids, te = teacher(g, rows, n, 9)
    ga, be = (1 + 0.1 * g.normal(size=n)).astype(R.NP[t]), g.normal(size=n).astype(R.NP[t])
    assert size in (2, 4)

    def execute(term, arrays):
        prog = A.build_program(list(term))
        outs = ctx.execute(prog.text, arrays, len(prog.outputs))
        for o, (_, elt) in zip(outs, prog.outputs):
            o.elt = elt
        return [o.download() for o in outs]
    P = A.param
    got = execute(A.logProbs(7, P(1, "i32"), P(2, t)), [view(tok), view(x)])
    R.check_log_probs(7, tok, x, got, adds(n))
    got = execute(A.distill(2.0, P(2, "i32"), P(2, "f32"), P(2, t)), [view(ids), view(te), view(x)])
    R.check_distill(2.0, ids, te, x, got, adds(n))
    up = np.ones(rows, np.float32)
    dx = execute([A.distillGrad(2.0, P(2, "i32"), P(2, "f32"), P(2, t), P(1, "f32"), P(1, "f32"))], [view(ids), view(te), view(x), view(got[1]), view(up)])[0]
    R.check_distill_grad(2.0, ids, te, x, got[1], up, dx)
    y, st = execute(A.layerNorm(1e-5, P(1, t), P(1, t), P(2, t)), [view(ga), view(be), view(x)])
    R.check_norm(1e-5, ga, be, x, (y, st), norm_adds(n))
    both = ctx.from_host(st)
    got = execute(A.layerNormGrad(P(1, t), P(2, t), P(1, ("f32", "f32")), P(2, t)), [view(ga), view(x), both, view(dy)])
    R.check_norm_grad(ga, x, st, dy, got, norm_adds(n), rows)
    got = execute(A.layerNormGrad(P(1, t), P(2, t), P(1, ("f32", "f32")), P(2, t)), [view(ga, 0), view(x, 0), both, view(dy)])
    R.check_norm_grad(ga, x, st, dy, got, norm_adds(n), rows)


def test_offsets_beyond_32_bits(gpu_ctx):
    """Arrays of more than 2^31 elements: the last rows come out as the first ones do."""
    import torch

    from accelerate_b200 import sharded
    ex = sharded.GpuExecutor(gpu_ctx)
    n, rows = 131072 + 8, 16500
    assert rows * n > 2 ** 31
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(rows, n, device="cuda", dtype=torch.float16)
    x[:8] = torch.randn(8, n, device="cuda", generator=gen) * 3
    x[8:-8] = 0
    x[-8:] = x[:8]
    tok = torch.arange(rows, device="cuda", dtype=torch.int32)
    tok[-8:] = tok[:8]
    torch.cuda.synchronize()

    def leaves(term, arrays):
        prog = A.build_program(list(term))
        outs = gpu_ctx.execute(prog.text, arrays, len(prog.outputs))
        gpu_ctx.sync()                   # (the views below are read on torch's stream)
        return [o if o.shape == tuple(x.shape) else [ex.tensor(o, k).cpu().numpy() for k in range(len(o.leaf_types))] for o in outs]
    P = A.param
    dx_ = ex.wrap(x, "f16")
    stats, top = leaves(A.logProbs(5, P(1, "i32"), P(2, "f16")), [ex.wrap(tok, "i32"), dx_])
    for a in stats + top:
        assert np.array_equal(a[:8], a[-8:])
    host = x[:8].cpu().numpy()
    R.check_log_probs(5, tok[:8].cpu().numpy(), host, [[a[:8] for a in stats], [a[:8] for a in top]], adds(n))
    ids = torch.arange(4, device="cuda", dtype=torch.int32).repeat(rows, 1) + (n - 9)
    te = torch.zeros(rows, 4, device="cuda")
    lse, one = torch.tensor(stats[1], device="cuda"), torch.ones(rows, device="cuda")
    torch.cuda.synchronize()
    (dx,) = leaves([A.distillGrad(1.0, P(2, "i32"), P(2, "f32"), P(2, "f16"), P(1, "f32"), P(1, "f32"))],
                   [ex.wrap(ids, "i32"), ex.wrap(te, "f32"), dx_, ex.wrap(lse, "f32"), ex.wrap(one, "f32")])
    d = ex.tensor(dx)
    assert torch.equal(d[:8], d[-8:])
    R.check_distill_grad(1.0, ids[:8].cpu().numpy(), te[:8].cpu().numpy(), host, stats[1][:8], np.ones(8, np.float32), d[:8].cpu().numpy())
    del d, dx
    v = torch.ones(n, device="cuda")
    torch.cuda.synchronize()
    y, st = leaves(A.layerNorm(1e-5, P(1, "f32"), P(1, "f32"), P(2, "f16")), [ex.wrap(v, "f32"), ex.wrap(v, "f32"), dx_])
    t = ex.tensor(y)
    assert torch.equal(t[:8], t[-8:])
    R.check_norm(1e-5, np.ones(n, np.float32), np.ones(n, np.float32), host, (t[:8].cpu().numpy(), [a[:8] for a in st]), norm_adds(n))


def test_a_token_behind_the_row_is_reported(gpu_ctx):
    x = np.zeros((3, 10), np.float32)
    ids, te = np.array([[0], [10], [1]], np.int32), np.zeros((3, 1), np.float32)
    for term in (A.logProbs(2, np.array([0, 10, 1], np.int32), x), A.logProbs(2, np.array([0, 1 << 40, 1]), x), A.distill(1.0, ids, te, x),
                 [A.distillGrad(1.0, ids, te, x, np.zeros(3, np.float32), np.zeros(3, np.float32))]):
        with pytest.raises(backend.B200Error) as e:
            RUN(term)
        assert e.value.code == 5 and "index out of bounds" in str(e.value)
    RUN(A.logProbs(2, np.array([0, 9, -5], np.int32), x))     # the context stays usable


def test_shapes_that_do_not_match_are_refused(gpu_ctx):
    x, v = np.zeros((3, 10), np.float32), np.zeros(10, np.float32)
    ids, te, two, three = np.zeros((3, 2), np.int32), np.zeros((3, 2), np.float32), np.zeros(2, np.float32), np.zeros(3, np.float32)
    for term in (A.logProbs(1, np.zeros(2, np.int32), x), A.distill(1.0, ids[:2], te[:2], x), A.distill(1.0, ids, te[:, :1], x),
                 [A.distillGrad(1.0, ids, te, x, two, three)], [A.distillGrad(1.0, ids, te, x, three, two)],
                 A.layerNorm(1e-5, v[:9], v, x), A.layerNorm(1e-5, v, v[:9], x),
                 A.layerNormGrad(v[:9], x, (three, three), x), A.layerNormGrad(v, x, (two, two), x), A.layerNormGrad(v, x, (three, three), x[:, :9])):
        with pytest.raises(backend.B200Error) as e:
            RUN(term)
        assert e.value.code == 5 and "shape mismatch" in str(e.value)


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
def test_a_capture_is_refused(gpu_ctx):
    import torch
    stream = torch.cuda.ExternalStream(gpu_ctx.stream())
    v = gpu_ctx.from_host(np.ones(8, np.float32))
    x = gpu_ctx.from_host(np.ones((2, 8), np.float32))
    prog = A.build_program(list(A.layerNorm(1e-5, A.param(1, "f32"), A.param(1, "f32"), A.param(2, "f32"))))
    gpu_ctx.execute(prog.text, [v, v, x], 2)
    gpu_ctx.sync()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(backend.B200Error) as e:
        with torch.cuda.graph(graph, stream=stream):
            gpu_ctx.execute(prog.text, [v, v, x], 2)
    assert e.value.code == 6 and "captured" in str(e.value)
    y, _ = gpu_ctx.execute(prog.text, [v, v, x], 2)
    assert np.array_equal(y.download(), np.ones((2, 8), np.float32))


def test_too_many_teacher_entries_are_refused(gpu_ctx):
    x, ids, te = np.zeros((1, 5000), np.float32), np.zeros((1, 4097), np.int32), np.zeros((1, 4097), np.float32)
    one = np.ones(1, np.float32)
    for term in (A.distill(1.0, ids, te, x), [A.distillGrad(1.0, ids, te, x, one, one)]):
        with pytest.raises(backend.B200Error) as e:
            RUN(term)
        assert e.value.code == 6 and "4096" in str(e.value)


def test_memory_that_cannot_be_an_array_is_refused(gpu_ctx):
    import torch

    from accelerate_b200 import sharded
    ex = sharded.GpuExecutor(gpu_ctx)
    t = torch.zeros(4, 6, device="cuda")
    torch.cuda.synchronize()
    with pytest.raises(ValueError):
        ex.wrap(t.t(), "f32")
    with pytest.raises(ValueError):
        gpu_ctx.wrap(("f32", "f32"), (4,), [t.data_ptr()])
    prog = A.build_program(list(A.layerNorm(1e-5, A.param(1, "f32"), A.param(1, "f32"), A.param(2, "f32"))))
    v = gpu_ctx.from_host(np.ones(5, np.float32))
    off = gpu_ctx.wrap("f32", (2, 5), [t.data_ptr() + 2])
    with pytest.raises(backend.B200Error) as e:
        gpu_ctx.execute(prog.text, [v, v, off], 2)
    assert e.value.code == 7 and "boundary" in str(e.value)


def test_inside_a_loop(gpu_ctx):
    """Foreign functions in the body of an awhile: the state goes through the kernel every trip."""
    g = G(22)
    x, ga, be = g.normal(size=(3, 40)).astype(np.float32), np.full(40, 1.5, np.float32), np.full(40, 0.25, np.float32)

    def loop():
        return A.awhile(lambda s: A.unit(A.the(s[1]) < 3), lambda s: (A.layerNorm(1e-5, ga, be, s[0])[0], A.map(lambda n: n + 1, s[1])),
                        (A.use(x), A.unit(A.constant(0))))
    got, want = backend.run(list(loop())), oracle.run(list(loop()))
    # three norms, each a sum of 40 Floats of size at most 10, applied to the last one's error
    assert int(got[1]) == 3 and np.max(np.abs(got[0].astype(np.float64) - want[0])) < 3 * 60 * 2.0 ** -24 * 10


def test_a_teacher_that_is_not_a_number(gpu_ctx):
    x = np.zeros((3, 70), np.float32)
    ids, te = np.array([[1, 2], [3, 3], [-1, 5]], np.int32), np.array([[np.nan, 0], [np.inf, 1], [np.nan, 0]], np.float32)
    loss, lse = RUN(A.distill(1.0, ids, te, x))
    assert np.isnan(loss).tolist() == [True, True, False]
    d = RUN([A.distillGrad(1.0, ids, te, x, lse, np.ones(3, np.float32))])[0]
    want = oracle.run(A.distillGrad(1.0, ids, te, x, lse, np.ones(3, np.float32)))
    assert np.all(np.isnan(d[:2])) and np.all(np.isnan(want[:2])) and np.allclose(d[2], want[2], atol=1e-6)


def test_calls_from_two_threads_and_two_contexts(gpu_ctx):
    import threading
    g = G(20)
    x, tok = R.logits(g, (50, 5001), "f16"), g.integers(0, 5001, 50).astype(np.int32)
    other = backend.Context(gpu_ctx.device)
    want, failed = RUN(A.logProbs(9, tok, x)), []

    def work(ctx):
        try:
            for _ in range(5):
                got = backend.run(list(A.logProbs(9, tok, x)), ctx)
                for a, b in zip(want, got):
                    assert all(np.array_equal(u, v) for u, v in zip(a, b))
        except Exception as e:  # noqa: BLE001
            failed.append(e)
    A.language.reset_names()
    threads = [threading.Thread(target=work, args=(c,)) for c in (gpu_ctx, gpu_ctx, other)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    other.close()
    assert not failed, failed


def test_one_program_from_the_norm_to_its_gradient(gpu_ctx):
    """Teacher and student heads over the same hidden rows, in one program: norm, logits, the teacher's top alternatives, the
    student's distillation loss, its gradient back through the head to the norm's weights; kernels against definitions."""
    g = G(21)
    rows, width, n, k, tau = 6, 48, 130, 5, 2.0
    h = g.normal(size=(rows, width)).astype(np.float32)
    ga, be = (1 + 0.1 * g.normal(size=width)).astype(np.float32), (0.1 * g.normal(size=width)).astype(np.float32)
    wt, ws = (g.normal(size=(n, width)) * 0.3).astype(np.float32), (g.normal(size=(n, width)) * 0.3).astype(np.float32)
    tok = g.integers(0, n, rows).astype(np.int32)
    add = lambda a, b: a + b  # noqa: E731

    def product(a, b, across):           # a (rows, m) times b (columns, m) or, across, times b (m, columns)
        a, b = A.use(a), A.use(b)
        cols = b.shape[1] if across else b.shape[0]
        return A.compute(A.fold(add, 0.0, A.generate(A.index(a.shape[0], cols, a.shape[1]),
                                                     lambda ix: a[A.index(ix[0], ix[2])] * (b[A.index(ix[2], ix[1])] if across else b[A.index(ix[1], ix[2])]))))

    def step(h, ga, be, wt, ws, tok):
        hidden, st = A.layerNorm(1e-5, ga, be, h)
        stats, top = A.logProbs(k, tok, product(hidden, wt, False))
        ids, lp = A.map(lambda e: e[0], top), A.map(lambda e: e[1], top)
        student = product(hidden, ws, False)
        loss, lse = A.distill(tau, ids, lp, student)
        one = A.fill(loss.shape, A.constant(np.float32(1)))
        d = A.distillGrad(tau, ids, lp, student, lse, one)
        dh, dga, dbe = A.layerNormGrad(ga, h, st, product(d, ws, True))
        return [stats, top, loss, d, dh, dga, dbe]
    args = (h, ga, be, wt, ws, tok)
    got = backend.run(step(*args))
    want = oracle.run(step(*args))
    assert np.array_equal(got[1][0], want[1][0])
    for a, b in zip(got, want):
        for u, v in zip(a if isinstance(a, tuple) else (a,), b if isinstance(b, tuple) else (b,)):
            # six steps of sums of at most 130 Floats of size one: 6 * 130 * 2^-24
            assert np.max(np.abs(u.astype(np.float64) - v)) < 6 * 130 * 2.0 ** -24 * max(1.0, np.max(np.abs(v))), (u, v)
    again = backend.runN(lambda *xs: step(*xs))(*args)
    assert all(np.array_equal(u, v) for u, v in zip(again[4:], got[4:]))
