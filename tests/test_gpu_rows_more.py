"""The row operators' kernels between the sizes of test_gpu_rows.py: alternatives up to the most, lengths around the splits
of a row over a cluster, indices beyond 32 bits in every operator, a context that another thread keeps busy."""
import numpy as np
import pytest

import accelerate_b200 as A
import rows_cases as R
from accelerate_b200 import sharded
from test_gpu_rows_far import RUN, adds
from test_rows import teacher

pytestmark = pytest.mark.gpu
G = np.random.default_rng
TILE = {"f16": 8192, "f32": 4096}         # 128 threads of 8 blocks of 16 bytes


@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("k", [21, 33, 64, 100, 124, 125, 127, 128])
@pytest.mark.parametrize("rows,n", [(2, 70001), (700, 9000)])
def test_alternatives_up_to_the_most(gpu_ctx, t, k, rows, n):
    """(From 125 on a third of random rows lists more blocks in its first tile than there is room for.)"""
    g = G(k)
    x = R.logits(g, (rows, n), t)
    tok = g.integers(-1, n, rows).astype(np.int32)
    R.check_log_probs(k, tok, x, RUN(A.logProbs(k, tok, x)), adds(n))


@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("off", [-1, 0, 1])
@pytest.mark.parametrize("tiles", [1, 2, 4, 8])
def test_lengths_around_the_splits_of_a_row(gpu_ctx, t, tiles, off):
    n, rows = tiles * TILE[t] + off, 3
    g = G(n)
    x = R.logits(g, (rows, n), t)
    x[:, -1] += 30                        # the last element is one of the alternatives
    x[0, TILE[t] - 2:TILE[t] + 2] += 25
    tok = np.array([n - 1, 0, n // 2], np.int32)
    R.check_log_probs(20, tok, x, RUN(A.logProbs(20, tok, x)), adds(n))
    ids, te = teacher(g, rows, n, 9)
    ids[0, :2] = n - 1, 0
    got = RUN(A.distill(2.0, ids, te, x))
    R.check_distill(2.0, ids, te, x, got, adds(n))
    up = g.uniform(0.5, 2, rows).astype(np.float32)
    R.check_distill_grad(2.0, ids, te, x, got[1], up, RUN([A.distillGrad(2.0, ids, te, x, got[1], up)])[0])


def execute(ctx, term, arrays):
    prog = A.build_program(list(term))
    outs = ctx.execute(prog.text, arrays, len(prog.outputs))
    ctx.sync()                            # (the views are read on torch's stream)
    return outs


def test_distillation_beyond_32_bits(gpu_ctx):
    import torch
    ex = sharded.GpuExecutor(gpu_ctx)
    n, rows = 131072 + 8, 16500
    assert rows * n > 2 ** 31
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.zeros(rows, n, device="cuda", dtype=torch.float16)
    x[:8] = torch.randn(8, n, device="cuda", generator=gen) * 3
    x[-8:] = x[:8]
    ids = torch.arange(4, device="cuda", dtype=torch.int32).repeat(rows, 1) + (n - 9)
    te = torch.randn(rows, 4, device="cuda", generator=gen)
    te[-8:] = te[:8]
    torch.cuda.synchronize()
    P = A.param
    loss, lse = execute(gpu_ctx, A.distill(2.0, P(2, "i32"), P(2, "f32"), P(2, "f16")), [ex.wrap(ids, "i32"), ex.wrap(te, "f32"), ex.wrap(x, "f16")])
    got = [ex.tensor(a).cpu().numpy() for a in (loss, lse)]
    for a in got:
        assert np.array_equal(a[:8], a[-8:])
    R.check_distill(2.0, ids[:8].cpu().numpy(), te[:8].cpu().numpy(), x[:8].cpu().numpy(), [a[:8] for a in got], adds(n))


@pytest.mark.parametrize("n", [4096, 4095, 131072 + 8])
def test_norm_gradients_beyond_32_bits(gpu_ctx, n):
    """(Rows that stay in registers, on any boundary, and rows that are read again.)"""
    import torch
    ex = sharded.GpuExecutor(gpu_ctx)
    rows = 2 ** 31 // n + 50
    gen = torch.Generator(device="cuda").manual_seed(3)
    x, dy = (torch.zeros(rows, n, device="cuda", dtype=torch.float16) for _ in range(2))
    for a in (x, dy):
        a[:8] = torch.randn(8, n, device="cuda", generator=gen)
        a[-8:] = torch.randn(8, n, device="cuda", generator=gen)
    gamma = 1 + 0.1 * torch.randn(n, device="cuda", generator=gen)
    mean, rstd = x.mean(-1, dtype=torch.float32), torch.ones(rows, device="cuda")
    torch.cuda.synchronize()
    P = A.param
    stats = gpu_ctx.wrap(("f32", "f32"), (rows,), [mean.data_ptr(), rstd.data_ptr()])
    dx, dg, db = execute(gpu_ctx, A.layerNormGrad(P(1, "f32"), P(2, "f16"), P(1, ("f32", "f32")), P(2, "f16")),
                         [ex.wrap(gamma, "f32"), ex.wrap(x, "f16"), stats, ex.wrap(dy, "f16")])
    ends = np.r_[0:8, rows - 8:rows]
    host = lambda a: torch.cat([a[:8], a[-8:]]).cpu().numpy()  # noqa: E731
    view = ex.tensor(dx)
    assert not view[8:-8].any(), "rows without a gradient have none"
    # (the rows between add zeros: the sums over rows have as many terms as these sixteen)
    R.check_norm_grad(gamma.cpu().numpy(), host(x), (host(mean), host(rstd)), host(dy), (host(view), ex.tensor(dg).cpu().numpy(), ex.tensor(db).cpu().numpy()),
                      max(32, n // 512 + 1), len(ends))


def test_python_runs_while_a_context_is_busy(gpu_ctx):
    """One thread waits in a download, another for its turn on the same context; a third, this one, goes on."""
    import threading
    import time

    import torch
    g = G(7)
    x, tok = R.logits(g, (4, 1000), "f32"), np.zeros(4, np.int32)
    prog = A.build_program(list(A.logProbs(3, A.param(1, "i32"), A.param(2, "f32"))))
    ins = [gpu_ctx.from_host(tok), gpu_ctx.from_host(x)]
    first = gpu_ctx.execute(prog.text, ins, 2)
    gpu_ctx.sync()
    with torch.cuda.stream(torch.cuda.ExternalStream(gpu_ctx.stream())):
        torch.cuda._sleep(1_000_000_000)   # half a second
    later = []
    threads = [threading.Thread(target=first[0].download), threading.Thread(target=lambda: later.append(gpu_ctx.execute(prog.text, ins, 2)))]
    began = last = time.perf_counter()
    longest = 0.0
    for t in threads:
        t.start()
        time.sleep(0.02)
    while any(t.is_alive() for t in threads):
        time.sleep(0.001)
        now = time.perf_counter()
        longest, last = max(longest, now - last), now
    assert last - began > 0.3 and longest < 0.2
    for a, b in zip(first, later[0]):
        assert all(np.array_equal(u, v) for u, v in zip(a.download(), b.download()))
