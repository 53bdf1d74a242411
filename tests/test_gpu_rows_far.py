"""The row operators' kernels where the logits are large next to the differences that matter (rows_far_cases.py)."""
import numpy as np
import pytest

import accelerate_b200 as A
import rows_far_cases as F
from accelerate_b200 import backend
from test_rows import teacher

pytestmark = pytest.mark.gpu
G = np.random.default_rng
RUN = lambda term: backend.run(list(term))  # noqa: E731


def adds(n):
    """The longest chain of additions on the way to a row's sum: one per tile (128 threads of 8 blocks: 4096 Floats or
    8192 Halves), inside a tile 16 pairs and 2, and 5, 3 and 7 to join lanes, warps and a cluster's CTAs."""
    return n // 4096 + 34


SIZES = [(3, 33), (2, 4097), (1, 70001), (1200, 513)]


@pytest.mark.parametrize("rows,n", SIZES)
@pytest.mark.parametrize("t,offset", F.OFFSETS)
def test_log_probabilities_do_not_depend_on_a_constant_part(gpu_ctx, t, offset, rows, n):
    g = G(n)
    x = F.rows_with_a_constant(g, rows, n, t, offset)
    tok = g.integers(-1, n, rows).astype(np.int32)
    F.check_log_probs(5, tok, x, RUN(A.logProbs(5, tok, x)), adds(n))


@pytest.mark.parametrize("rows,n", SIZES)
@pytest.mark.parametrize("t", ["f16", "f32"])
def test_a_row_of_the_lowest_value_is_uniform(gpu_ctx, t, rows, n):
    x = np.full((rows, n), F.LOWEST[t])
    tok = np.arange(rows, dtype=np.int32) % n
    F.check_log_probs(3, tok, x, RUN(A.logProbs(3, tok, x)), adds(n))


@pytest.mark.parametrize("tau", [1.0, 0.25, 1e-4, 3.0])
@pytest.mark.parametrize("rows,n", SIZES)
@pytest.mark.parametrize("t,offset", F.OFFSETS)
def test_the_loss_does_not_depend_on_a_constant_part(gpu_ctx, t, offset, rows, n, tau):
    g = G(n)
    x = F.rows_with_a_constant(g, rows, n, t, offset)
    ids, te = teacher(g, rows, n, 6)
    ids[0, 4:] = -1
    F.check_distill(tau, ids, te, x, RUN(A.distill(tau, ids, te, x)), adds(n))


@pytest.mark.parametrize("tau", [1.0, 0.25, 4.0])
@pytest.mark.parametrize("rows,n", SIZES)
@pytest.mark.parametrize("t", ["f16", "f32"])
def test_the_loss_of_a_row_of_the_lowest_value_is_that_of_a_uniform_student(gpu_ctx, t, rows, n, tau):
    g = G(n)
    x = np.full((rows, n), F.LOWEST[t])
    ids, te = teacher(g, rows, n, 6)
    F.check_distill(tau, ids, te, x, RUN(A.distill(tau, ids, te, x)), adds(n))


def grad_adds(n):
    """The same for the row that the gradient sums itself: 256 threads add their blocks (4 Floats or 8 Halves) one after
    the other, and lanes and warps join in 5 and 8 steps."""
    return n // 1024 + 1 + 8 + 13


GRAD_SIZES = [(3, 33), (2, 4097), (2, 70001), (700, 513)]

@pytest.mark.parametrize("tau", [1.0, 0.25, 1e-4, 3.0])
@pytest.mark.parametrize("rows,n", GRAD_SIZES)
@pytest.mark.parametrize("t,offset", F.OFFSETS)
def test_the_gradient_behind_the_loss_does_not_depend_on_a_constant_part(gpu_ctx, t, offset, rows, n, tau):
    g = G(4)
    x = F.rows_with_a_constant(g, rows, n, t, offset)
    ids, te = teacher(g, rows, n, 6)
    ids[0, 4:] = -1
    ids[1, :] = -1
    up = g.uniform(0.5, 2, rows).astype(np.float32)
    _, lse = RUN(A.distill(tau, ids, te, x))
    F.check_distill_grad(tau, ids, te, x, lse, up, RUN([A.distillGrad(tau, ids, te, x, lse, up)])[0], max(adds(n), grad_adds(n)))


@pytest.mark.parametrize("tau", [1.0, 0.25, 4.0])
@pytest.mark.parametrize("rows,n", GRAD_SIZES)
@pytest.mark.parametrize("t", ["f16", "f32"])
def test_the_gradient_of_rows_of_the_lowest_value_is_that_of_a_uniform_student(gpu_ctx, t, rows, n, tau):
    g = G(5)
    x = np.full((rows, n), F.LOWEST[t])
    x[1, 5:] = -np.inf                    # a few of them, the others masked
    ids, te = teacher(g, rows, 5, 4)
    up = np.full(rows, 2, np.float32)
    _, lse = RUN(A.distill(tau, ids, te, x))
    F.check_distill_grad(tau, ids, te, x, lse, up, RUN([A.distillGrad(tau, ids, te, x, lse, up)])[0], max(adds(n), grad_adds(n)))


@pytest.mark.parametrize("rows,n", GRAD_SIZES)
def test_a_normaliser_that_is_not_the_rows_own_is_taken_as_given(gpu_ctx, rows, n):
    """A row may be a part of a longer one, whose normaliser is larger."""
    g = G(6)
    x = F.rows_with_a_constant(g, rows, n, "f32", 20000.0)
    ids, te = teacher(g, rows, n, 6)
    up = np.ones(rows, np.float32)
    _, lse = RUN(A.distill(1.0, ids, te, x))
    whole = lse + np.float32(1.5)
    assert np.all(whole - lse == 1.5) and np.all(lse > 2 ** 14)
    got = RUN([A.distillGrad(1.0, ids, te, x, whole, up)])[0]
    q = np.zeros(x.shape)
    np.put_along_axis(q, ids, F.teacher_q(1.0, ids, te), -1)
    d = x.astype(np.float64) - whole.astype(np.float64)[:, None]
    p = np.exp(d)
    F.close(got, p - q, F.U * (p * (16 + 5 * np.abs(d)) + q * 200) + F.half_step(p - q, "f32") + 2.0 ** -126, "gradient")


@pytest.mark.parametrize("tau", [1.0, 0.25])
@pytest.mark.parametrize("t", ["f16", "f32"])
def test_rows_of_the_highest_value_are_uniform(gpu_ctx, t, tau):
    """(At a temperature below 1 the normaliser of such Floats is +inf, rounded.)"""
    g = G(8)
    rows, n = 2, 20001
    x = np.full((rows, n), -F.LOWEST[t])
    tok = np.array([3, n - 1], np.int32)
    F.check_log_probs(3, tok, x, RUN(A.logProbs(3, tok, x)), adds(n))
    ids, te = teacher(g, rows, n, 6)
    up = np.ones(rows, np.float32)
    got = RUN(A.distill(tau, ids, te, x))
    F.check_distill(tau, ids, te, x, got, adds(n))
    F.check_distill_grad(tau, ids, te, x, got[1], up, RUN([A.distillGrad(tau, ids, te, x, got[1], up)])[0], max(adds(n), grad_adds(n)))
