"""The row operators' definitions in array code where the logits are large next to the differences that matter."""
import numpy as np
import pytest

import accelerate_b200 as A
import rows_far_cases as F
from oracle import oracle
from test_rows import teacher

G = np.random.default_rng
RUN = lambda term: oracle.run(list(term))  # noqa: E731


@pytest.mark.parametrize("t,offset", F.OFFSETS)
def test_log_probabilities_do_not_depend_on_a_constant_part(t, offset):
    g = G(1)
    x = F.rows_with_a_constant(g, 3, 40, t, offset)
    tok = np.array([0, 7, -1], np.int32)
    F.check_log_probs(5, tok, x, oracle.run(list(A.logProbs(5, tok, x))), 40)


@pytest.mark.parametrize("t", ["f16", "f32"])
def test_a_row_of_the_lowest_value_is_uniform(t):
    x = np.full((2, 32), F.LOWEST[t])
    tok = np.array([3, 31], np.int32)
    F.check_log_probs(3, tok, x, oracle.run(list(A.logProbs(3, tok, x))), 32)


@pytest.mark.parametrize("tau", [1.0, 0.25, 1e-4, 3.0])
@pytest.mark.parametrize("t,offset", F.OFFSETS)
def test_the_loss_does_not_depend_on_a_constant_part(t, offset, tau):
    g = G(2)
    x = F.rows_with_a_constant(g, 3, 40, t, offset)
    ids, te = teacher(g, 3, 40, 6)
    ids[1, 4:] = -1
    F.check_distill(tau, ids, te, x, oracle.run(list(A.distill(tau, ids, te, x))), 40)


@pytest.mark.parametrize("tau", [1.0, 0.25, 4.0])
@pytest.mark.parametrize("t", ["f16", "f32"])
def test_the_loss_of_a_row_of_the_lowest_value_is_that_of_a_uniform_student(t, tau):
    """(At a temperature below 1 the normaliser of such Floats is -inf, rounded; the student is uniform all the same.)"""
    g = G(3)
    x = np.full((2, 32), F.LOWEST[t])
    ids, te = teacher(g, 2, 32, 6)
    F.check_distill(tau, ids, te, x, oracle.run(list(A.distill(tau, ids, te, x))), 32)


@pytest.mark.parametrize("tau", [1.0, 0.25, 1e-4, 3.0])
@pytest.mark.parametrize("t,offset", F.OFFSETS)
def test_the_gradient_behind_the_loss_does_not_depend_on_a_constant_part(t, offset, tau):
    g = G(4)
    rows, n = 3, 40
    x = F.rows_with_a_constant(g, rows, n, t, offset)
    ids, te = teacher(g, rows, n, 6)
    ids[0, 4:] = -1
    ids[1, :] = -1
    up = g.uniform(0.5, 2, rows).astype(np.float32)
    _, lse = RUN(A.distill(tau, ids, te, x))
    F.check_distill_grad(tau, ids, te, x, lse, up, RUN([A.distillGrad(tau, ids, te, x, lse, up)])[0], n)


@pytest.mark.parametrize("tau", [1.0, 0.25, 4.0])
@pytest.mark.parametrize("t", ["f16", "f32"])
def test_the_gradient_of_rows_of_the_lowest_value_is_that_of_a_uniform_student(t, tau):
    g = G(5)
    rows, n = 2, 32
    x = np.full((rows, n), F.LOWEST[t])
    x[1, 5:] = -np.inf                    # a few of them, the others masked
    ids, te = teacher(g, rows, 5, 4)
    up = np.full(rows, 2, np.float32)
    _, lse = RUN(A.distill(tau, ids, te, x))
    F.check_distill_grad(tau, ids, te, x, lse, up, RUN([A.distillGrad(tau, ids, te, x, lse, up)])[0], n)


def test_a_normaliser_that_is_not_the_rows_own_is_taken_as_given():
    """A row may be a part of a longer one, whose normaliser is larger."""
    g = G(6)
    rows, n = 3, 40
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
def test_rows_of_the_highest_value_are_uniform(t, tau):
    """(At a temperature below 1 the normaliser of such Floats is +inf, rounded.)"""
    g = G(8)
    rows, n = 2, 32
    x = np.full((rows, n), -F.LOWEST[t])
    tok = np.array([3, n - 1], np.int32)
    F.check_log_probs(3, tok, x, RUN(A.logProbs(3, tok, x)), n)
    ids, te = teacher(g, rows, n, 6)
    up = np.ones(rows, np.float32)
    got = RUN(A.distill(tau, ids, te, x))
    F.check_distill(tau, ids, te, x, got, n)
    F.check_distill_grad(tau, ids, te, x, got[1], up, RUN([A.distillGrad(tau, ids, te, x, got[1], up)])[0], n)
