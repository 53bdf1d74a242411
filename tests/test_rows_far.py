"""The row operators' definitions in array code where the logits are large next to the differences that matter."""
import numpy as np
import pytest

import accelerate_b200 as A
import rows_far_cases as F
from oracle import oracle
from test_rows import teacher

G = np.random.default_rng


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
