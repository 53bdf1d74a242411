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
