"""The row operators on the CPU: their definitions in array code on the oracle against the formulas in 64 bits, their
checks of arguments, and their kernels through the compiler."""
import numpy as np
import pytest

import accelerate_b200 as A
import rows_cases as R
from oracle import oracle

G = np.random.default_rng


def teacher(g, rows, n, k, t="f32"):
    ids = np.stack([g.permutation(n)[:k] if k <= n else g.integers(0, n, k) for _ in range(rows)]).astype(np.int32).reshape(rows, k)
    return ids, (g.normal(size=(rows, k)) * 2).astype(R.NP[t])


@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (3, 7, 3), (2, 5, 8), (4, 33, 0), (0, 9, 2)])
def test_log_probs_definition(t, rows, n, k):
    g = G(1)
    x = R.logits(g, (rows, n), t)
    if rows > 2:
        x[1, :] = -np.inf
        x[2, : n - 1] = -np.inf
    tok = g.integers(-1, n, rows).astype(np.int32)
    got = oracle.run(list(A.logProbs(k, tok, x)))
    R.check_log_probs(k, tok, x, got, n)


def test_log_probs_of_a_vector_and_of_rank_three():
    g = G(2)
    x = R.logits(g, (11,), "f32")
    R.check_log_probs(3, np.int32(4), x, oracle.run(list(A.logProbs(3, np.array(4, np.int32), x))), 11)
    x = R.logits(g, (2, 3, 6), "f16")
    tok = g.integers(0, 6, (2, 3))
    R.check_log_probs(2, tok, x, oracle.run(list(A.logProbs(2, tok, x))), 6)


def test_equal_logits_rank_by_index_and_nan_comes_first():
    x = np.array([[1, 3, 3, 0, -0.0, 3], [0, np.nan, 5, np.inf, np.nan, 1]], np.float32)
    (_, lse, ent), (ids, top) = oracle.run(list(A.logProbs(6, np.array([-1, -1], np.int32), x)))
    assert ids.tolist() == [[1, 2, 5, 0, 3, 4], [1, 4, 3, 2, 5, 0]]
    assert np.isnan(lse[1]) and np.isnan(ent[1]) and np.all(np.isnan(top[1]))


@pytest.mark.parametrize("t,tt,tau", [("f16", "f32", 1.0), ("f32", "f16", 2.0), ("f16", "f16", 0.5)])
def test_distill_definitions(t, tt, tau):
    g = G(3)
    rows, n, k = 5, 19, 6
    x = R.logits(g, (rows, n), t)
    ids, te = teacher(g, rows, n, k, tt)
    ids[0, 3:] = -1                       # a short list
    ids[1, :] = -1                        # none
    ids[2, 4] = ids[2, 1]                 # an entry twice
    te[3, 2] = -np.inf                    # an entry without weight
    x[4, [j for j in range(n) if j not in ids[4]]] = -np.inf
    got = oracle.run(list(A.distill(tau, ids, te, x)))
    R.check_distill(tau, ids, te, x, got, n)
    up = g.uniform(0.5, 2, rows).astype(np.float32)
    R.check_distill_grad(tau, ids, te, x, got[1], up, oracle.run(A.distillGrad(tau, ids, te, x, got[1], up)))


def test_distill_where_the_student_has_no_probability():
    x = np.full((2, 4), -np.inf, np.float32)
    x[0, 1] = 0.0
    ids, te = np.array([[0, 1], [2, 3]], np.int32), np.zeros((2, 2), np.float32)
    loss, lse = oracle.run(list(A.distill(1.0, ids, te, x)))
    assert np.all(loss == np.inf) and lse.tolist() == [0.0, -np.inf]
    got = oracle.run(A.distillGrad(1.0, ids, te, x, lse, np.ones(2, np.float32)))
    assert got.tolist() == [[-0.5, 0.5, 0, 0], [0, 0, -0.5, -0.5]]


@pytest.mark.parametrize("t,pt", [("f16", "f16"), ("f16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 17), (5, 64), (0, 8)])
def test_norm_definitions(t, pt, rows, n):
    g = G(4)
    x = (g.normal(size=(rows, n)) + 0.5).astype(R.NP[t])
    ga, be = (1 + 0.1 * g.normal(size=n)).astype(R.NP[pt]), g.normal(size=n).astype(R.NP[pt])
    y, st = oracle.run(list(A.layerNorm(1e-3, ga, be, x)))
    R.check_norm(1e-3, ga, be, x, (y, st), n)
    dy = g.normal(size=(rows, n)).astype(R.NP[t])
    R.check_norm_grad(ga, x, st, dy, oracle.run(list(A.layerNormGrad(ga, x, st, dy))), n, rows)


def test_gradients_are_the_differences_of_the_losses():
    """The definitions' gradients against central differences of the 64-bit formulas."""
    g = G(5)
    n, k, tau = 9, 3, 1.5
    x, (ids, te) = g.normal(size=(1, n)).astype(np.float32), teacher(g, 1, n, k)
    q = R.teacher_q(tau, ids, te)

    def loss(v):
        lse, _ = R._softmax_parts(v, tau)
        return tau * tau * np.sum(q * (np.log(q) - (np.take_along_axis(v, ids, -1) / tau - lse[:, None])))
    _, lse = oracle.run(list(A.distill(tau, ids, te, x)))
    got = oracle.run(A.distillGrad(tau, ids, te, x, lse, np.ones(1, np.float32)))
    X, h = x.astype(np.float64), 1e-5
    want = [(loss(X + h * np.eye(n)[j]) - loss(X - h * np.eye(n)[j])) / (2 * h) for j in range(n)]
    # differences are off by h^2/6 times the third derivative (below 1 / tau here) and 2^-52 loss / h
    assert np.max(np.abs(got[0] - want)) < 1e-6
    x = g.normal(size=(4, n)).astype(np.float32)
    ga, be, w = (1 + 0.1 * g.normal(size=n)).astype(np.float32), np.zeros(n, np.float32), g.normal(size=(4, n)).astype(np.float32)
    _, st = oracle.run(list(A.layerNorm(1e-2, ga, be, x)))
    dx, dg, db = oracle.run(list(A.layerNormGrad(ga, x, st, w)))

    def value(v, gam):
        m, r, _ = R.norm_stats(v, 1e-2)
        return np.sum(w * ((v - m[:, None]) * r[:, None] * gam))
    X, Ga = x.astype(np.float64), ga.astype(np.float64)
    for i in range(4):
        for j in range(n):
            e = np.zeros((4, n))
            e[i, j] = h
            assert abs(dx[i, j] - (value(X + e, Ga) - value(X - e, Ga)) / (2 * h)) < 2e-5
    for j in range(n):
        e = h * np.eye(n)[j]
        assert abs(dg[j] - (value(X, Ga + e) - value(X, Ga - e)) / (2 * h)) < 2e-5
    assert np.allclose(db, w.sum(0), atol=1e-5)


def test_arguments_are_checked():
    x, v = np.zeros((2, 4), np.float32), np.zeros(4, np.float32)
    tok = np.zeros(2, np.int32)
    ids = np.zeros((2, 3), np.int32)
    bad = [
        lambda: A.logProbs(129, tok, x), lambda: A.logProbs(-1, tok, x), lambda: A.logProbs(1.5, tok, x),
        lambda: A.logProbs(1, tok, x.astype(np.float64)), lambda: A.logProbs(1, tok.astype(np.int16), x), lambda: A.logProbs(1, ids, x),
        lambda: A.distill(0.0, ids, ids.astype(np.float32), x), lambda: A.distill(float("nan"), ids, ids.astype(np.float32), x),
        lambda: A.distill(1.0, ids.astype(np.int64), ids.astype(np.float32), x), lambda: A.distill(1.0, ids, ids, x),
        lambda: A.distillGrad(1.0, ids, ids.astype(np.float32), x, tok, tok.astype(np.float32)),
        lambda: A.layerNorm(-1.0, v, v, x), lambda: A.layerNorm(float("nan"), v, v, x), lambda: A.layerNorm(1e-5, v, v.astype(np.float16), x),
        lambda: A.layerNorm(1e-5, v.astype(np.float16), v.astype(np.float16), x), lambda: A.layerNorm(1e-5, v, v, x.astype(np.float64)),
        lambda: A.layerNormGrad(v, x, (tok.astype(np.float32), tok), x),
        lambda: A.layerNormGrad(v, x, (tok.astype(np.float32), tok.astype(np.float32)), x.astype(np.float16)),
    ]
    for f in bad:
        with pytest.raises(TypeError):
            f()


def test_numpy_numbers_are_numbers():
    x = np.zeros((2, 4), np.float32)
    A.logProbs(np.int64(2), np.zeros(2, np.int32), x)
    A.distill(np.float32(2), np.zeros((2, 1), np.int32), np.zeros((2, 1), np.float32), x)


def _texts():
    out = {}
    for t in ("f16", "f32"):
        x, v = A.param(2, t), A.param(1, "f32")
        ids, te = A.param(2, "i32"), A.param(2, "f32")
        out["logProbs", t] = list(A.logProbs(5, A.param(1, "i64"), x))
        out["logProbs0", t] = list(A.logProbs(0, A.param(1, "i32"), x))
        out["distill", t] = list(A.distill(2.0, ids, te, x))
        out["distillGrad", t] = [A.distillGrad(2.0, ids, te, x, A.param(1, "f32"), A.param(1, "f32"))]
        out["layerNorm", t] = list(A.layerNorm(1e-5, v, v, x))
        out["layerNormGrad", t] = list(A.layerNormGrad(v, x, A.param(1, ("f32", "f32")), A.param(2, t)))
    return {key: A.build_program(r).text for key, r in out.items()}


def test_kernels_compile(lib_built):
    from accelerate_b200 import backend
    for text in _texts().values():
        log = backend.compile_check(text)
        assert "ok rows_" in log and "elementwise" not in log, "one operator's kernels and nothing of its definition"


def test_program_text_is_checked_by_the_library(lib_built):
    from accelerate_b200 import backend
    texts = _texts()
    lp, di, ln, lg = texts["logProbs", "f32"], texts["distill", "f32"], texts["layerNorm", "f32"], texts["layerNormGrad", "f32"]
    cases = [
        (lp.replace("(consts 5)", "(consts 129)"), 6), (lp.replace("(consts 5)", "(consts 2.5)"), 6), (lp.replace("(consts 5)", "(consts)"), 2),
        (lp.replace("(consts 5)", "(consts five)"), 1), (lp.replace("b200.logProbs", "b200.distill"), 2),
        (di.replace("(consts 0x1.0000000000000p+1)", "(consts 0)"), 7), (di.replace("(consts 0x1.0000000000000p+1)", "(consts nan)"), 7),
        (ln.replace("(consts 0x", "(consts -0x"), 7), (lg.replace("b200.layerNormGrad", "b200.distillGrad"), 2),
    ]
    for text, code in cases:
        assert text not in texts.values()
        with pytest.raises(backend.B200Error) as e:
            backend.compile_check(text)
        assert e.value.code == code, (e.value, text[:200])


def test_a_function_of_another_backend_runs_its_definition(lib_built):
    from accelerate_b200 import backend
    text = ("(program (in a0 (array 1 f32)) (let a1 (aforeign vendor.twice (consts) (afun ((a2 (array 1 f32))) "
            "(let a3 (generate f32 (shape a2) (lam ((v0 (tup i64))) (prim mul f32 (index a2 (var v0)) (const f32 2))))) (out a3)) (args a0))) (out a1))")
    assert "ok elementwise" in backend.compile_check(text)
    x = np.arange(5, dtype=np.float32)
    assert np.array_equal(oracle.run_text(text, [((5,), [x])])[0][1][0], 2 * x)
