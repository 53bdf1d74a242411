"""The row operators in 64 bits, straight from their formulas, and how far Float arithmetic may be from them.

Bounds: u = 2^-24 is half a step of Float; a sum of `adds` additions in a row (and a tree of at most 16 more)
is off by at most (adds + 16) u times the sum of its terms' sizes; 2^x comes with 2^-22 = 4 u, and an exponent t
that is off by half a step changes 2^t by at most |t| u ln 2.  A result is rounded once to its type, half a step:
2^-11 of the value for Half (2^-25 near 0), u for Float."""
import numpy as np

U = 2.0 ** -24
NP = {"f16": np.float16, "f32": np.float32}


def half_step(v, t):
    return np.abs(v) * 2.0 ** -11 + 2.0 ** -25 if t == "f16" else np.abs(v) * U + 2.0 ** -149


def logits(g, shape, t, scale=3.0):
    return (g.normal(size=shape) * scale).astype(NP[t])


def _softmax_parts(x, tau):
    """ln sum e^(x/tau) of rows with an element above -inf (else -inf), and the largest x/tau (else 0)."""
    x = x.astype(np.float64) / tau
    m = np.max(x, -1, initial=-np.inf)
    m = np.where(m == -np.inf, 0.0, m)
    with np.errstate(divide="ignore", invalid="ignore"):
        z = np.exp(x - m[..., None]).sum(-1)
        return m + np.log(z), m


def _range(x, tau, lse):
    """Size of the exponents that matter: elements whose probability is above 2^-40."""
    with np.errstate(invalid="ignore"):
        d = lse[..., None] - x.astype(np.float64) / tau
    return np.max(np.where(np.isfinite(d) & (d < 28), np.abs(d), 0.0), -1, initial=0.0)


def lse_bound(x, tau, adds):
    lse, m = _softmax_parts(x, tau)
    fin = np.where(np.isfinite(lse), np.abs(lse), 0.0)
    return U * (adds + 32 + 3 * _range(x, tau, lse) + 4 * (fin + np.abs(m)))


def check_log_probs(k, tok, x, got, adds):
    (logp, lse, ent), (ids, top) = got
    n = x.shape[-1]
    X = x.astype(np.float64)
    want_lse, _ = _softmax_parts(x, 1.0)
    masked = want_lse == -np.inf
    bound = lse_bound(x, 1.0, adds)
    close(lse, want_lse, bound, "lse")
    with np.errstate(invalid="ignore", divide="ignore"):
        lp = np.where(masked[..., None], -np.inf, X - want_lse[..., None])
        p = np.exp(lp)
        want_ent = np.where(masked, 0.0, -np.where(p > 0, p * np.where(p > 0, lp, 0.0), 0.0).sum(-1))
        spread = np.where(p > 0, p * np.abs(np.where(p > 0, lp, 0.0)), 0.0).sum(-1)
    t = np.asarray(tok, np.int64)
    given = np.take_along_axis(lp, np.maximum(t, 0)[..., None], -1)[..., 0] if n else np.zeros(t.shape)
    want = np.where(t < 0, 0.0, given)
    close(logp, want, bound + U * np.where(np.isfinite(want), np.abs(want), 0.0), "log probability")
    close(ent, want_ent, (bound + U * (adds + 48)) * (2 + spread), "entropy")
    # falling values, equal ones by rising index
    assert ids.shape == x.shape[:-1] + (k,) and ids.dtype == np.int32
    order = np.argsort(-X, axis=-1, kind="stable")[..., :k]
    real = min(k, n)
    assert np.array_equal(ids[..., :real], order), "alternatives"
    assert np.all(ids[..., real:] == -1) and np.all(top[..., real:] == -np.inf)
    w = np.take_along_axis(lp, order, -1)
    close(top[..., :real], w, bound[..., None] + U * np.where(np.isfinite(w), np.abs(w), 0.0), "alternatives' log probabilities")


def teacher_q(tau, ids, te):
    t = np.where(ids < 0, -np.inf, te.astype(np.float64) / tau)
    m = np.max(t, -1, initial=-np.inf)
    e = np.exp(t - np.where(m == -np.inf, 0.0, m)[..., None])
    z = e.sum(-1, keepdims=True)
    return np.where(z > 0, e / np.where(z > 0, z, 1.0), 0.0)


def check_distill(tau, ids, te, x, got, adds):
    loss, lse = got
    X = x.astype(np.float64) / tau
    want_lse, _ = _softmax_parts(x, tau)
    bound = lse_bound(x, tau, adds)
    close(lse, want_lse, bound, "normaliser")
    q = teacher_q(tau, ids, te)
    with np.errstate(invalid="ignore", divide="ignore"):
        lp = np.take_along_axis(X, np.maximum(ids, 0), -1) - want_lse[..., None]
        lp = np.where(want_lse[..., None] == -np.inf, -np.inf, lp)
        terms = np.where(q > 0, q * (np.log(np.where(q > 0, q, 1.0)) - lp), 0.0)
    want = tau * tau * terms.sum(-1)
    # every term's size, with the teacher's and the student's exponents
    t = te.astype(np.float64) / tau
    dt = np.where(q > 0, np.max(np.where(ids < 0, -np.inf, t), -1, keepdims=True, initial=-np.inf) - t, 0.0)
    s = np.where(q > 0, np.abs(np.take_along_axis(X, np.maximum(ids, 0), -1)), 0.0)
    size = np.where(q > 0, q * (dt + np.where(np.isfinite(s), s, 0.0)), 0.0).sum(-1) + np.abs(np.where(np.isfinite(want_lse), want_lse, 0.0)) + 1
    close(loss, want, tau * tau * (bound + U * (ids.shape[-1] + 40) * size * (2 + np.max(dt, -1, initial=0.0))) + U * np.where(np.isfinite(want), want, 0.0), "loss")


def check_distill_grad(tau, ids, te, x, lse, g, got):
    q = teacher_q(tau, ids, te)
    X = x.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        ex = X / tau - lse.astype(np.float64)[..., None]
        p = np.where(X == -np.inf, 0.0, np.exp(ex))
    asked = np.zeros(x.shape)
    flat, fi, fq = asked.reshape(-1, x.shape[-1]), ids.reshape(-1, ids.shape[-1]), q.reshape(-1, ids.shape[-1])
    for r in range(flat.shape[0]):
        for i in range(fi.shape[1]):
            if fi[r, i] >= 0:
                flat[r, fi[r, i]] += fq[r, i]
    has = (q.sum(-1) > 0)[..., None]
    scale = (g.astype(np.float64) * tau)[..., None]
    want = np.where(has, scale * (p - asked), 0.0)
    t = te.astype(np.float64) / tau
    far = np.max(np.where(q > 0, np.max(np.where(ids < 0, -np.inf, t), -1, keepdims=True, initial=-np.inf) - t, 0.0), -1, initial=0.0)[..., None]
    bound = np.abs(scale) * (p * U * (12 + 3 * np.where(np.isfinite(ex), np.abs(ex), 0.0)) + asked * U * (2 * ids.shape[-1] + 40 + 6 * far))
    ty = "f16" if x.dtype == np.float16 else "f32"
    assert got.dtype == x.dtype
    close(got, want, bound + half_step(want, ty) + bound * 2.0 ** -10 + np.abs(scale) * 2.0 ** -126, "gradient")


def norm_stats(x, eps):
    X = x.astype(np.float64)
    mean = X.mean(-1)
    var = ((X - mean[..., None]) ** 2).mean(-1)
    return mean, 1 / np.sqrt(var + eps), var


def check_norm(eps, ga, be, x, got, adds):
    y, (mean, rstd) = got
    X = x.astype(np.float64)
    wm, wr, var = norm_stats(x, eps)
    a = U * (adds + 16)
    bm = a * np.abs(X).mean(-1) + U * np.abs(wm)
    close(mean, wm, bm, "mean")
    # the variance around a mean that is off by bm gains bm^2; each deviation is off by its own half step
    br = wr * (0.5 * (a + 6 * U + 4 * U * bm + bm * bm * wr * wr) + 3 * U)
    close(rstd, wr, br, "rstd")
    G, B = ga.astype(np.float64), be.astype(np.float64)
    xh = (X - wm[..., None]) * wr[..., None]
    want = xh * G + B
    bound = np.abs(G) * (np.abs(xh) * (br / wr)[..., None] + bm[..., None] * wr[..., None] + 4 * U * np.abs(xh)) + 2 * U * np.abs(want)
    assert y.dtype == x.dtype
    ty = "f16" if x.dtype == np.float16 else "f32"
    close(y, want, bound + half_step(want, ty) + bound * 2.0 ** -10, "norm")


def check_norm_grad(ga, x, stats, dy, got, adds, rows_adds):
    dx, dg, db = got
    n = x.shape[-1]
    X, D, G = x.astype(np.float64), dy.astype(np.float64), ga.astype(np.float64)
    mean, rstd = stats[0].astype(np.float64)[..., None], stats[1].astype(np.float64)[..., None]
    xh = (X - mean) * rstd
    exh = 2 * U * np.abs(xh)
    A = D * G
    ma, mb = A.mean(-1, keepdims=True), (A * xh).mean(-1, keepdims=True)
    want = rstd * (A - ma - xh * mb)
    ea = U * (adds + 18) * np.abs(A).mean(-1, keepdims=True)
    eb = U * (adds + 22) * np.abs(A * xh).mean(-1, keepdims=True)
    bound = rstd * (ea + np.abs(xh) * eb + exh * np.abs(mb) + 5 * U * (np.abs(A) + np.abs(ma) + np.abs(xh * mb)))
    ty = "f16" if x.dtype == np.float16 else "f32"
    assert dx.dtype == x.dtype and dg.dtype == ga.dtype and db.dtype == ga.dtype
    close(dx, want, bound + half_step(want, ty) + bound * 2.0 ** -10, "rows' gradient")
    pt = "f16" if ga.dtype == np.float16 else "f32"
    P, Q = (D * xh).reshape(-1, n), D.reshape(-1, n)
    for v, terms, extra, name in ((dg, P, 3, "gamma's gradient"), (db, Q, 0, "beta's gradient")):
        w = terms.sum(0)
        b = U * (rows_adds + 24 + extra) * np.abs(terms).sum(0)
        close(v, w, b + half_step(w, pt) + b * 2.0 ** -10, name)


def close(got, want, bound, what):
    got, want, bound = np.asarray(got, np.float64), np.asarray(want, np.float64), np.broadcast_to(bound, np.shape(want))
    assert got.shape == want.shape, (what, got.shape, want.shape)
    with np.errstate(invalid="ignore"):
        ok = np.where(np.isfinite(want), np.abs(got - want) <= bound, (got == want) | (np.isnan(got) & np.isnan(want)))
    if not np.all(ok):
        bad = np.argwhere(~ok)[:4].tolist()
        raise AssertionError(f"{what}: {np.count_nonzero(~ok)} of {ok.size} out of bounds at {bad}: got {got[~ok][:4]}, want {want[~ok][:4]}, bound {bound[~ok][:4]}")
