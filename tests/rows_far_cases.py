"""The row operators in 64 bits where the logits are large next to the differences that matter (a constant part, masks of
the type's lowest value, small temperatures): everything relative to the row's maximum m, as a softmax is stable.

Bounds, u = 2^-24: x - m is off by half a step of itself, (x - m) / tau by three; an exponent t that is off by three half
steps changes e^t by 3 |t| u, and e^t itself comes with 4 u; a sum of `adds` additions and a tree of 16 more loses
(adds + 16) u.  So ln Z, Z = sum e^((x - m) / tau), is off by u (adds + 20 + 3 range + 2 |ln Z|), range being the largest
|t| of an element that counts (above 2^-40), and nothing in a log probability is as large as the logits."""
import numpy as np

from rows_cases import NP, U, close, half_step, teacher_q


def parts(x, tau):
    """t = (x - m) / tau and ln Z in 64 bits; rows without an element above -inf: -inf and -inf."""
    X = x.astype(np.float64)
    m = np.max(X, -1, initial=-np.inf, keepdims=True)
    t = (X - np.where(m == -np.inf, 0.0, m)) / tau
    with np.errstate(divide="ignore"):
        return t, np.log(np.exp(t).sum(-1)), np.where(m == -np.inf, 0.0, m)[..., 0] / tau


def ln_z_bound(t, ln_z, adds):
    far = np.max(np.where(t > -28, -t, 0.0), -1, initial=0.0)
    return U * (adds + 20 + 3 * far + 2 * np.where(np.isfinite(ln_z), np.abs(ln_z), 0.0))


def check_log_probs(k, tok, x, got, adds):
    (logp, lse, ent), (ids, top) = got
    t, ln_z, m = parts(x, 1.0)
    bound = ln_z_bound(t, ln_z, adds)
    # (the normaliser itself is one Float: half a step of each of its two parts, and of their sum)
    with np.errstate(over="ignore"):
        close(lse, m + ln_z, bound + U * (np.abs(m) + 2 * np.abs(np.where(np.isfinite(ln_z), m + ln_z, 0.0))), "normaliser")
    lp = np.where(ln_z[..., None] == -np.inf, -np.inf, t - np.where(np.isfinite(ln_z), ln_z, 0.0)[..., None])

    def off(want, exponent, b):
        with np.errstate(invalid="ignore"):
            return b + U * np.where(np.isfinite(want), np.abs(want) + np.abs(exponent), 0.0)
    at = np.maximum(np.asarray(tok, np.int64), 0)[..., None]
    given, d = np.take_along_axis(lp, at, -1)[..., 0], np.take_along_axis(t, at, -1)[..., 0]
    want = np.where(np.asarray(tok) < 0, 0.0, given)
    close(logp, want, off(want, d, bound), "log probability")
    order = np.argsort(-x.astype(np.float64), axis=-1, kind="stable")[..., :k]
    assert np.array_equal(ids, order), "alternatives"
    w, d = np.take_along_axis(lp, order, -1), np.take_along_axis(t, order, -1)
    close(top, w, off(w, d, bound[..., None]), "alternatives' log probabilities")


def check_distill(tau, ids, te, x, got, adds):
    loss, lse = got
    t, ln_z, _ = parts(x, tau)
    q = teacher_q(tau, ids, te)
    s = np.take_along_axis(t, np.maximum(ids, 0), -1)
    with np.errstate(divide="ignore", invalid="ignore"):
        terms = np.where(q > 0, q * (np.log(np.where(q > 0, q, 1.0)) - (s - ln_z[..., None])), 0.0)
    want = tau * tau * terms.sum(-1)
    tt = np.where(ids < 0, -np.inf, te.astype(np.float64) / tau)
    with np.errstate(invalid="ignore"):
        dt = np.where(q > 0, np.max(tt, -1, keepdims=True, initial=-np.inf) - tt, 0.0)
    # q is off by u (k + 20 + 3 dt) of itself and meets terms of size dt + |s| + |ln Z|; the sum over the entries adds k + 16
    far = np.max(dt, -1, initial=0.0)
    size = np.where(q > 0, q * (dt + np.where(np.isfinite(s), np.abs(s), 0.0)), 0.0).sum(-1) + np.abs(ln_z) + np.log(ids.shape[-1] + 1.0)
    bound = tau * tau * (ln_z_bound(t, ln_z, adds) + U * (2 * ids.shape[-1] + 40 + 3 * far) * size) + 4 * U * np.where(np.isfinite(want), np.abs(want), 0.0)
    close(loss, want, bound, "loss")


def check_distill_grad(tau, ids, te, x, lse, g, got, adds):
    """The gradient behind `distill`, whose normaliser `lse` it was given: tau g (softmax(x / tau) - q) of the logits
    themselves.  A normaliser below 2^14 is taken as it is, with what its rounding does to every probability."""
    t, ln_z, m = parts(x, tau)
    q = teacher_q(tau, ids, te)
    p = np.where(ln_z[..., None] == -np.inf, 0.0, np.exp(t - np.where(np.isfinite(ln_z), ln_z, 0.0)[..., None]))
    asked = np.zeros(x.shape)
    for r in range(x.shape[0]):
        for i in range(ids.shape[1]):
            if ids[r, i] >= 0:
                asked[r, ids[r, i]] += q[r, i]
    scale = (g.astype(np.float64) * tau)[..., None]
    want = np.where((q.sum(-1) > 0)[..., None], scale * (p - asked), 0.0)
    tt = np.where(ids < 0, -np.inf, te.astype(np.float64) / tau)
    with np.errstate(invalid="ignore"):
        far = np.max(np.where(q > 0, np.max(tt, -1, keepdims=True, initial=-np.inf) - tt, 0.0), -1, initial=0.0)[..., None]
    with np.errstate(invalid="ignore", over="ignore"):
        rounded = np.where(np.abs(lse) < 2.0 ** 14, U * (np.abs(m) + 3 * np.abs(lse)), 0.0)
    off = (ln_z_bound(t, ln_z, adds) + rounded)[..., None] + U * (16 + 5 * np.where(np.isfinite(t), np.abs(t), 0.0))
    bound = np.abs(scale) * (p * off + asked * U * (2 * ids.shape[-1] + 40 + 6 * far) + 2.0 ** -126)
    ty = "f16" if x.dtype == np.float16 else "f32"
    assert got.dtype == x.dtype
    close(got, want, bound * (1 + 2.0 ** -10) + half_step(want, ty), "gradient")


def rows_with_a_constant(g, rows, n, t, offset):
    """Logits around `offset`, in steps that the type holds there."""
    return (np.clip(g.normal(size=(rows, n)) * 6, -40, 40) + offset).astype(NP[t])


LOWEST = {"f16": np.float16(-65504), "f32": np.finfo(np.float32).min}
OFFSETS = [("f16", 1000.0), ("f16", -60000.0), ("f32", 1e4), ("f32", -3e6), ("f32", 2e8)]

__all__ = ["parts", "ln_z_bound", "check_log_probs", "check_distill", "check_distill_grad", "rows_with_a_constant", "LOWEST", "OFFSETS", "half_step"]
