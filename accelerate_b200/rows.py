"""Row operators: statistics along the innermost dimension and what is computed from them.

A ``fold`` reduces a row with one function and reads it once.  The functions here need several statistics of a row,
a selection from it, or the row again behind its statistics; as folds and maps each of them is a handful of passes
over memory.  They are foreign array functions (``Aforeign``, AST.hs:307-316): every one is *defined* in array code,
which is what a backend without an implementation runs (the oracle does), and this backend puts a hand-written kernel
behind the definition.

Rows are ``Half`` or ``Float``; statistics are ``Float`` whatever the rows' type.  ``sh`` is any outer shape: a vector
is one row, a matrix ``Z :. rows :. n`` many.  All arguments of a call have the same outer shape; the call fails with
"shape mismatch" otherwise.  Calls cannot be captured into a CUDA graph (their results come from the context's pool).
"""
from __future__ import annotations

import math
import numbers

from .language import (INT, Exp, _control, _avars, compute, cond, constant, exp, fold, from_index, from_integral, generate, index, is_nan, lift,
                       log, lor, land, lnot, max_, map_, shape_size, sqrt, tup, use, _as_list)

__all__ = ["logProbs", "distill", "distillGrad", "layerNorm", "layerNormGrad"]

_REAL = ("f16", "f32")
_NONE = 2 ** 31 - 1                      # an index behind every row
# distillGrad: a normaliser of this size is too coarse, and so near (relative) is the row's own
_NORMALISER_LARGE, _NORMALISER_STEPS = 2.0 ** 14, 3 * 2.0 ** -23


def _foreign(name, consts, fallback, *args):
    """``Aforeign`` under a name that the backend has an implementation for."""
    xs = [compute(use(x)) for x in args]
    ps = _avars(xs)
    rs = [compute(use(x)) for x in _as_list(fallback(*ps))]
    out = _control("aforeign", rs, [a.node for a in xs], [(ps, rs)], args=xs)
    out[0].node.foreign = (name, [float(c).hex() if isinstance(c, float) else str(int(c)) for c in consts])
    return out[0] if len(out) == 1 else tuple(out)


def _need(ok, message):
    if not ok:
        raise TypeError(message)


def _f(v):
    return Exp("f32", constant(float(v), "f32").sx)


def _wide(e):
    return e if e.ty == "f32" else Exp("f32", f"(prim tofloating {e.ty} f32 {e.sx})", e.deps)


def _as(e, ty):
    return e if e.ty == ty else Exp(ty, f"(prim tofloating {e.ty} {ty} {e.sx})", e.deps)


def _outer(ix, rank):
    return index(*[ix[d] for d in range(rank - 1)])


def _inner(outer, rank, j):
    return index(*[outer[d] for d in range(rank - 1)], j)


def _len(a):
    return a.shape[a.rank - 1]


_add = lambda a, b: a + b  # noqa: E731


def _normaliser(tau, xs):
    """ln sum e^(x / tau) of every row, its maximum m (0 for a row without an element above -inf), and
    z = sum e^((x - m) / tau) (0 for such a row)."""
    r = xs.rank
    m = compute(map_(lambda v: cond(v.eq(_f(-math.inf)), _f(0), v), fold(max_, _f(-math.inf), map_(_wide, xs))))
    z = compute(fold(_add, _f(0), generate(xs.shape, lambda ix: exp((_wide(xs[ix]) - m[_outer(ix, r)]) / _f(tau)))))
    lse = compute(generate(m.shape, lambda o: m[o] / _f(tau) + log(z[o])))
    return lse, m, z


def _log_probability(x, tau, m, z):
    """(x - m) / tau - ln z: the differences inside the row, whatever its elements' size (the normaliser, one Float, has
    lost them at 1e8).  A row without an element above -inf gives none of its elements any probability."""
    return cond(z.eq(_f(0)), _f(-math.inf), (x - m) / _f(tau) - log(z))


def _better(a, b):
    """Whether (value, index) ``a`` stands before ``b``: larger first (a NaN before everything), then the lower index."""
    na, nb = is_nan(a[0]), is_nan(b[0])
    value = lor(land(na, lnot(nb)), land(land(lnot(na), lnot(nb)), a[0] > b[0]))
    same = lor(land(na, nb), land(land(lnot(na), lnot(nb)), a[0].eq(b[0])))
    return lor(value, land(same, a[1] < b[1]))


def logProbs(k, tokens, logits):
    """Log probabilities of given tokens, with entropy and the ``k`` top alternatives, of every row of ``logits``.

    ``logProbs :: Int -> Array sh Int32 -> Array (sh:.Int) t -> (Array sh (Float, Float, Float), Array (sh:.Int) (Int32, Float))``

    For a row x with lse = ln sum e^x the first result holds (x_token - lse, lse, entropy), the second the indices and
    log probabilities of the k largest logits, in falling order, equal ones by rising index.  k goes from 0 to 128;
    tokens may be Int32 or Int.  Log probabilities come from the distances to the row's largest logit, not from the rounded
    lse: they are as good for logits around 1e8 as around 0.

    A negative token is no token: its log probability is 0.  A token behind the row's end is an error ("index out of
    bounds", reported by the next download or sync).  Logits of -inf are masked: probability 0, and no part of the entropy.  A row
    with nothing else has lse and log probabilities of -inf and entropy 0.  NaN and +inf make a row's numbers NaN;
    among the alternatives a NaN comes first.  A row shorter than k ends in alternatives (-1, -inf)."""
    tokens, logits = use(tokens), use(logits)
    _need(isinstance(k, numbers.Integral) and 0 <= k <= 128, "logProbs: the number of alternatives is a whole number from 0 to 128")
    _need(logits.rank >= 1 and logits.elt in _REAL, "logProbs: the logits must be an array of Half or Float of rank 1 or more")
    _need(tokens.rank == logits.rank - 1 and tokens.elt in ("i32", "i64"), "logProbs: the given tokens must be Int32 or Int, one per row")

    k = int(k)

    def definition(tok, xs):
        r = xs.rank
        lse, m, z = _normaliser(1.0, xs)

        def spread(ix):
            d = _wide(xs[ix]) - m[_outer(ix, r)]
            return cond(exp(d).eq(_f(0)), _f(0), exp(d) * d)
        w = compute(fold(_add, _f(0), generate(xs.shape, spread)))

        def stats(o):
            t = from_integral(tok[o], INT)
            logp = cond(t < 0, _f(0), _log_probability(_wide(xs[_inner(o, r, t)]), 1.0, m[o], z[o]))
            return tup(logp, lse[o], cond(z[o].eq(_f(0)), _f(0), log(z[o]) - w[o] / z[o]))
        best, last = [], None
        for _ in range(k):
            # the best element behind the one before it in the order
            def candidate(ix, last=last):
                e = tup(_wide(xs[ix]), from_integral(ix[r - 1], "i32"))
                return e if last is None else cond(_better(last[_outer(ix, r)], e), e, tup(_f(-math.inf), constant(_NONE, "i32")))
            last = compute(fold(lambda a, b: cond(_better(a, b), a, b), tup(_f(-math.inf), constant(_NONE, "i32")), generate(xs.shape, candidate)))
            best.append(last)

        def alternative(ix):
            o = _outer(ix, r)
            e = lift((-math.inf, _NONE), ("f32", "i32"))
            for j in reversed(range(k)):
                e = cond(ix[r - 1].eq(lift(j, INT)), best[j][o], e)
            there = e[1].ne(constant(_NONE, "i32"))
            return tup(cond(there, e[1], constant(-1, "i32")), cond(there, _log_probability(e[0], 1.0, m[o], z[o]), _f(-math.inf)))
        outer = _outer(xs.shape, r)
        return generate(outer, stats), generate(_inner(outer, r, lift(k, INT)), alternative)
    return _foreign("b200.logProbs", [k], definition, tokens, logits)


def _teacher(tau, ids, ts):
    """The teacher's distribution over its entries: maximum and sum of every list (sum 0: no entry), and e^((t - max)/tau)."""
    r = ids.rank

    def there(ix):
        return cond(ids[ix] < constant(0, "i32"), _f(-math.inf), _wide(ts[ix]))
    m = compute(map_(lambda v: cond(v.eq(_f(-math.inf)), _f(0), v), fold(max_, _f(-math.inf), generate(ids.shape, there))))
    e = lambda ix: exp((there(ix) - m[_outer(ix, r)]) / _f(tau))  # noqa: E731
    total = compute(fold(_add, _f(0), generate(ids.shape, e)))
    return m, total, e


def _check_distill(what, tau, ids, teacher, student):
    _need(isinstance(tau, numbers.Real) and 1e-4 <= tau <= 1e4, f"{what}: the temperature must lie between 1e-4 and 1e4")
    _need(student.rank >= 1 and student.elt in _REAL, f"{what}: the student's logits must be an array of Half or Float of rank 1 or more")
    _need(ids.rank == student.rank and ids.elt == "i32", f"{what}: the teacher's tokens must be Int32, one list per row")
    _need(teacher.rank == student.rank and teacher.elt in _REAL, f"{what}: the teacher's logits must be Half or Float, one list per row")


def distill(tau, ids, teacher, student):
    """Distillation loss of every row of a student's logits against a teacher's top entries.

    ``distill :: Float -> Array (sh:.Int) Int32 -> Array (sh:.Int) t' -> Array (sh:.Int) t -> (Array sh Float, Array sh Float)``

    ``ids`` and ``teacher`` hold a few tokens per row (at most 4096) and the teacher's logits (or log probabilities) for them, as
    ``logProbs`` yields them.  With q the softmax of teacher / tau over the entries and p that of student / tau over the
    whole row, the loss is tau^2 sum q (ln q - ln p).  The second result is ln sum e^(student / tau), which
    ``distillGrad`` takes.

    A negative id is no entry; so is a logit of -inf.  A row without entries has loss 0.  An id that occurs twice counts
    twice.  An id behind the row's end is an error ("index out of bounds", reported by the next download or sync).  A student
    that gives an entry no probability at all has loss +inf."""
    ids, teacher, student = use(ids), use(teacher), use(student)
    _check_distill("distill", tau, ids, teacher, student)

    def definition(ids, ts, xs):
        r = xs.rank
        lse, top, z = _normaliser(tau, xs)
        m, total, e = _teacher(tau, ids, ts)

        def term(ix):
            o = _outer(ix, r)
            w = e(ix) / total[o]
            lp = _log_probability(_wide(xs[_inner(o, r, from_integral(ids[ix], INT))]), tau, top[o], z[o])
            return cond(ids[ix] < constant(0, "i32"), _f(0),
                        cond(e(ix).eq(_f(0)), _f(0), w * ((_wide(ts[ix]) - m[o]) / _f(tau) - log(total[o]) - lp)))
        loss = fold(_add, _f(0), generate(ids.shape, term))
        return map_(lambda v: _f(tau) * _f(tau) * v, loss), lse
    return _foreign("b200.distill", [float(tau)], definition, ids, teacher, student)


def distillGrad(tau, ids, teacher, student, normaliser, gradient):
    """Gradient of ``distill``'s loss with respect to the student's logits.

    ``distillGrad :: Float -> Array (sh:.Int) Int32 -> Array (sh:.Int) t' -> Array (sh:.Int) t -> Array sh Float -> Array sh Float -> Array (sh:.Int) t``

    ``normaliser`` is ``distill``'s second result, ``gradient`` that of the whole with respect to every row's loss; the
    result is gradient tau (p - q), p = e^(student / tau - normaliser), rounded once to the student's type.

    The normaliser is one Float, and half a step of it is a relative error of every p: 2^-24 of its size, so up to 2^-10
    (with what ``distill`` rounded on the way) below 2^14.  From 2^14 on, where logits this large, small temperatures or rows
    of the type's lowest value lead, p comes from the row itself, p = e^((student - max) / tau) / Z, as long as the given
    normaliser is the row's own, up to three steps of it; another one (that of a longer row, of which this is a part) is taken
    as it is."""
    ids, teacher, student, normaliser, gradient = use(ids), use(teacher), use(student), use(normaliser), use(gradient)
    _check_distill("distillGrad", tau, ids, teacher, student)
    for a in (normaliser, gradient):
        _need(a.rank == student.rank - 1 and a.elt == "f32", "distillGrad: normaliser and gradient must be Float, one per row")

    def definition(ids, ts, xs, lse, g):
        r = xs.rank
        _, total, e = _teacher(tau, ids, ts)
        own, top, z = _normaliser(tau, xs)

        def share(ix):                   # sh :. n :. k: what entry k asks for element j
            o, j = index(*[ix[d] for d in range(r - 1)]), ix[r - 1]
            at = _inner(o, r, ix[r])
            return cond(from_integral(ids[at], INT).eq(j), e(at), _f(0))
        asked = compute(fold(_add, _f(0), generate(index(*[xs.shape[d] for d in range(r)], _len(ids)), share)))

        def one(ix):
            o = _outer(ix, r)
            size = abs(lse[o])
            close = lor(lse[o].eq(own[o]), abs(lse[o] - own[o]) <= size * _f(_NORMALISER_STEPS))
            from_row = land(land(size >= _f(_NORMALISER_LARGE), z[o] > _f(0)), close)
            p = cond(_wide(xs[ix]).eq(_f(-math.inf)), _f(0),
                     cond(from_row, exp((_wide(xs[ix]) - top[o]) / _f(tau)) / z[o], exp(_wide(xs[ix]) / _f(tau) - lse[o])))
            return _as(cond(total[o].eq(_f(0)), _f(0), g[o] * _f(tau) * (p - asked[ix] / total[o])), xs.elt)
        return generate(xs.shape, one)
    return _foreign("b200.distillGrad", [float(tau)], definition, ids, teacher, student, normaliser, gradient)


def layerNorm(eps, gamma, beta, xs):
    """Layer norm of every row: ((x - mean) * rstd * gamma + beta, (mean, rstd)), rstd = 1 / sqrt(var + eps) with the
    biased variance.

    ``layerNorm :: Float -> Vector g -> Vector g -> Array (sh:.Int) t -> (Array (sh:.Int) t, Array sh (Float, Float))``

    gamma and beta have the rows' length and either the rows' type or Float.  The result is rounded once to the rows' type.
    eps may be 0 (a constant row is then NaN).  Rows of length zero have NaN statistics."""
    gamma, beta, xs = use(gamma), use(beta), use(xs)
    _need(isinstance(eps, numbers.Real) and 0 <= eps <= 3.4e38, "layerNorm: epsilon must be finite and not negative")
    _need(xs.rank >= 1 and xs.elt in _REAL, "layerNorm: the rows must be an array of Half or Float of rank 1 or more")
    _need(gamma.rank == 1 and gamma.elt in (xs.elt, "f32") and beta.rank == 1 and beta.elt == gamma.elt,
          "layerNorm: gamma and beta must be vectors of the rows' type or of Float")

    def definition(ga, be, xs):
        r = xs.rank
        n = Exp("f32", f"(prim fromintegral i64 f32 {_len(xs).sx})", _len(xs).deps)
        mean = compute(map_(lambda s: s / n, fold(_add, _f(0), map_(_wide, xs))))

        def square(ix):
            d = _wide(xs[ix]) - mean[_outer(ix, r)]
            return d * d
        rstd = compute(map_(lambda s: _f(1) / sqrt(s / n + _f(eps)), fold(_add, _f(0), generate(xs.shape, square))))

        def one(ix):
            o, j = _outer(ix, r), index(ix[r - 1])
            return _as((_wide(xs[ix]) - mean[o]) * rstd[o] * _wide(ga[j]) + _wide(be[j]), xs.elt)
        return generate(xs.shape, one), generate(mean.shape, lambda o: tup(mean[o], rstd[o]))
    return _foreign("b200.layerNorm", [float(eps)], definition, gamma, beta, xs)


def layerNormGrad(gamma, xs, stats, dys):
    """Gradients of ``layerNorm`` with respect to the rows, gamma and beta.

    ``layerNormGrad :: Vector g -> Array (sh:.Int) t -> Array sh (Float, Float) -> Array (sh:.Int) t -> (Array (sh:.Int) t, Vector g, Vector g)``

    ``stats`` is ``layerNorm``'s second result, ``dys`` the gradient with respect to its first.  The weights' gradients
    are sums over all rows in Float, in an order that does not change from call to call, rounded once to gamma's type."""
    gamma, xs, stats, dys = use(gamma), use(xs), use(stats), use(dys)
    _need(xs.rank >= 1 and xs.elt in _REAL, "layerNormGrad: the rows must be an array of Half or Float of rank 1 or more")
    _need(gamma.rank == 1 and gamma.elt in (xs.elt, "f32"), "layerNormGrad: gamma must be a vector of the rows' type or of Float")
    _need(stats.rank == xs.rank - 1 and stats.elt == ("f32", "f32"), "layerNormGrad: the statistics must be pairs of Floats, one per row")
    _need(dys.rank == xs.rank and dys.elt == xs.elt, "layerNormGrad: the gradient must have the rows' type and rank")

    def definition(ga, xs, st, dys):
        r = xs.rank
        n = Exp("f32", f"(prim fromintegral i64 f32 {_len(xs).sx})", _len(xs).deps)
        hat = lambda ix: (_wide(xs[ix]) - st[_outer(ix, r)][0]) * st[_outer(ix, r)][1]  # noqa: E731
        a = lambda ix: _wide(dys[ix]) * _wide(ga[index(ix[r - 1])])  # noqa: E731
        ma = compute(map_(lambda s: s / n, fold(_add, _f(0), generate(xs.shape, a))))
        mb = compute(map_(lambda s: s / n, fold(_add, _f(0), generate(xs.shape, lambda ix: a(ix) * hat(ix)))))

        def one(ix):
            o = _outer(ix, r)
            return _as(st[o][1] * (a(ix) - ma[o] - hat(ix) * mb[o]), xs.elt)
        outer = _outer(xs.shape, r)
        rows = shape_size(outer)

        def over_rows(f):                # n :. rows, folded
            def at(ix):
                return f(_inner(from_index(outer, ix[1]), r, ix[0]))
            return map_(lambda s: _as(s, ga.elt), fold(_add, _f(0), generate(index(_len(xs), rows), at)))
        return generate(xs.shape, one), over_rows(lambda ix: _wide(dys[ix]) * hat(ix)), over_rows(lambda ix: _wide(dys[ix]))
    return _foreign("b200.layerNormGrad", [], definition, gamma, xs, stats, dys)
