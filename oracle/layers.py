"""Layer norm and affine + tanh + residual layers on packed jets, and their adjoints.

TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``).

Every function takes packed rows (``full`` points of Q coefficients, then value rows).
``magnitude=True`` evaluates the same formula with every term replaced by its absolute
value: a bound on each result's sum of term sizes, which rounding errors scale with.
"""

import numpy as np

from oracle import jets as J


def parts(x, dim, full):
    q = J.q(dim)
    return x[:full * q].reshape(full, q, x.shape[1]), x[full * q:]


def joined(block, value):
    return np.concatenate([block.reshape(-1, value.shape[1]), value])


def corr(a, s, dim):
    """Adjoint of ``b -> a * b`` at ``s``: ``out_k = sum_j a_j s_(j+k)`` on axis 1."""
    out = np.zeros(np.broadcast_shapes(a.shape, s.shape))
    for alpha, terms in enumerate(J.pairs(dim)):
        for j, k in terms:
            out[:, k] += a[:, j] * s[:, alpha]
    return out


def cauchy(a, b, dim):
    a, b = np.broadcast_arrays(a, b)
    return J.cauchy(a, b, dim, 3)


def rsqrt(v, dim, magnitude=False):
    """Series of ``v^(-1/2)``: ``r_0 (1 - n/2 + 3 n^2/8 - 5 n^3/16)``, ``n = v/v_0 - 1``."""
    r0 = v[:, :1] ** -0.5
    n = v * r0 * r0
    n[:, 0] = 0.0
    n2 = cauchy(n, n, dim)
    n3 = cauchy(n2, n, dim)
    sign = -1.0 if not magnitude else 1.0
    out = sign * 0.5 * n + 0.375 * n2 + sign * 0.3125 * n3
    out[:, 0] = 1.0
    return r0 * out


def layer_norm(x, gain, bias, eps, dim, full, magnitude=False):
    """``(out, stats)``."""
    block, value = parts(x, dim, full)
    size = np.abs if magnitude else (lambda a: a)
    mean, vmean = block.mean(2, keepdims=True), value.mean(1, keepdims=True)
    d, dv = block - mean, value - vmean
    v = cauchy(d, d, dim).mean(2, keepdims=True)
    v[:, 0] += eps
    vv = (dv * dv).mean(1, keepdims=True) + eps
    if magnitude:
        mean, vmean = np.abs(block).mean(2, keepdims=True), np.abs(value).mean(1, keepdims=True)
        d, dv = np.abs(block) + mean, np.abs(value) + vmean
        v0 = v[:, :1].copy()
        v = cauchy(d, d, dim).mean(2, keepdims=True)
        # relative to the true v_0: what an error in v becomes in r
        grow = 1.0 + v[:, :1] / v0
        v[:, :1] = v0
        r, rv = rsqrt(v, dim, True) * grow, vv ** -0.5 * (1.0 + (dv * dv).mean(1, keepdims=True) / vv)
    else:
        r, rv = rsqrt(v, dim), vv ** -0.5
    out = joined(cauchy(r, d, dim), rv * dv) * size(gain)
    zero = zero_rows(dim, full, len(value))
    out[zero] += size(bias)
    stats = np.stack([np.concatenate([mean.ravel(), vmean.ravel()]), np.concatenate([r.ravel(), rv.ravel()])], 1)
    return out, stats


def zero_rows(dim, full, value):
    q = J.q(dim)
    return np.concatenate([np.arange(full) * q, full * q + np.arange(value)]).astype(int)


def layer_norm_vjp(x, gain, stats, seed, skip, dim, full, magnitude=False):
    """``(d_value, d_gain, d_bias)``."""
    size = np.abs if magnitude else (lambda a: a)
    sign = 1.0 if magnitude else -1.0
    c = x.shape[1]
    x, stats, seed, gain = size(x), size(stats), size(seed), size(gain)
    (d, dv), (g, gv) = parts(x + sign * stats[:, :1], dim, full), parts(seed, dim, full)
    r, rv = parts(stats[:, 1:], dim, full)
    p, pv = corr(d, g, dim), dv * gv
    d_gain = (r * p).sum((0, 1)) + (rv * pv).sum(0)
    d_bias = g[:, 0].sum(0) + gv.sum(0)
    s = (p * gain).sum(2, keepdims=True)
    w = sign * corr(cauchy(cauchy(r, r, dim), r, dim), s, dim) / c
    wv = sign * rv ** 3 * (pv * gain).sum(1, keepdims=True) / c
    g, gv = g * gain, gv * gain
    dx = corr(r, g + sign * g.mean(2, keepdims=True), dim) + corr(d, w, dim)
    dxv = rv * (gv + sign * gv.mean(1, keepdims=True)) + dv * wv
    out = joined(dx, dxv)
    return out + (0.0 if skip is None else size(skip)), d_gain, d_bias


def affine(h, w, b, residual, dim, full, activation, magnitude=False):
    """``(out, activated, aux)``; without the activation the last two are ``None``."""
    if magnitude:
        h, w, b = np.abs(h), np.abs(w), np.abs(b)
        residual = None if residual is None else np.abs(residual)
    z = h @ w.T
    z[zero_rows(dim, full, len(h) - full * J.q(dim))] += b
    if not activation:
        return z if residual is None else z + residual, None, None
    block, value = parts(z, dim, full)
    if magnitude:
        # tanh and its derivatives up to the fourth are below 4 1/8; an error of z_0 reaches
        # the coefficients through the next derivative
        lift = 4.125 * (1.0 + block[:, :1])
        delta = block.copy()
        delta[:, 0] = 0.0
        d2 = cauchy(delta, delta, dim)
        a = joined(lift * (1.0 + delta + d2 + cauchy(d2, delta, dim)), 4.125 * (1.0 + value))
        a1 = np.concatenate([lift[:, 0], 4.125 * (1.0 + value)])
    else:
        ab, a1b = J.tanh_jet(block, dim)
        av, a1v = J.tanh_jet(value[:, None], dim)
        a, a1 = joined(ab, av[:, 0]), np.concatenate([a1b, a1v])
    return a if residual is None else a + residual, a, a1


def affine_vjp(h, w, activated, aux, seed, dim, full, magnitude=False):
    """``(d_hidden, d_weight, d_bias)``."""
    if magnitude:
        h, w, seed = np.abs(h), np.abs(w), np.abs(seed)
    g, gv = parts(seed, dim, full)
    if activated is not None:
        a, _ = parts(np.abs(activated) if magnitude else activated, dim, full)
        slope = cauchy(a, a, dim) * (1.0 if magnitude else -1.0)
        slope[:, 0] = aux[:full]
        g, gv = corr(slope, g, dim), gv * aux[full:]
    dz = joined(g, gv)
    return dz @ w, dz.T @ h, dz[zero_rows(dim, full, len(gv))].sum(0)
