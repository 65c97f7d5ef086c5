"""Inputs and rounding bounds of the layer operators' tests."""

import numpy as np

from oracle import jets as J
from oracle import layers as L

#: half a unit in the last place, relative: one FP64 rounding
HALF = 2.0 ** -53


def jets(rng, dim, full, value, channels):
    """Packed rows whose coefficients fade with their order, values off zero."""
    x = rng.normal(size=(full * J.q(dim) + value, channels)) * 0.8 + 0.1
    fade = np.array([0.7 ** sum(a) for a in J.basis(dim)])
    x[:full * J.q(dim)] *= np.tile(fade, full)[:, None]
    return x


def norm_case(dim, full, value, channels, seed=0, skip=True):
    rng = np.random.default_rng(seed + 7 * channels + full)
    return dict(x=jets(rng, dim, full, value, channels), gain=1 + 0.1 * rng.normal(size=channels),
                bias=0.1 * rng.normal(size=channels), seed=jets(rng, dim, full, value, channels),
                skip=jets(rng, dim, full, value, channels) if skip else None)


def affine_case(dim, full, value, cin, cout, seed=0):
    rng = np.random.default_rng(seed + 7 * cin + cout + full)
    return dict(h=jets(rng, dim, full, value, cin), w=rng.normal(size=(cout, cin)) / np.sqrt(cin),
                b=0.1 * rng.normal(size=cout), residual=jets(rng, dim, full, value, cout),
                seed=jets(rng, dim, full, value, cout))


def worst(actual, expected, magnitude, roundings):
    """max |a - e| over the bound: every result is a sum of products whose factors carry at most
    ``roundings`` half units each between them; ``magnitude`` is the sum of the products' sizes."""
    a, e = np.asarray(actual, dtype=np.float64), np.asarray(expected)
    assert a.shape == e.shape, (a.shape, e.shape)
    assert np.isfinite(a).all()
    return float(np.max(np.abs(a - e) / (roundings * HALF * magnitude + 1e-300), initial=0.0))


# Roundings between the inputs and an output, both sides of the comparison together (hence the
# factor 2).  A sum of n terms rounds each term at most n times; a truncated product has at
# most T = 84 pairs, a series of r three factors of v, and v, mean and the adjoint's sums run
# over the channels.
def norm_roundings(channels):
    return 2 * (4 * (channels + 84) + 84)


def norm_vjp_roundings(channels, points=0):
    return 2 * (4 * 84 + 2 * channels + points)


def affine_roundings(cin):
    return 2 * (4 * (cin + 4) + 2 * 84)


def affine_vjp_roundings(terms):
    return 2 * (2 * 84 + 4 + terms)
