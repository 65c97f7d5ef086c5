"""The per-layer operators of a pre-norm residual network on packed jets, and the cases they are timed at.

Rows are packed as ``PackedLayout`` packs them: Q coefficients for each full point
(10 in 2-D, 20 in 3-D, factorial-normalized, |alpha| <= 3), then one row for each value
point; channels are contiguous and everything is FP64.  Four operators:

* ``norm``        layer norm over the channels, propagated through the jets
* ``norm_vjp``    its adjoint: input (with the skip connection's share), gain and bias gradients
* ``affine``      ``H W^T + b`` with the tanh jet and the residual added in its epilogue
* ``affine_vjp``  its adjoint: input, weight and bias gradients

``own`` false runs them as elementary torch operations, ``own`` true as the framework's calls.
"""

from itertools import product

import torch

own = False

EPS = 1e-5
#: most values of one packed tensor and most products of one affine layer that a drawn case may have:
#: those of the largest listed case
MOST_VALUES, MOST_PRODUCTS = 671_744 * 128, 671_744 * 128 * 128


def listed():
    return [
        # one collocation point through a layer norm of a 64-wide net: the launch's latency
        dict(name="norm_point", op="norm", dim=2, full=1, value=0, cin=64),
        # the 64-wide Kovasznay configuration's points (16,384 interior, 4,096 boundary values)
        dict(name="norm_2d_64", op="norm", dim=2, full=16384, value=4096, cin=64),
        # a space-time shard of the 128-wide configuration (an eighth of 262,144 + 65,536 points)
        dict(name="norm_3d_128", op="norm", dim=3, full=32768, value=8192, cin=128),
        # the adjoint inside a residual block: the skip connection's gradient joins on the way
        dict(name="norm_vjp_2d_64", op="norm_vjp", dim=2, full=16384, value=4096, cin=64, skip=True),
        # an uneven space-time set and a width that no tile divides, the net's first norm (no skip)
        dict(name="norm_vjp_3d_100", op="norm_vjp", dim=3, full=4099, value=1031, cin=100, skip=False),
        # answering: values alone on the 201 x 201 acceptance grid, nothing kept for a backward pass
        dict(name="affine_grid", op="affine", dim=2, full=0, value=40401, cin=64, cout=64, tanh=True,
             residual=True, keep=False),
        # training a 64-wide residual layer on the Kovasznay configuration
        dict(name="affine_2d_64", op="affine", dim=2, full=16384, value=4096, cin=64, cout=64, tanh=True,
             residual=True, keep=True),
        # the 128-wide configuration (65,536 + 16,384 points)
        dict(name="affine_2d_128", op="affine", dim=2, full=65536, value=16384, cin=128, cout=128, tanh=True,
             residual=True, keep=True),
        # uneven space-time points between two uneven widths, no residual
        dict(name="affine_3d_100_60", op="affine", dim=3, full=8193, value=2049, cin=100, cout=60, tanh=True,
             residual=False, keep=True),
        # the adjoints of the two trained layers
        dict(name="affine_vjp_2d_64", op="affine_vjp", dim=2, full=16384, value=4096, cin=64, cout=64, tanh=True),
        dict(name="affine_vjp_2d_128", op="affine_vjp", dim=2, full=65536, value=16384, cin=128, cout=128, tanh=True),
        # the output layer of the smallest configuration (2,048 + 512 points): three fields, no tanh
        dict(name="affine_vjp_tail", op="affine_vjp", dim=2, full=2048, value=512, cin=64, cout=3, tanh=False),
    ]


def draw(rng):
    """A case of the same ranges: 1 to 65,536 full points, up to a quarter as many values (or values alone), widths 8 to 192."""
    def spread(low, high):
        return int(round(low * (high / low) ** rng.random()))

    op = rng.choice(["norm", "norm_vjp", "affine", "affine", "affine_vjp", "affine_vjp"])
    dim = rng.choice([2, 2, 3])
    q = 10 if dim == 2 else 20
    cin, cout = spread(8, 192), spread(8, 192)
    if rng.random() < 0.25:
        cin = cout = rng.choice([32, 64, 128])
    if op == "affine_vjp" and rng.random() < 0.2:
        cout = 3
    width = max(cin, cout) if op.startswith("affine") else cin
    most = MOST_VALUES // width
    if op.startswith("affine"):
        most = min(most, MOST_PRODUCTS // (cin * cout))
    full = spread(1, max(1, min(65536, int(most / (q + 0.25)))))
    value = int(full * rng.random() / 4)
    case = dict(op=op, dim=dim, full=full, value=value, cin=cin)
    if op == "norm_vjp":
        case["skip"] = rng.random() < 0.7
    if op.startswith("affine"):
        case.update(cout=cout, tanh=cout != 3 and rng.random() < 0.8)
    if op == "affine":
        case.update(residual=rng.random() < 0.6, keep=rng.random() < 0.8)
        if not case["keep"]:
            case.update(full=0, value=spread(1, min(most, 65536)))
    return case


def basis(dim):
    """Multi-indices of total degree at most three, sorted by degree and then lexicographically."""
    return sorted((a for a in product(range(4), repeat=dim) if sum(a) <= 3), key=lambda a: (sum(a), a))


def tables(dim, device):
    """The truncated product's pairs: indices j, k and the index of their sum, with 0/1 matrices that add by the sum and by k."""
    order = basis(dim)
    at = {a: i for i, a in enumerate(order)}
    rows = [(j, k, at.get(tuple(x + y for x, y in zip(a, b)), -1)) for j, a in enumerate(order)
            for k, b in enumerate(order)]
    j, k, s = (torch.tensor(v, device=device) for v in zip(*[r for r in rows if r[2] >= 0]))
    which = torch.arange(len(order), device=device)[:, None]
    return {"j": j, "k": k, "s": s, "by_sum": (which == s).double(), "by_k": (which == k).double()}


def times(a, b, t):
    """Truncated product of [points, Q, channels] jets."""
    return t["by_sum"] @ (a[:, t["j"]] * b[:, t["k"]])


def against(a, b, t):
    """The product's adjoint: out_k = sum_j a_j b_(j+k)."""
    return t["by_k"] @ (a[:, t["j"]] * b[:, t["s"]])


def split(x, s):
    """The full points' [points, Q, channels] and the value rows."""
    q = len(s["t"]["by_k"])
    n = s["full"] * q
    return x[:n].view(s["full"], q, x.shape[1]), x[n:]


def joined(full, value):
    return torch.cat((full.reshape(-1, value.shape[1]), value))


def sech2(z):
    r = torch.exp(-z.abs())
    return (2 * r / (1 + r * r)) ** 2


def tanh_jet(z, t):
    z0 = z[:, :1]
    h, a1 = torch.tanh(z0), sech2(z0)
    d = torch.cat((torch.zeros_like(z0), z[:, 1:]), 1)
    d2 = times(d, d, t)
    out = a1 * d - h * a1 * d2 + a1 * (h * h - 1 / 3) * times(d2, d, t)
    return torch.cat((h, out[:, 1:]), 1), a1[:, 0]


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(int(seed))
    dim, full, value, cin = case["dim"], case["full"], case["value"], case["cin"]
    cout = case.get("cout", cin)
    q = len(basis(dim))

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, dtype=torch.float64, device="cuda") * scale

    def jets(channels):
        # values of order one, coefficients that get smaller with their order as a net's do
        x = normal(full * q + value, channels, scale=0.8) + 0.1
        fade = torch.tensor([0.7 ** sum(a) for a in basis(dim)], dtype=torch.float64, device="cuda")
        x[:full * q].view(full, q, channels).mul_(fade[:, None])
        return x

    s = {"op": case["op"], "dim": dim, "full": full, "value": value, "t": tables(dim, "cuda")}
    if case["op"] in ("norm", "norm_vjp"):
        s.update(x=jets(cin), gain=1 + normal(cin, scale=0.1), bias=normal(cin, scale=0.1))
        if case["op"] == "norm_vjp":
            s.update(seed=jets(cin), skip=jets(cin) if case["skip"] else None)
            s["stats"] = statistics(s)
        return s
    s.update(x=jets(cin), weight=normal(cout, cin, scale=cin ** -0.5), bias=normal(cout, scale=0.1), tanh=case["tanh"])
    if case["op"] == "affine":
        s.update(residual=jets(cout) if case["residual"] else None, keep=case["keep"])
    else:
        s["seed"] = jets(cout)
        s["activated"] = s["aux"] = None
        if s["tanh"]:
            _, s["activated"], s["aux"] = affine({**s, "residual": None})
    return s


def statistics(s):
    """Mean and reciprocal deviation of every row, as the forward pass hands them to the backward pass."""
    t = s["t"]
    full, value = split(s["x"], s)
    mean, d = full.mean(2), full - full.mean(2, keepdim=True)
    v = times(d, d, t).mean(2, keepdim=True)
    r0 = (v[:, :1] + EPS) ** -0.5
    n = torch.cat((torch.zeros_like(r0), v[:, 1:] * r0 * r0), 1)
    n2 = times(n, n, t)
    one = (torch.arange(len(t["by_k"]), device=v.device) == 0).double()[None, :, None]
    r = r0 * (one - n / 2 + n2 * 0.375 - times(n2, n, t) * 0.3125)
    vm = value.mean(1)
    vr = ((value - vm[:, None]).square().mean(1) + EPS) ** -0.5
    return torch.stack((torch.cat((mean.reshape(-1), vm)), torch.cat((r.reshape(-1), vr))), 1)


def norm(s):
    t, stats = s["t"], statistics(s)
    full, value = split(s["x"] - stats[:, :1], s)
    r, rv = split(stats[:, 1:], s)
    out = joined(times(r.expand_as(full), full, t), value * rv) * s["gain"]
    rows = torch.cat((torch.arange(s["full"], device=out.device) * len(t["by_k"]),
                      torch.arange(s["full"] * len(t["by_k"]), len(out), device=out.device)))
    out[rows] += s["bias"]
    return out, stats


def norm_vjp(s):
    t, stats, c = s["t"], s["stats"], s["x"].shape[1]
    d, dv = split(s["x"] - stats[:, :1], s)
    r, rv = split(stats[:, 1:], s)
    seed, seed_v = split(s["seed"], s)
    d_bias = seed[:, 0].sum(0) + seed_v.sum(0)
    d_gain = (seed * times(r.expand_as(d), d, t)).sum((0, 1)) + (seed_v * dv * rv).sum(0)
    g, gv = seed * s["gain"], seed_v * s["gain"]
    dr = against(d, g, t).sum(2, keepdim=True)
    dvar = against(times(times(r, r, t), r, t) * -0.5, dr, t)
    dx = against(r.expand_as(g), g - g.mean(2, keepdim=True), t) + against(d, dvar.expand_as(d), t) * (2 / c)
    dr_v = (dv * gv).sum(1, keepdim=True)
    dx_v = rv * (gv - gv.mean(1, keepdim=True)) - dv * rv ** 3 * dr_v / c
    out = joined(dx, dx_v)
    return (out if s["skip"] is None else out + s["skip"]), d_gain, d_bias


def affine(s):
    z = s["x"] @ s["weight"].T
    full, value = split(z, s)
    full[:, 0] += s["bias"]
    value += s["bias"]
    if not s["tanh"]:
        return (z if s["residual"] is None else z + s["residual"]), None, None
    a, a1 = tanh_jet(full, s["t"])
    h, aux = joined(a, torch.tanh(value)), torch.cat((a1, sech2(value)))
    return (h if s["residual"] is None else h + s["residual"]), h, aux


def affine_vjp(s):
    dz, dz_v = split(s["seed"], s)
    if s["tanh"]:
        a, _ = split(s["activated"], s)
        aux, aux_v = s["aux"][:s["full"]], s["aux"][s["full"]:]
        f = torch.cat((aux[:, None], -times(a, a, s["t"])[:, 1:]), 1)
        dz, dz_v = against(f, dz, s["t"]), dz_v * aux_v
    z = joined(dz, dz_v)
    return z @ s["weight"], z.T @ s["x"], dz[:, 0].sum(0) + dz_v.sum(0)


def run(s):
    if own:
        return calls(s)
    if s["op"] == "norm":
        return norm(s)
    if s["op"] == "norm_vjp":
        return norm_vjp(s)
    if s["op"] == "affine_vjp":
        return affine_vjp(s)
    out, h, aux = affine(s)
    return (out, h, aux) if s["keep"] and s["tanh"] else out


def calls(s):
    from flashns_b200.jet_packed import PackedLayout
    from flashns_b200.native import NativeCUDA
    native, layout = NativeCUDA(), PackedLayout(s["full"], s["value"], s["dim"])
    if s["op"] == "norm":
        return native.layer_norm(layout, s["x"], s["gain"], s["bias"], eps=EPS)
    if s["op"] == "norm_vjp":
        return native.layer_norm_vjp(layout, s["x"], s["gain"], s["stats"], s["seed"], skip=s["skip"])
    if s["op"] == "affine":
        if s["tanh"]:
            return native.affine_activation(layout, s["x"], s["weight"], s["bias"], residual=s["residual"],
                                            keep=s["keep"])
        return native.affine(layout, s["x"], s["weight"], s["bias"], residual=s["residual"])
    if s["tanh"]:
        return native.affine_activation_vjp(layout, s["x"], s["weight"], s["activated"], s["aux"], s["seed"])
    return native.affine_vjp(layout, s["x"], s["weight"], s["seed"])


def work(case):
    q, t = (10, 35) if case["dim"] == 2 else (20, 84)
    full, value, cin = case["full"], case["value"], case["cin"]
    rows, points, cout = full * q + value, full + value, case.get("cout", case["cin"])
    if case["op"] == "norm":  # centring, its square, the product with r
        return {"bytes": 8 * (2 * rows * cin + 2 * rows + 2 * cin),
                "flops": (full * (3 * t + 3 * q) + value * 7) * cin}
    if case["op"] == "norm_vjp":  # two correlations of D, one of r, the means
        return {"bytes": 8 * ((3 + case["skip"]) * rows * cin + 2 * rows + 3 * cin),
                "flops": (full * (6 * t + 6 * q) + value * 14) * cin}
    pointwise = (full * 4 * t + value * 4) * cout if case["tanh"] else 0
    if case["op"] == "affine":
        kept = rows * cout * bool(case["residual"]) + points * cout if case["keep"] and case["tanh"] else 0
        return {"bytes": 8 * (rows * cin + rows * cout * (1 + case["residual"]) + kept + cout * (cin + 1)),
                "flops": 2 * rows * cin * cout + pointwise}
    kept = rows * cout + points * cout if case["tanh"] else 0
    return {"bytes": 8 * (2 * rows * cin + rows * cout + kept + cout * (2 * cin + 1)),
            "flops": 4 * rows * cin * cout + pointwise}


# ---- from the definitions: jets as polynomials, kept as {multi-index: [points, channels]}

def polynomial(x, dim, full, value):
    order = basis(dim)
    block = x[:full * len(order)].view(full, len(order), x.shape[1])
    return {a: block[:, i] for i, a in enumerate(order)}, {(0,) * dim: x[full * len(order):]}


def rows_of(poly, values, dim, channels):
    order = basis(dim)
    block = torch.stack([poly[a].expand(-1, channels) for a in order], 1)
    return torch.cat((block.reshape(-1, channels), values[(0,) * dim].expand(-1, channels)))


def cut_product(a, b):
    out = {}
    for i, x in a.items():
        for j, y in b.items():
            k = tuple(u + v for u, v in zip(i, j))
            if sum(k) <= 3 and k in a:
                out[k] = out[k] + x * y if k in out else x * y
    return out


def normalized(p):
    """(mean, reciprocal deviation, normalized polynomial): the series of (v + eps)^(-1/2) by Newton's iteration."""
    mean = {k: v.mean(1, keepdim=True) for k, v in p.items()}
    d = {k: v - mean[k] for k, v in p.items()}
    var = {k: v.mean(1, keepdim=True) for k, v in cut_product(d, d).items()}
    zero = next(k for k in p if sum(k) == 0)
    var[zero] = var[zero] + EPS
    r = {k: torch.zeros_like(v) for k, v in var.items()}
    r[zero] = 1 / torch.sqrt(var[zero])
    for _ in range(2 if len(p) > 1 else 0):  # the right order doubles each time: 0, 1, 3
        e = {k: -v / 2 for k, v in cut_product(var, cut_product(r, r)).items()}
        e[zero] = e[zero] + 1.5
        r = cut_product(r, e)
    return mean, r, cut_product(r, d)


def tanh_series(p):
    """tanh of a polynomial, degree by degree, from E h = (1 - h^2) E z with E x^k = |k| x^k."""
    zero = next(k for k in p if sum(k) == 0)
    slope = 1 / torch.cosh(p[zero]).square()
    h = {zero: torch.tanh(p[zero])}
    for degree in range(1, 4 if len(p) > 1 else 1):
        lower = {}
        for i, x in h.items():
            for j, y in h.items():
                k = tuple(u + v for u, v in zip(i, j))
                if 0 < sum(k) < degree:
                    lower[k] = lower[k] - x * y if k in lower else -x * y
        lower[zero] = slope
        for k in [k for k in p if sum(k) == degree]:
            terms = [lower[i] * p[j] * sum(j) for i in lower for j in p
                     if sum(j) and tuple(u + v for u, v in zip(i, j)) == k]
            h[k] = torch.stack(terms).sum(0) / degree
    return h, slope


def exact(case, seed):
    s = prepare(case, seed)
    dim, full, value, x = case["dim"], case["full"], case["value"], s["x"]
    zero = (0,) * dim
    if case["op"] in ("norm", "norm_vjp"):
        back = case["op"] == "norm_vjp"
        x, gain, bias = (v.clone().requires_grad_(back) for v in (x, s["gain"], s["bias"]))
        with torch.set_grad_enabled(back):
            parts = [normalized(p) for p in polynomial(x, dim, full, value)]
            outs = [{k: v * gain + (bias if k == zero else 0) for k, v in y.items()} for _, _, y in parts]
            out = rows_of(outs[0], outs[1], dim, x.shape[1])
        if not back:
            return out, torch.cat([rows_of(parts[0][i], parts[1][i], dim, 1) for i in (0, 1)], 1)
        d_x, d_gain, d_bias = torch.autograd.grad(out, (x, gain, bias), s["seed"])
        return (d_x + s["skip"] if case["skip"] else d_x), d_gain, d_bias
    if case["op"] == "affine":
        parts = polynomial(torch.einsum("rk,ck->rc", x, s["weight"]), dim, full, value)
        parts = [{k: v + s["bias"] if k == zero else v for k, v in p.items()} for p in parts]
        aux = None
        if case["tanh"]:
            parts, aux = zip(*[tanh_series(p) for p in parts])
        h = rows_of(parts[0], parts[1], dim, case["cout"])
        out = h + s["residual"] if case["residual"] else h
        return (out, h, torch.cat(aux)) if case["keep"] and case["tanh"] else out
    parts = list(polynomial(s["seed"], dim, full, value))
    if case["tanh"]:
        a, _ = polynomial(s["activated"], dim, full, value)
        slope = {k: -v for k, v in cut_product(a, a).items()}
        slope[zero] = s["aux"][:full]
        parts = [{k: sum(slope[i] * parts[0][j] for i in slope for j in slope
                         if tuple(u - v for u, v in zip(j, i)) == k) for k in slope},
                 {zero: parts[1][zero] * s["aux"][full:]}]
    dz = rows_of(parts[0], parts[1], dim, case["cout"])
    d_bias = parts[0][zero].sum(0) + parts[1][zero].sum(0)
    return torch.einsum("rc,ck->rk", dz, s["weight"]), torch.einsum("rc,rk->ck", dz, x), d_bias
