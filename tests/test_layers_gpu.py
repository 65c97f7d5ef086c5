"""GPU: layer norm and affine + tanh + residual on packed jets, and their adjoints, against
the 64-bit oracle within counted roundings."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import jets as J
from oracle import layers as L
from tests.layers_cases import (HALF, affine_case, affine_roundings, affine_vjp_roundings, norm_case, norm_roundings,
                                norm_vjp_roundings, worst)

pytestmark = pytest.mark.gpu
EPS = 1e-5


def T(a, dev):
    return None if a is None else torch.tensor(np.asarray(a), dtype=torch.float64, device=dev)


def parts(dim, full, value):
    from flashns_b200.jet_packed import PackedLayout
    from flashns_b200.native import NativeCUDA
    return NativeCUDA(), PackedLayout(full, value, dim)


POINTS = [(1, 0), (0, 1), (3, 0), (0, 5), (7, 11), (130, 47)]
WIDTHS = [1, 3, 8, 16, 17, 32, 33, 64, 65, 100, 128, 129, 200, 257, 515, 1100]


def check_norm(cuda, dim, full, value, c, skip=True):
    k = norm_case(dim, full, value, c, skip=skip)
    nat, layout = parts(dim, full, value)
    x, gain, bias, seed, extra = (T(k[n], cuda) for n in ("x", "gain", "bias", "seed", "skip"))
    out, stats = nat.layer_norm(layout, x, gain, bias, eps=EPS)
    e_out, e_stats = L.layer_norm(k["x"], k["gain"], k["bias"], EPS, dim, full)
    m_out, m_stats = L.layer_norm(k["x"], k["gain"], k["bias"], EPS, dim, full, magnitude=True)
    n = norm_roundings(c)
    assert worst(out.cpu(), e_out, m_out, n) <= 1
    assert worst(stats.cpu(), e_stats, m_stats, n) <= 1
    got = nat.layer_norm_vjp(layout, x, gain, T(e_stats, cuda), seed, skip=extra)
    exp = L.layer_norm_vjp(k["x"], k["gain"], e_stats, k["seed"], k["skip"], dim, full)
    mag = L.layer_norm_vjp(k["x"], k["gain"], e_stats, k["seed"], k["skip"], dim, full, magnitude=True)
    for g, e, m, r in zip(got, exp, mag, (0, layout.rows, layout.rows)):
        assert worst(g.cpu(), e, m, norm_vjp_roundings(c, r)) <= 1


@pytest.mark.parametrize("dim", [2, 3])
@pytest.mark.parametrize("full,value", POINTS)
@pytest.mark.parametrize("c", [1, 17, 64, 100])
def test_norm_matches_oracle_at_small_point_sets(cuda, dim, full, value, c):
    check_norm(cuda, dim, full, value, c)


@pytest.mark.parametrize("dim", [2, 3])
@pytest.mark.parametrize("c", WIDTHS)
def test_norm_matches_oracle_at_every_width(cuda, dim, c):
    check_norm(cuda, dim, 41, 29, c, skip=c % 2 == 0)


@pytest.mark.parametrize("dim,full,value,c", [(2, 4099, 1031, 64), (3, 2051, 515, 128), (2, 3001, 7000, 30)])
def test_norm_matches_oracle_at_many_points(cuda, dim, full, value, c):
    check_norm(cuda, dim, full, value, c)


def check_affine(cuda, dim, full, value, cin, cout, activation, residual=True, seed=0):
    k = affine_case(dim, full, value, cin, cout, seed)
    if not residual:
        k["residual"] = None
    nat, layout = parts(dim, full, value)
    h, w, b, res, g = (T(k[n], cuda) for n in ("h", "w", "b", "residual", "seed"))
    exp = L.affine(k["h"], k["w"], k["b"], k["residual"], dim, full, activation)
    mag = L.affine(k["h"], k["w"], k["b"], k["residual"], dim, full, activation, magnitude=True)
    if activation:
        got = nat.affine_activation(layout, h, w, b, residual=res)
        alone = nat.affine_activation(layout, h, w, b, residual=res, keep=False)
        assert torch.equal(alone, got[0])
        assert residual or got[1] is got[0]
    else:
        got = (nat.affine(layout, h, w, b, residual=res),)
    for x, e, m in zip(got, exp, mag):
        assert worst(x.cpu(), e, m, affine_roundings(cin)) <= 1
    if activation:
        back = nat.affine_activation_vjp(layout, h, w, T(exp[1], cuda), T(exp[2], cuda), g)
    else:
        back = nat.affine_vjp(layout, h, w, g)
    exp_b = L.affine_vjp(k["h"], k["w"], exp[1], exp[2], k["seed"], dim, full)
    mag_b = L.affine_vjp(k["h"], k["w"], exp[1], exp[2], k["seed"], dim, full, magnitude=True)
    for x, e, m, n in zip(back, exp_b, mag_b, (cout, layout.rows, layout.rows)):
        assert worst(x.cpu(), e, m, affine_vjp_roundings(n)) <= 1


SHAPES = [(1, 1), (3, 64), (64, 3), (64, 64), (65, 33), (32, 32), (31, 66), (128, 128), (100, 60), (200, 130),
          (8, 300), (130, 64), (64, 130), (16, 128), (257, 20), (64, 65), (100, 127), (66, 129), (112, 64), (114, 64), (12, 40)]


@pytest.mark.parametrize("dim", [2, 3])
@pytest.mark.parametrize("full,value", POINTS)
@pytest.mark.parametrize("cin,cout", [(64, 64), (33, 17), (128, 100)])
def test_affine_matches_oracle_at_small_point_sets(cuda, dim, full, value, cin, cout):
    check_affine(cuda, dim, full, value, cin, cout, True)
    check_affine(cuda, dim, full, value, cin, cout, False, residual=False)


@pytest.mark.parametrize("dim", [2, 3])
@pytest.mark.parametrize("activation", [False, True])
@pytest.mark.parametrize("cin,cout", SHAPES)
def test_affine_matches_oracle_at_every_shape(cuda, dim, activation, cin, cout):
    check_affine(cuda, dim, 41, 29, cin, cout, activation, residual=(cin + cout) % 2 == 0)


@pytest.mark.parametrize("dim,full,value,cin,cout", [(2, 4099, 1031, 64, 64), (3, 1031, 515, 64, 64),
                                                     (2, 2051, 509, 128, 128), (3, 1027, 300, 100, 60),
                                                     (2, 0, 9001, 64, 64), (2, 4000, 900, 64, 3), (2, 3001, 77, 64, 97),
                                                     (3, 1500, 401, 128, 66), (2, 3500, 1, 30, 62)])
def test_affine_matches_oracle_at_many_points(cuda, dim, full, value, cin, cout):
    check_affine(cuda, dim, full, value, cin, cout, cout != 3)


@pytest.mark.parametrize("dim", [2, 3])
@pytest.mark.parametrize("cin,cout", [(64, 64), (33, 17), (128, 100), (200, 66), (257, 20), (8, 5)])
def test_value_rows_alone_match_oracle(cuda, dim, cin, cout):
    for value in (1, 41, 333):
        check_affine(cuda, dim, 0, value, cin, cout, True, residual=value != 41)


@pytest.mark.parametrize("dim", [2, 3])
def test_one_tensor_may_be_several_inputs(cuda, dim):
    """The block's input is its own residual; the norm's input is its own seed and skip."""
    full, value, c = 21, 13, 64
    k, n = affine_case(dim, full, value, c, c), norm_case(dim, full, value, c)
    nat, layout = parts(dim, full, value)
    h, w, b, gain, bias = (T(v, cuda) for v in (k["h"], k["w"], k["b"], n["gain"], n["bias"]))
    out, act, aux = nat.affine_activation(layout, h, w, b, residual=h)
    other = nat.affine_activation(layout, h, w, b, residual=h.clone())
    assert all(torch.equal(p, q) for p, q in zip((out, act, aux), other))
    for p, q in zip(nat.affine_activation_vjp(layout, act, w, act, aux, act),
                    nat.affine_activation_vjp(layout, act.clone(), w, act, aux, act.clone())):
        assert torch.equal(p, q)
    _, stats = nat.layer_norm(layout, h, gain, bias)
    for p, q in zip(nat.layer_norm_vjp(layout, h, gain, stats, h, skip=h),
                    nat.layer_norm_vjp(layout, h, gain, stats, h.clone(), skip=h.clone())):
        assert torch.equal(p, q)


def test_offsets_past_32_bits(cuda):
    """More than 2^31 values in a tensor: the last rows match the oracle within the counted
    roundings (their bits may differ from those of the same rows alone: a row's place in its unit
    decides which products are fused into the sums)."""
    if torch.cuda.mem_get_info()[0] < 90 << 30:
        pytest.skip("90 GB of free device memory needed")
    f64 = dict(dtype=torch.float64, device=cuda)
    tail, c = 4096, 64
    rows = (1 << 31) // c + 81 * 1000 + tail
    nat, layout = parts(2, 0, rows)
    x = torch.empty(rows, c, **f64).uniform_(-1, 1)
    gain, bias, w = torch.rand(c, **f64), torch.rand(c, **f64), torch.randn(c, c, **f64) / 8
    end, n_gain, n_bias, n_w = (t.cpu().numpy() for t in (x[-tail:], gain, bias, w))
    out, stats = nat.layer_norm(layout, x, gain, bias, eps=EPS)
    for got, e, m in zip((out, stats), L.layer_norm(end, n_gain, n_bias, EPS, 2, 0),
                         L.layer_norm(end, n_gain, n_bias, EPS, 2, 0, magnitude=True)):
        assert worst(got[-tail:].cpu(), e, m, norm_roundings(c)) <= 1
    del out, got
    n_stats = stats[-tail:].cpu().numpy()
    dx, _, dbias = nat.layer_norm_vjp(layout, x, gain, stats, x)
    e, m = (L.layer_norm_vjp(end, n_gain, n_stats, end, None, 2, 0, magnitude=v)[0] for v in (False, True))
    assert worst(dx[-tail:].cpu(), e, m, norm_vjp_roundings(c)) <= 1
    # every row is summed once: rows roundings of values below 1
    assert float((dbias - x.sum(0)).abs().max()) <= 2 * rows * HALF * rows
    del dx, stats
    for act in (True, False):
        got = nat.affine_activation(layout, x, w, bias, residual=x, keep=False) if act else \
            nat.affine(layout, x, w, bias, residual=x)
        e, m = (L.affine(end, n_w, n_bias, end, 2, 0, act, magnitude=v)[0] for v in (False, True))
        assert worst(got[-tail:].cpu(), e, m, affine_roundings(c)) <= 1
        del got
    dh, _, _ = nat.affine_vjp(layout, x, w, x)
    e, m = (L.affine_vjp(end, n_w, None, None, end, 2, 0, magnitude=v)[0] for v in (False, True))
    assert worst(dh[-tail:].cpu(), e, m, affine_vjp_roundings(c)) <= 1


def test_layer_kernels_raise_no_device_fault(cuda):
    """Their bounded waits on copies all end in time: the word that a wait that gives up sets is clear."""
    from flashns_b200 import _lib
    for case in ((2, 1500, 400, 64, 64), (3, 300, 90, 100, 128), (2, 0, 900, 64, 64)):
        calls(cuda, *case)()
    torch.cuda.synchronize()
    fault = ctypes.c_int(-1)
    assert _lib.library().flashns_b200_device_fault(ctypes.byref(fault), 0) == 0 and fault.value == 0


def test_no_points_give_empty_outputs_and_zero_gradients(cuda):
    for dim in (2, 3):
        nat, layout = parts(dim, 0, 0)
        x, w = torch.empty(0, 6, dtype=torch.float64, device=cuda), torch.ones(4, 6, dtype=torch.float64, device=cuda)
        one, y = torch.ones(6, dtype=torch.float64, device=cuda), x[:, :4].contiguous()
        out, stats = nat.layer_norm(layout, x, one, one)
        assert out.shape == (0, 6) and stats.shape == (0, 2)
        dx, dg, db = nat.layer_norm_vjp(layout, x, one, stats, x)
        assert dx.shape == (0, 6) and not dg.any() and not db.any()
        out, a, aux = nat.affine_activation(layout, x, w, one[:4])
        assert out.shape == (0, 4) and aux.shape == (0, 4)
        for back in (nat.affine_activation_vjp(layout, x, w, a, aux, y), nat.affine_vjp(layout, x, w, y)):
            assert back[0].shape == (0, 6) and not back[1].any() and not back[2].any()


def off_by_one(t):
    """The same values at an address that is a multiple of 8 but not of 16."""
    if t is None:
        return None
    big = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    view = big[1:].view(t.shape)
    view.copy_(t)
    assert view.data_ptr() % 16 == 8 and view.is_contiguous()
    return view


def calls(cuda, dim, full, value, c, cout, place=lambda t: t):
    """Every entry point's outputs on one set of inputs, each input placed by ``place``."""
    n, a = norm_case(dim, full, value, c), affine_case(dim, full, value, c, cout)
    nat, layout = parts(dim, full, value)
    x, gain, bias, seed, skip = (place(T(n[k], cuda)) for k in ("x", "gain", "bias", "seed", "skip"))
    h, w, b, res, g = (place(T(a[k], cuda)) for k in ("h", "w", "b", "residual", "seed"))

    def run():
        out, stats = nat.layer_norm(layout, x, gain, bias)
        back = nat.layer_norm_vjp(layout, x, gain, place(stats), seed, skip=skip)
        y, act, aux = nat.affine_activation(layout, h, w, b, residual=res)
        back2 = nat.affine_activation_vjp(layout, h, w, place(act), place(aux), g)
        z = nat.affine(layout, h, w, b)
        back3 = nat.affine_vjp(layout, h, w, g)
        return [out, stats, *back, y, act, aux, *back2, z, *back3]
    return run


@pytest.mark.parametrize("dim,full,value,c,cout", [(2, 97, 31, 64, 64), (3, 33, 17, 128, 128), (2, 40, 9, 34, 70)])
def test_unaligned_tensors_give_the_same_values(cuda, dim, full, value, c, cout):
    aligned, odd = calls(cuda, dim, full, value, c, cout)(), calls(cuda, dim, full, value, c, cout, off_by_one)()
    rows = full * J.q(dim) + value
    for p, q in zip(aligned, odd):
        # another path may sum in another order: both are within the sums' roundings
        assert float((p - q).abs().max()) <= 8 * (rows + c + cout + 84) * HALF * (1 + float(p.abs().max()))


@pytest.mark.parametrize("dim,full,value,c,cout", [(2, 1500, 400, 64, 64), (3, 300, 90, 100, 128)])
def test_results_repeat_bit_for_bit_on_any_stream_and_in_graphs(cuda, dim, full, value, c, cout):
    run = calls(cuda, dim, full, value, c, cout)
    first = [t.clone() for t in run()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = run()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    graphs = []
    for _ in range(2):  # two graphs of the same calls, replayed in turn and together
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run()
        graphs.append((graph, outs))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for (graph, outs), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                for t in outs:
                    t.fill_(float("nan"))
                graph.replay()
    torch.cuda.synchronize()
    for _, outs in graphs:
        assert all(torch.equal(p, q) for p, q in zip(first, outs))


@pytest.mark.parametrize("dim", [2, 3])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_one_points_nonfinite_values_stay_with_it(cuda, dim, bad):
    full, value, c = 40, 30, 64
    n, a = norm_case(dim, full, value, c), affine_case(dim, full, value, c, c)
    nat, layout = parts(dim, full, value)
    q = J.q(dim)
    x, gain, bias, w, b = (T(v, cuda) for v in (n["x"], n["gain"], n["bias"], a["w"], a["b"]))
    hit = x.clone()
    hit[5 * q + 3, 7] = bad  # a coefficient of full point 5
    hit[full * q + 11, 9] = bad  # value point 11
    keep = torch.ones(layout.rows, dtype=torch.bool, device=cuda)
    keep[5 * q:6 * q] = False
    keep[full * q + 11] = False
    seed = T(n["seed"], cuda)
    for f in (lambda v: nat.layer_norm(layout, v, gain, bias)[0],
              lambda v: nat.layer_norm_vjp(layout, v, gain, nat.layer_norm(layout, x, gain, bias)[1], seed)[0],
              lambda v: nat.affine_activation(layout, v, w, b, residual=x)[0],
              lambda v: nat.affine(layout, v, w, b),
              lambda v: nat.affine_vjp(layout, x, w, v)[0]):
        p, r = f(x), f(hit)
        assert torch.equal(p[keep], r[keep])
        assert not torch.isfinite(r[5 * q:6 * q]).all()
        # tanh(+-inf) = +-1: an infinite pre-activation is a finite value
        assert not torch.isfinite(r[full * q + 11]).all() or (bad == float("inf") and bool((r - x)[full * q + 11].abs().max() <= 1 + 4 * HALF * (1 + x.abs().max())))
    for back in (nat.affine_vjp(layout, hit, w, seed), nat.affine_vjp(layout, x, w, hit)):
        assert not torch.isfinite(back[1]).all()
    _, dgain, _ = nat.layer_norm_vjp(layout, hit, gain, nat.layer_norm(layout, x, gain, bias)[1], seed)
    assert not torch.isfinite(dgain).all()


def test_equal_channels_are_normalized_to_the_bias(cuda):
    """Variance zero everywhere: r = eps^(-1/2), the output is the bias and nothing divides by zero."""
    for dim in (2, 3):
        nat, layout = parts(dim, 5, 7)
        x = torch.full((layout.rows, 32), 0.75, dtype=torch.float64, device=cuda)
        gain, bias = torch.rand(32, dtype=torch.float64, device=cuda), torch.rand(32, dtype=torch.float64, device=cuda)
        out, stats = nat.layer_norm(layout, x, gain, bias, eps=EPS)
        expected = torch.zeros_like(x)
        expected[layout.zero_rows(cuda)] = bias
        assert torch.equal(out, expected)
        np.testing.assert_allclose(stats[0].cpu(), [0.75, EPS ** -0.5], rtol=1e-15)
        dx, _, _ = nat.layer_norm_vjp(layout, x, gain, stats, x)
        assert torch.isfinite(dx).all()


def guarded(count, cuda, pad=64):
    """A NaN-filled buffer of ``count`` doubles between sentinels, and the whole allocation."""
    whole = torch.full((count + 2 * pad,), 12345.5, dtype=torch.float64, device=cuda)
    whole[pad:pad + count] = float("nan")
    return whole[pad:pad + count], whole, pad


@pytest.mark.parametrize("dim,full,value,c,cout", [(2, 37, 13, 64, 64), (3, 21, 27, 100, 60), (2, 9, 5, 130, 140),
                                                   (2, 33, 4, 7, 3), (3, 9, 0, 128, 128), (2, 0, 23, 64, 64)])
def test_writes_stay_inside_the_callers_buffers(cuda, dim, full, value, c, cout):
    from flashns_b200 import _lib
    lib = _lib.library()
    n, a = norm_case(dim, full, value, c), affine_case(dim, full, value, c, cout)
    rows, points = full * J.q(dim) + value, full + value
    ptr = lambda t: ctypes.c_void_p(t.data_ptr()) if t is not None else None
    buffers = []

    def fresh(count):
        view, whole, pad = guarded(count, cuda)
        buffers.append((view, whole, pad))
        return view

    def check(status, outputs):
        assert status == 0
        torch.cuda.synchronize()
        for view, whole, pad in buffers:
            assert bool((whole[:pad] == 12345.5).all()) and bool((whole[len(whole) - pad:] == 12345.5).all())
        for t in outputs:
            assert torch.isfinite(t).all()
        buffers.clear()

    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    size = ctypes.c_size_t()
    x, gain, bias, seed, skip = (T(n[k], cuda) for k in ("x", "gain", "bias", "seed", "skip"))
    out, stats = fresh(rows * c), fresh(rows * 2)
    check(lib.flashns_b200_layer_norm(dim, *map(ptr, (x, gain, bias, out, stats)), EPS, full, value, c, stream),
          [out, stats])
    stats = stats.clone()
    assert lib.flashns_b200_layer_norm_vjp_scratch(dim, full, value, c, ctypes.byref(size)) == 0
    outs, scratch = [fresh(rows * c), fresh(c), fresh(c)], fresh(size.value // 8)
    check(lib.flashns_b200_layer_norm_vjp(dim, *map(ptr, (x, gain, stats, seed, skip, *outs, scratch)), size.value,
                                          full, value, c, stream), outs)
    h, w, b, res, g = (T(a[k], cuda) for k in ("h", "w", "b", "residual", "seed"))
    outs = [fresh(rows * cout), fresh(rows * cout), fresh(points * cout)]
    check(lib.flashns_b200_affine(dim, 1, *map(ptr, (h, w, b, res, *outs)), full, value, c, cout, stream), outs)
    act, aux = outs[1].clone(), outs[2].clone()
    outs = [fresh(rows * cout)]
    check(lib.flashns_b200_affine(dim, 0, *map(ptr, (h, w, b, None, *outs, None, None)), full, value, c, cout, stream),
          outs)
    for on in (0, 1):
        assert lib.flashns_b200_affine_vjp_scratch(dim, on, full, value, c, cout, ctypes.byref(size)) == 0
        outs, scratch = [fresh(rows * c), fresh(cout * c), fresh(cout)], fresh(size.value // 8)
        check(lib.flashns_b200_affine_vjp(dim, on, *map(ptr, (h, w, act if on else None, aux if on else None, g, *outs,
                                                             scratch)), size.value, full, value, c, cout, stream), outs)
        # one byte short of the size that the query gave
        assert lib.flashns_b200_affine_vjp(dim, on, *map(ptr, (h, w, act, aux, g, *outs, scratch)), size.value - 1,
                                           full, value, c, cout, stream) == 1


def test_hooks_check_shapes(cuda):
    nat, layout = parts(2, 2, 3)
    f64 = dict(dtype=torch.float64, device=cuda)
    x, g, w, stats, aux = (torch.zeros(layout.rows, 4, **f64), torch.zeros(4, **f64), torch.zeros(6, 4, **f64),
                           torch.zeros(layout.rows, 2, **f64), torch.zeros(layout.points, 6, **f64))
    y, b = torch.zeros(layout.rows, 6, **f64), torch.zeros(6, **f64)
    for call in (lambda: nat.layer_norm(layout, x[1:], g, g), lambda: nat.layer_norm(layout, x, g[1:], g),
                 lambda: nat.layer_norm(layout, x, g, g, eps=0.0), lambda: nat.layer_norm(layout, x, g, g, eps=float("inf")),
                 lambda: nat.layer_norm(layout, x.T.contiguous().T, g, g), lambda: nat.layer_norm(layout, x.float(), g, g),
                 lambda: nat.layer_norm_vjp(layout, x, g, stats[1:], x), lambda: nat.layer_norm_vjp(layout, x, g, stats, y),
                 lambda: nat.layer_norm_vjp(layout, x, g, stats, x, skip=y),
                 lambda: nat.affine(layout, x, w, g), lambda: nat.affine(layout, y, w, b),
                 lambda: nat.affine(layout, x, w, b, residual=x), lambda: nat.affine(layout, x, w[:0], b[:0]),
                 lambda: nat.affine_activation(layout, x, w.T, b),
                 lambda: nat.affine_vjp(layout, x, w, x), lambda: nat.affine_activation_vjp(layout, x, w, y, aux[1:], y),
                 lambda: nat.affine_activation_vjp(layout, x, w, x, aux, y)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError):
        nat.layer_norm(layout, x.requires_grad_(), g, g)


class ResidualNet:
    """Pre-norm residual net on the hooks: coordinates -> tanh layer -> blocks
    ``x + W2 tanh(W1 norm(x) + b1) + b2`` -> norm -> (u, v, p); NS loss and every gradient."""

    def __init__(self, rng, dim, width, inner, blocks):
        normal = lambda *s: rng.normal(size=s)
        self.p = {"w0": normal(width, dim), "b0": 0.1 * normal(width)}
        for i in range(blocks):
            self.p.update({f"g{i}": 1 + 0.1 * normal(width), f"s{i}": 0.1 * normal(width),
                           f"u{i}": normal(inner, width) / np.sqrt(width), f"c{i}": 0.1 * normal(inner),
                           f"v{i}": normal(width, inner) / np.sqrt(inner), f"d{i}": 0.1 * normal(width)})
        self.p.update({"g": 1 + 0.1 * normal(width), "s": 0.1 * normal(width), "w": normal(3, width) / np.sqrt(width),
                       "b": 0.1 * normal(3)})
        self.blocks = blocks

    def on_hooks(self, x, ni, pw, bw, target, loss, cuda):
        nat, layout = parts(2, ni, len(x) - ni)
        p = {k: T(v, cuda) for k, v in self.p.items()}
        x, pw, bw, target = (T(v, cuda) for v in (x, pw, bw, target))
        h, a0 = nat.coordinate_affine_activation(layout, x, p["w0"], p["b0"])
        first, kept = h, []
        for i in range(self.blocks):
            n, stats = nat.layer_norm(layout, h, p[f"g{i}"], p[f"s{i}"])
            a, _, aux = nat.affine_activation(layout, n, p[f"u{i}"], p[f"c{i}"])
            kept.append((h, n, stats, a, aux))
            h = nat.affine(layout, a, p[f"v{i}"], p[f"d{i}"], residual=h)
        n, stats = nat.layer_norm(layout, h, p["g"], p["s"])
        y = nat.affine(layout, n, p["w"], p["b"])
        total, di, db = nat.seed(y[:ni * 10].view(ni, 10, 3), y[ni * 10:], pw, bw, target, loss)
        d = torch.cat((di.view(ni * 10, 3), db))
        grads = {}
        d, grads["w"], grads["b"] = nat.affine_vjp(layout, n, p["w"], d)
        d, grads["g"], grads["s"] = nat.layer_norm_vjp(layout, h, p["g"], stats, d)
        for i in reversed(range(self.blocks)):
            h, n, stats, a, aux = kept[i]
            e, grads[f"v{i}"], grads[f"d{i}"] = nat.affine_vjp(layout, a, p[f"v{i}"], d)
            e, grads[f"u{i}"], grads[f"c{i}"] = nat.affine_activation_vjp(layout, n, p[f"u{i}"], a, aux, e)
            d, grads[f"g{i}"], grads[f"s{i}"] = nat.layer_norm_vjp(layout, h, p[f"g{i}"], stats, e, skip=d)
        grads["w0"], grads["b0"] = nat.coordinate_activation_wgrad(layout, x, first, a0, d)
        return total, grads

    def by_differentiation(self, x, ni, pw, bw, target, loss):
        """The same loss by nested differentiation of the net at each point (CPU)."""
        from flashns_b200 import codegen
        p = {k: torch.tensor(v, requires_grad=True) for k, v in self.p.items()}
        pts = torch.tensor(x, requires_grad=True)

        def norm(h, g, s):  # in elementary operations: it is differentiated four times
            d = h - h.mean(1, keepdim=True)
            return g * d / torch.sqrt((d * d).mean(1, keepdim=True) + EPS) + s

        h = torch.tanh(pts @ p["w0"].T + p["b0"])
        for i in range(self.blocks):
            inner = torch.tanh(norm(h, p[f"g{i}"], p[f"s{i}"]) @ p[f"u{i}"].T + p[f"c{i}"])
            h = h + inner @ p[f"v{i}"].T + p[f"d{i}"]
        y = norm(h, p["g"], p["s"]) @ p["w"].T + p["b"]
        raw = {}

        def derivative(field, alpha):
            if (field, alpha) not in raw:
                if sum(alpha) == 0:
                    raw[field, alpha] = y[:, field]
                else:
                    axis = 0 if alpha[0] else 1
                    below = tuple(v - (j == axis) for j, v in enumerate(alpha))
                    raw[field, alpha] = torch.autograd.grad(derivative(field, below).sum(), pts, create_graph=True)[0][:, axis]
            return raw[field, alpha]

        residuals, groups = codegen.residuals_uvp()
        value = 0.0
        for r, group in zip(residuals, groups):
            total = 0.0
            for key, (a, b) in r.items():
                term = a + b * loss.viscosity
                for field, alpha in key:
                    term = term * derivative(field, alpha)
                total = total + term
            weight = torch.tensor(pw) * (loss.gradient_weight if group else 1.0)
            value = value + 0.5 * (weight * total[:ni] ** 2).sum()
        value = value + loss.boundary_weight * (torch.tensor(bw) * (y[ni:] - torch.tensor(target)) ** 2).sum()
        grads = torch.autograd.grad(value, list(p.values()))
        return float(value.detach()), dict(zip(p, (g.numpy() for g in grads)))


@pytest.mark.parametrize("width,inner,blocks,ni,nb", [(16, 24, 1, 9, 5), (64, 64, 2, 33, 14), (20, 7, 3, 1, 1)])
def test_residual_net_on_the_hooks_matches_nested_differentiation(cuda, width, inner, blocks, ni, nb):
    from flashns_b200.ns_seed import NSLoss
    from tests.cases import random_case, rel_norm
    c = random_case(ni, nb, [2, width, 3], seed=4)
    loss = NSLoss(0.07, 0.2, 5.0)
    net = ResidualNet(np.random.default_rng(9), 2, width, inner, blocks)
    total, grads = net.on_hooks(c["x"], ni, c["pw"], c["bw"], c["target"], loss, cuda)
    value, expected = net.by_differentiation(c["x"], ni, c["pw"], c["bw"], c["target"], loss)
    # the framework's own criterion for a loss and its gradient: 1e-10 of their norm
    assert abs(float(total) - value) <= 1e-10 * abs(value)
    assert set(grads) == set(expected)
    for k in expected:
        assert rel_norm(grads[k].cpu(), expected[k]) <= 1e-10, k


# Odd or wide inputs (four, three or two groups of warps by turns) with several tiles for every group
# and one more for some, both ways round; dW with several stages a block, asked for by TMA or not.
@pytest.mark.parametrize("dim,full,value,cin,cout", [(2, 5003, 41, 33, 17), (2, 4800, 0, 33, 64), (2, 4000, 900, 130, 64),
                                                     (2, 3001, 77, 96, 190), (2, 3001, 77, 300, 40), (2, 5001, 13, 65, 191),
                                                     (3, 4001, 37, 33, 17), (3, 1500, 401, 190, 150), (3, 2600, 77, 258, 40),
                                                     (3, 2003, 9, 161, 131)])
@pytest.mark.parametrize("activation", [False, True])
def test_affine_by_small_groups_matches_oracle_at_many_points(cuda, dim, full, value, cin, cout, activation):
    check_affine(cuda, dim, full, value, cin, cout, activation)


# a stream function's two outputs and two inputs; outputs below a box's 16 columns; widths whose boxes
# find no room (82 to 112 inputs forward, 74 to 96 outputs backward, above 64 outputs)
@pytest.mark.parametrize("dim", [2, 3])
@pytest.mark.parametrize("full,value", [(41, 29), (2101, 333)])
@pytest.mark.parametrize("cin,cout", [(2, 64), (64, 2), (2, 2), (64, 4), (64, 10), (96, 96), (82, 74), (112, 80), (64, 96),
                                      (90, 66), (8, 90)])
def test_affine_at_narrow_widths_and_without_boxes(cuda, dim, full, value, cin, cout):
    for activation in (False, True):
        check_affine(cuda, dim, full, value, cin, cout, activation, residual=activation)
    check_affine(cuda, dim, full, value, cin, cout, True, residual=False)


def past_32_bits(cuda, full, value, widths, dim=2):
    """Random packed rows of these widths, and the trailing points as a small layout of their own:
    their row count and (full, value).  90 GB are needed."""
    if torch.cuda.mem_get_info()[0] < 90 << 30:
        torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 90 << 30:
        pytest.skip("90 GB of free device memory needed")
    end = (64, value) if value < 4096 else (0, 4096)
    rows = full * J.q(dim) + value
    assert rows * max(widths) > 1 << 31
    x = torch.empty(rows, widths[0], dtype=torch.float64, device=cuda).uniform_(-1, 1)
    return x, end[0] * J.q(dim) + end[1], end


@pytest.mark.parametrize("full,value,cin,cout", [(3_400_003, 5, 8, 64), (1_003, 33_600_000, 8, 64), (3_400_003, 5, 64, 8),
                                                 (3_300_003, 7, 8, 66), (1_700_003, 3, 8, 130)])
def test_full_points_and_kept_values_past_32_bits(cuda, full, value, cin, cout):
    """More than 2^31 values with full points, `activated` and `aux` kept, through the adjoint: the
    last points match the oracle.  The seed is zero but there, so that the weight and bias gradients
    are sums over them alone and their bound is as tight as at that size."""
    x, tail, (e_full, e_value) = past_32_bits(cuda, full, value, (cin, cout))
    f64 = dict(dtype=torch.float64, device=cuda)
    nat, layout = parts(2, full, value)
    points = e_full + e_value
    w, b = torch.randn(cout, cin, **f64) / cin ** 0.5, torch.rand(cout, **f64)
    h, n_w, n_b = (t.cpu().numpy() for t in (x[-tail:], w, b))
    _, act, aux = nat.affine_activation(layout, x, w, b)
    exp, mag = (L.affine(h, n_w, n_b, None, 2, e_full, True, magnitude=v) for v in (False, True))
    for got, e, m in zip((act[-tail:], act[-tail:], aux[-points:]), exp, mag):
        assert worst(got.cpu(), e, m, affine_roundings(cin)) <= 1
    seed = torch.zeros(layout.rows, cout, **f64)
    seed[-tail:].uniform_(-1, 1)
    n_act, n_aux, n_seed = (t.cpu().numpy() for t in (act[-tail:], aux[-points:], seed[-tail:]))
    back = nat.affine_activation_vjp(layout, x, w, act, aux, seed)
    assert not back[0][:-tail].any()
    exp, mag = (L.affine_vjp(h, n_w, n_act, n_aux, n_seed, 2, e_full, magnitude=v) for v in (False, True))
    for got, e, m, n in zip((back[0][-tail:], *back[1:]), exp, mag, (cout, tail, tail)):
        assert worst(got.cpu(), e, m, affine_vjp_roundings(n)) <= 1
    del x, act, aux, seed, back, got
    torch.cuda.empty_cache()


@pytest.mark.parametrize("full,value", [(3_400_003, 5), (1_003, 33_600_000)])
def test_norm_of_full_points_past_32_bits(cuda, full, value):
    c = 64
    x, tail, (e_full, _) = past_32_bits(cuda, full, value, (c,))
    f64 = dict(dtype=torch.float64, device=cuda)
    nat, layout = parts(2, full, value)
    gain, bias = torch.rand(c, **f64), torch.rand(c, **f64)
    end, n_gain, n_bias = (t.cpu().numpy() for t in (x[-tail:], gain, bias))
    out, stats = nat.layer_norm(layout, x, gain, bias, eps=EPS)
    exp, mag = (L.layer_norm(end, n_gain, n_bias, EPS, 2, e_full, magnitude=v) for v in (False, True))
    for got, e, m in zip((out, stats), exp, mag):
        assert worst(got[-tail:].cpu(), e, m, norm_roundings(c)) <= 1
    del out, got
    seed = torch.zeros_like(x)
    seed[-tail:].uniform_(-1, 1)
    n_stats, n_seed = stats[-tail:].cpu().numpy(), seed[-tail:].cpu().numpy()
    back = nat.layer_norm_vjp(layout, x, gain, stats, seed)
    assert not back[0][:-tail].any()
    exp, mag = (L.layer_norm_vjp(end, n_gain, n_stats, n_seed, None, 2, e_full, magnitude=v) for v in (False, True))
    for got, e, m, n in zip((back[0][-tail:], *back[1:]), exp, mag, (0, tail, tail)):
        assert worst(got.cpu(), e, m, norm_vjp_roundings(c, n)) <= 1
    del x, stats, seed, back, got
    torch.cuda.empty_cache()
