"""CPU: the layer oracle against differences and nested derivatives, the generated products
as host C++, and the layer entry points' refusals."""

import ctypes
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import jets as J
from oracle import layers as L
from tests.layers_cases import affine_case, norm_case, worst

ROOT = Path(__file__).resolve().parents[1]
D = ctypes.POINTER(ctypes.c_double)
EPS = 1e-5


@pytest.mark.parametrize("dim", [2, 3])
def test_norm_adjoint_matches_differences(dim):
    full, value, c = 2, 3, 7
    k = norm_case(dim, full, value, c)
    _, stats = L.layer_norm(k["x"], k["gain"], k["bias"], EPS, dim, full)
    got = L.layer_norm_vjp(k["x"], k["gain"], stats, k["seed"], None, dim, full)
    loss = lambda x, g, b: float((L.layer_norm(x, g, b, EPS, dim, full)[0] * k["seed"]).sum())
    args = [k["x"], k["gain"], k["bias"]]
    rng = np.random.default_rng(5)
    for i, grad in enumerate(got):
        step = rng.normal(size=args[i].shape)
        # central difference, h = 1e-5: h^2 f'''/6 ~ 1e-9 and rounding 1e-16 |f| / h ~ 1e-9
        plus, minus = ([a + s * 1e-5 * step if j == i else a for j, a in enumerate(args)] for s in (1, -1))
        slope = (loss(*plus) - loss(*minus)) / 2e-5
        assert abs(slope - float((grad * step).sum())) <= 1e-6 * (1 + abs(slope)), i


@pytest.mark.parametrize("dim", [2, 3])
@pytest.mark.parametrize("activation", [False, True])
def test_affine_adjoint_matches_differences(dim, activation):
    full, value, cin, cout = 2, 3, 5, 4
    k = affine_case(dim, full, value, cin, cout)
    _, a, a1 = L.affine(k["h"], k["w"], k["b"], k["residual"], dim, full, activation)
    got = L.affine_vjp(k["h"], k["w"], a, a1, k["seed"], dim, full)
    loss = lambda h, w, b: float((L.affine(h, w, b, k["residual"], dim, full, activation)[0] * k["seed"]).sum())
    args = [k["h"], k["w"], k["b"]]
    rng = np.random.default_rng(6)
    for i, grad in enumerate(got):
        step = rng.normal(size=args[i].shape)
        plus, minus = ([a + s * 1e-5 * step if j == i else a for j, a in enumerate(args)] for s in (1, -1))
        slope = (loss(*plus) - loss(*minus)) / 2e-5
        assert abs(slope - float((grad * step).sum())) <= 1e-6 * (1 + abs(slope)), i


@pytest.mark.parametrize("dim", [2, 3])
def test_norm_jets_are_the_derivatives_of_the_normalized_field(dim):
    """Taylor coefficients of layer_norm(field(x)) by nested differentiation."""
    rng = np.random.default_rng(3)
    c = 5
    w, gain, bias = rng.normal(size=(c, dim)), 1 + 0.1 * rng.normal(size=c), rng.normal(size=c)
    x = torch.tensor(rng.normal(size=dim), requires_grad=True)
    field = lambda p: torch.sin(torch.tensor(w) @ p) + 0.3 * (torch.tensor(w) @ p) ** 2

    def coefficients(f):
        rows = []
        for alpha in J.basis(dim):
            row = []
            for ch in range(c):
                y = f(x)[ch]
                for axis, times in enumerate(alpha):
                    for _ in range(times):
                        y = torch.autograd.grad(y, x, create_graph=True)[0][axis]
                row.append(float(y.detach()))
            rows.append(row)
        return np.array(rows) / J.recovery(dim)[:, None]

    def normalized(p):
        f = field(p)
        d = f - f.mean()
        return torch.tensor(gain) * d / torch.sqrt((d * d).mean() + EPS) + torch.tensor(bias)

    out, _ = L.layer_norm(coefficients(field), gain, bias, EPS, dim, 1)
    np.testing.assert_allclose(out, coefficients(normalized), rtol=1e-10, atol=1e-10)


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    folder = tmp_path_factory.mktemp("host_products")
    source = folder / "host_products.cpp"
    source.write_text("""
#include <cmath>
#define __device__
#define __forceinline__ inline
using std::sqrt;
#include "products_generated.cuh"
using namespace flashns_b200;
extern "C" void products(int dim, const double* a, const double* b, double* out) {
  if (dim == 2) {
    jet_square_2d3(a, out); jet_mul_2d3(a, b, out + 20); jet_corr_2d3(a, b, out + 40);
    for (int i = 0; i < 10; ++i) out[60 + i] = b[i];
    jet_corr_add_2d3(a, b, out + 60); jet_rsqrt_2d3(b, out + 80);
  } else {
    jet_square_3d3(a, out); jet_mul_3d3(a, b, out + 20); jet_corr_3d3(a, b, out + 40);
    for (int i = 0; i < 20; ++i) out[60 + i] = b[i];
    jet_corr_add_3d3(a, b, out + 60); jet_rsqrt_3d3(b, out + 80);
  }
}
""")
    out = folder / "host_products.so"
    subprocess.run([gxx, "-O2", "-std=c++17", "-ffp-contract=off", "-shared", "-fPIC",
                    f"-I{ROOT / 'flashns_b200' / 'csrc'}", str(source), "-o", str(out)], check=True,
                   capture_output=True)
    lib = ctypes.CDLL(str(out))
    lib.products.argtypes = [ctypes.c_int, D, D, D]
    return lib


@pytest.mark.parametrize("dim", [2, 3])
def test_generated_products_match_oracle(host, dim):
    rng = np.random.default_rng(dim)
    q = J.q(dim)
    for _ in range(20):
        a, b = rng.normal(size=(1, q, 1)), rng.normal(size=(1, q, 1))
        b[0, 0, 0] = 0.3 + abs(b[0, 0, 0])
        out = np.zeros(100)
        host.products(dim, *(np.ascontiguousarray(v).ctypes.data_as(D) for v in (a, b)), out.ctypes.data_as(D))
        got = out.reshape(5, 20)[:, :q]
        pa, pb = np.abs(a), np.abs(b)
        for k, (e, m) in enumerate([(L.cauchy(a, a, dim), L.cauchy(pa, pa, dim)), (L.cauchy(a, b, dim), L.cauchy(pa, pb, dim)),
                                    (L.corr(a, b, dim), L.corr(pa, pb, dim)),
                                    (b + L.corr(a, b, dim), pb + L.corr(pa, pb, dim)),
                                    (L.rsqrt(b, dim), L.rsqrt(pb, dim, True))]):
            # a product of at most 20 pairs and, in the series, three such factors; both sides
            assert worst(got[k], e[0, :, 0], m[0, :, 0], 2 * 3 * 25) <= 1, k
    # the definition: (v^(-1/2))^2 v = 1, error relative to the sizes of the terms
    r = L.rsqrt(b, dim)
    one = L.cauchy(L.cauchy(r, r, dim), b, dim)[0, :, 0]
    size = L.cauchy(L.cauchy(L.rsqrt(pb, dim, True), L.rsqrt(pb, dim, True), dim), pb, dim)[0, :, 0]
    expected = np.zeros(q)
    expected[0] = 1.0
    assert worst(one, expected, size, 2 * 5 * 25) <= 1


def test_layer_entry_points_check_arguments_before_any_launch():
    """Invalid sizes, missing or overlapping buffers return cudaErrorInvalidValue (1) and empty
    inputs success, before any device call; the pointers are never dereferenced."""
    from flashns_b200 import _lib, build
    build.build()
    lib = _lib.library()
    p = [ctypes.c_void_p((k + 1) << 24) for k in range(10)]
    size = ctypes.c_size_t()
    norm = lambda dim=2, x=p[0], out=p[3], stats=p[4], eps=1e-5, full=3, value=2, c=8: lib.flashns_b200_layer_norm(
        dim, x, p[1], p[2], out, stats, eps, full, value, c, None)
    for bad in (dict(dim=4), dict(x=None), dict(out=None), dict(stats=None), dict(eps=0.0), dict(eps=-1.0),
                dict(eps=float("nan")), dict(eps=float("inf")), dict(full=-1), dict(value=-1), dict(c=0),
                dict(full=1 << 61), dict(out=p[0]), dict(stats=p[3])):
        assert norm(**bad) == 1, bad
    assert norm(full=0, value=0, x=None) == 0
    assert lib.flashns_b200_layer_norm_vjp_scratch(2, 3, 2, 0, ctypes.byref(size)) == 1
    assert lib.flashns_b200_layer_norm_vjp_scratch(2, 3, 2, 8, None) == 1
    assert lib.flashns_b200_layer_norm_vjp_scratch(2, 0, 0, 8, ctypes.byref(size)) == 0 and size.value == 0
    vjp = lambda dim=2, x=p[0], seed=p[3], dx=p[5], dg=p[6], scratch=p[8], full=3, value=2, c=8: \
        lib.flashns_b200_layer_norm_vjp(dim, x, p[1], p[2], seed, None, dx, dg, p[7], scratch, 1 << 20, full, value,
                                        c, None)
    for bad in (dict(dim=1), dict(x=None), dict(seed=None), dict(dx=None), dict(dg=None), dict(scratch=None),
                dict(full=-1), dict(c=0), dict(dx=p[0]), dict(dx=p[3])):
        assert vjp(**bad) == 1, bad
    aff = lambda dim=2, act=1, h=p[0], res=p[3], out=p[4], a=p[5], aux=p[6], full=3, value=2, cin=8, cout=4: \
        lib.flashns_b200_affine(dim, act, h, p[1], p[2], res, out, a, aux, full, value, cin, cout, None)
    for bad in (dict(dim=0), dict(act=2), dict(act=0), dict(full=0, cin=1 << 30, cout=1 << 30), dict(h=None), dict(out=None), dict(full=-1), dict(cin=0),
                dict(cout=0), dict(out=p[0]), dict(out=p[3]), dict(a=p[4]), dict(a=p[0])):
        assert aff(**bad) == 1, bad
    assert aff(full=0, value=0, h=None, out=None) == 0
    assert lib.flashns_b200_affine_vjp_scratch(2, 2, 3, 2, 8, 4, ctypes.byref(size)) == 1
    assert lib.flashns_b200_affine_vjp_scratch(2, 1, 0, 0, 8, 4, ctypes.byref(size)) == 0 and size.value == 0
    avjp = lambda dim=2, act=1, h=p[0], a=p[2], aux=p[3], seed=p[4], dh=p[5], dw=p[6], scratch=p[8], n=1 << 22, \
        full=3, value=2, cin=8, cout=4: lib.flashns_b200_affine_vjp(
            dim, act, h, p[1], a, aux, seed, dh, dw, p[7], scratch, n, full, value, cin, cout, None)
    for bad in (dict(dim=5), dict(act=-1), dict(h=None), dict(a=None), dict(aux=None), dict(seed=None), dict(dh=None),
                dict(dw=None), dict(scratch=None), dict(scratch=ctypes.c_void_p((9 << 24) + 8)), dict(n=0), dict(full=-1), dict(cin=0), dict(cout=-3),
                dict(dh=p[0]), dict(dh=p[4]), dict(dh=p[2])):
        assert avjp(**bad) == 1, bad


def test_layer_hooks_refuse_host_and_narrow_tensors():
    from flashns_b200.jet_packed import PackedLayout
    from flashns_b200.native import NativeCUDA
    nat, layout = NativeCUDA(), PackedLayout(1, 2, 2)
    x = torch.zeros(layout.rows, 4, dtype=torch.float64)
    g, w, aux = torch.zeros(4, dtype=torch.float64), torch.zeros(4, 4, dtype=torch.float64), x[:3]
    for call in (lambda: nat.layer_norm(layout, x, g, g), lambda: nat.layer_norm_vjp(layout, x, g, x[:, :2], x),
                 lambda: nat.affine(layout, x, w, g), lambda: nat.affine_activation(layout, x, w, g),
                 lambda: nat.affine_vjp(layout, x, w, x),
                 lambda: nat.affine_activation_vjp(layout, x, w, x, aux, x)):
        with pytest.raises(ValueError, match="CUDA FP64"):
            call()


def test_layer_entry_points_refuse_every_overlap_of_an_output():
    """An output or the scratch over any input or any other output, from the same address to the
    last byte: cudaErrorInvalidValue (1) before any device call; the pointers are never dereferenced."""
    from flashns_b200 import _lib, build
    build.build()
    lib = _lib.library()
    full, value, cin, cout, scratch = 3, 2, 8, 4, 1 << 20
    rows, points = full * 10 + value, full + value
    # (argument, doubles, is written), in the order of the call
    norm = [("value", rows * cin, 0), ("gain", cin, 0), ("bias", cin, 0), ("out", rows * cin, 1), ("stats", rows * 2, 1)]
    norm_vjp = [("value", rows * cin, 0), ("gain", cin, 0), ("stats", rows * 2, 0), ("seed", rows * cin, 0),
                ("skip", rows * cin, 0), ("d_value", rows * cin, 1), ("d_gain", cin, 1), ("d_bias", cin, 1),
                ("scratch", scratch // 8, 1)]
    affine = [("hidden", rows * cin, 0), ("weight", cout * cin, 0), ("bias", cout, 0), ("residual", rows * cout, 0),
              ("out", rows * cout, 1), ("activated", rows * cout, 1), ("aux", points * cout, 1)]
    affine_vjp = [("hidden", rows * cin, 0), ("weight", cout * cin, 0), ("activated", rows * cout, 0),
                  ("aux", points * cout, 0), ("seed", rows * cout, 0), ("d_hidden", rows * cin, 1),
                  ("d_weight", cout * cin, 1), ("d_bias", cout, 1), ("scratch", scratch // 8, 1)]
    calls = [(norm, lambda p: lib.flashns_b200_layer_norm(2, *p, 1e-5, full, value, cin, None)),
             (norm_vjp, lambda p: lib.flashns_b200_layer_norm_vjp(2, *p, scratch, full, value, cin, None)),
             (affine, lambda p: lib.flashns_b200_affine(2, 1, *p, full, value, cin, cout, None)),
             (affine_vjp, lambda p: lib.flashns_b200_affine_vjp(2, 1, *p, scratch, full, value, cin, cout, None))]
    for arguments, call in calls:
        for i, (name, size, written) in enumerate(arguments):
            for j, (other, length, also) in enumerate(arguments):
                if i == j or not written or (also and j > i):
                    continue
                # the scratch stays on a 16-byte boundary
                for at in {0, 8 * (length - 1) // 16 * 16, -(8 * (size - 1) // 16 * 16)}:
                    p = [(k + 1) << 24 for k in range(len(arguments))]
                    p[i] = p[j] + at
                    assert call(p) == 1, (name, other, at)


@pytest.mark.parametrize("groups", [2, 3, 4])
def test_affine_turns_end_for_every_tile_count(groups):
    """The forward kernels' groups take turns by the protocol of the evaluation's: group g of block b
    has the tiles b + (g + groups k) per, which are the block's tiles g, g + groups, ..., so every
    order of the groups ends with no arrival pending."""
    import itertools
    from tests.test_turn_protocol import count, run
    for blocks, tiles in itertools.product((1, 3), range(0, 40)):
        per = min(max(tiles, 1), blocks)
        for b in range(per):
            mine = len(range(b, tiles, per))
            for g in range(groups):
                first, step = b + g * per, per * groups
                assert ((tiles - 1 - first) // step + 1 if first < tiles else 0) == count(mine, g, groups)
    for order in itertools.permutations(range(groups)):
        for m in range(0, 40):
            run(m, order, groups)
