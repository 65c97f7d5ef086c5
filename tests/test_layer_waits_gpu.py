"""GPU: a layer kernel whose wait on a copy gives up sets the fault word, writes nothing from the
copy, lets what is under way land and returns; the calls after it are as before.

The waits are made to give up by polling zero times (the copies themselves are ordinary ones)."""

import ctypes

import pytest
import torch

from oracle import jets as J
from tests.layers_cases import affine_case
from tests.test_layers_gpu import T, guarded, parts

pytestmark = pytest.mark.gpu
POLLS = 1 << 17


@pytest.fixture
def lib(cuda):
    from flashns_b200 import _lib
    lib = _lib.library()
    assert fault(lib, clear=True) == 0
    yield lib
    assert lib.flashns_b200_layer_wait_polls(POLLS, POLLS) == 0
    fault(lib, clear=True)


def fault(lib, clear=False):
    torch.cuda.synchronize()
    word = ctypes.c_int(-1)
    assert lib.flashns_b200_device_fault(ctypes.byref(word), int(clear)) == 0
    return word.value


def ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


class Call:
    """One C call on fresh guarded outputs; ``run(tile, late)`` polls that often in its waits."""

    def __init__(self, lib, cuda, sizes, launch):
        self.lib, self.cuda, self.sizes, self.launch = lib, cuda, sizes, launch

    def run(self, tile=POLLS, late=POLLS):
        buffers = [guarded(n, self.cuda) for n in self.sizes]
        assert self.lib.flashns_b200_layer_wait_polls(tile, late) == 0
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        assert self.launch([view for view, _, _ in buffers], stream) == 0
        torch.cuda.synchronize()
        assert self.lib.flashns_b200_layer_wait_polls(POLLS, POLLS) == 0
        for _, whole, pad in buffers:
            assert bool((whole[:pad] == 12345.5).all()) and bool((whole[len(whole) - pad:] == 12345.5).all())
        return [view for view, _, _ in buffers]


def untouched(t):
    return bool(torch.isnan(t).all())


def forward(lib, cuda, dim, full, value, cin, cout, residual, activation=True):
    k = affine_case(dim, full, value, cin, cout)
    h, w, b, res = (T(k[n], cuda) for n in ("h", "w", "b", "residual"))
    rows = full * J.q(dim) + value

    def launch(views, stream):
        out, act, aux = views if activation else (*views, None, None)
        return lib.flashns_b200_affine(dim, int(activation), *map(ptr, (h, w, b, res if residual else None, out, act, aux)),
                                       full, value, cin, cout, stream)
    return Call(lib, cuda, [rows * cout] * 2 + [(full + value) * cout] if activation else [rows * cout], launch)


def adjoint(lib, cuda, dim, full, value, cin, cout, activation=True):
    """Outputs d_hidden, d_weight, d_bias, then the scratch."""
    k = affine_case(dim, full, value, cin, cout)
    h, w, b, g = (T(k[n], cuda) for n in ("h", "w", "b", "seed"))
    _, act, aux = parts(dim, full, value)[0].affine_activation(parts(dim, full, value)[1], h, w, b)
    size = ctypes.c_size_t()
    assert lib.flashns_b200_affine_vjp_scratch(dim, int(activation), full, value, cin, cout, ctypes.byref(size)) == 0

    def launch(views, stream):
        kept = (act, aux) if activation else (None, None)
        return lib.flashns_b200_affine_vjp(dim, int(activation), *map(ptr, (h, w, *kept, g, *views)), size.value, full,
                                           value, cin, cout, stream)
    return Call(lib, cuda, [h.numel(), w.numel(), cout, size.value // 8], launch)


def recovers(call, lib, expected):
    assert fault(lib, clear=True) == 1
    assert fault(lib) == 0
    for p, q in zip(call.run(), expected):
        assert torch.equal(p, q)
    assert fault(lib) == 0


# the residual and the outputs through boxes of their own, boxes in the tile's place, by threads
FORWARD = [(2, 3000, 100, 64, 64), (2, 40, 9, 64, 40), (2, 3100, 77, 128, 128), (2, 21, 5, 114, 96), (3, 1300, 90, 64, 64),
           (3, 700, 50, 32, 100), (3, 700, 50, 128, 128), (2, 3000, 100, 64, 63)]


@pytest.mark.parametrize("dim,full,value,cin,cout", FORWARD)
@pytest.mark.parametrize("residual", [False, True])
def test_forward_gives_up_on_a_tile(cuda, lib, dim, full, value, cin, cout, residual):
    call = forward(lib, cuda, dim, full, value, cin, cout, residual)
    expected = call.run()
    assert fault(lib) == 0
    for late in (POLLS, 0):
        assert all(map(untouched, call.run(tile=0, late=late)))
        recovers(call, lib, expected)


@pytest.mark.parametrize("dim,full,value,cin,cout", FORWARD)
def test_forward_gives_up_on_a_residual(cuda, lib, dim, full, value, cin, cout):
    call = forward(lib, cuda, dim, full, value, cin, cout, True)
    expected = call.run()
    got = call.run(late=0)
    if cout % 2 or (dim == 3 and cin == 128):  # by threads: there is no second wait
        assert fault(lib) == 0 and all(map(torch.equal, got, expected))
    else:
        assert untouched(got[0]) and untouched(got[1])
        recovers(call, lib, expected)


# dH through boxes of its own, boxes in the tile's place, by threads; one kernel (to 64 wide), then two
ADJOINT = [(2, 3000, 100, 64, 64), (2, 9, 5, 64, 64), (2, 3000, 100, 30, 62), (2, 3000, 100, 64, 3), (3, 1300, 90, 64, 64),
           (2, 2500, 77, 128, 128), (2, 2500, 77, 100, 80), (3, 900, 50, 128, 66), (2, 2500, 77, 65, 66)]


@pytest.mark.parametrize("dim,full,value,cin,cout", ADJOINT)
@pytest.mark.parametrize("activation", [False, True])
def test_adjoint_gives_up_on_a_tile(cuda, lib, dim, full, value, cin, cout, activation):
    call = adjoint(lib, cuda, dim, full, value, cin, cout, activation)
    expected = call.run()[:3]
    assert fault(lib) == 0
    got = call.run(tile=0)
    if cout % 2 or (max(cin, cout) <= 64 and cin % 2):  # no tile comes by TMA: nothing waits
        assert fault(lib) == 0 and all(map(torch.equal, got, expected))
    else:
        assert untouched(got[0])
        recovers(call, lib, expected)


@pytest.mark.parametrize("dim,full,value,cin,cout", [c for c in ADJOINT if max(c[3:]) <= 64 and c[4] % 2 == 0])
def test_adjoint_gives_up_on_its_input(cuda, lib, dim, full, value, cin, cout):
    """H, which takes A's place behind the products of dH."""
    call = adjoint(lib, cuda, dim, full, value, cin, cout)
    expected = call.run()[:3]
    assert untouched(call.run(late=0)[0])
    recovers(call, lib, expected)


# several stages a block; one stage; blocks with fewer stages than others; 64 to 256 wide blocks
WGRAD = [(2, 3000, 100, 64, 130), (2, 3, 1, 64, 130), (2, 1500, 93, 130, 140), (3, 1300, 90, 200, 192), (2, 9000, 41, 66, 320)]


@pytest.mark.parametrize("dim,full,value,cin,cout", WGRAD)
@pytest.mark.parametrize("tile,late", [(0, POLLS), (2000, 0)])
def test_weight_gradient_gives_up(cuda, lib, dim, full, value, cin, cout, tile, late):
    """Above 128 outputs only the weight gradient waits: on its stages, and (`late`) for a free one."""
    call = adjoint(lib, cuda, dim, full, value, cin, cout, activation=False)
    expected = call.run()[:3]
    got = call.run(tile=tile, late=late)
    assert torch.equal(got[0], expected[0])
    if tile and full == 3:  # one stage: there is none to free
        assert fault(lib) == 0 and all(map(torch.equal, got, expected))
    else:
        recovers(call, lib, expected)


def test_polls_are_bounded(lib):
    assert lib.flashns_b200_layer_wait_polls(POLLS + 1, 1) == 1 and lib.flashns_b200_layer_wait_polls(1, POLLS + 1) == 1
