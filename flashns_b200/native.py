"""Hook providers with the reference's binding interface, on this library's kernels.

``NativeCUDA`` has the methods of ``experiments/pinn_v8/native.py:11-221`` (packed
layout hooks for ``PackedPINN``) and ``Native`` those of
``experiments/cuda_jet_h100/gpu.py`` (dense ``[B,Q,C]`` activation, VJP and dgrad).
Launches are asynchronous on the current stream; shape/dtype errors raise
``ValueError``, nonzero CUDA statuses ``RuntimeError``.
"""

import ctypes
from functools import lru_cache

import torch

from flashns_b200 import _lib
from flashns_b200.jet_spec import JetSpec


def _ptr(t):
    return t.data_ptr() if t is not None and t.numel() else None


def _launch(name, args, tensors):
    """One call on the current stream of ``tensors[0]``'s device.  ``tensors``: what must outlive the
    launch where it came from another stream (tensors allocated for this call need not be named)."""
    call = getattr(_lib.library(), name)
    index = tensors[0].get_device()
    if index == torch.cuda.current_device():
        status = _on_stream(call, args, tensors, index)
    else:
        with torch.cuda.device(index):
            status = _on_stream(call, args, tensors, index)
    if status:
        raise RuntimeError(f"{name} returned CUDA error {status}")


_streams = {}  # (device, handle) -> Stream: making the object again costs more than a small launch


def _on_stream(call, args, tensors, index):
    handle = torch._C._cuda_getCurrentRawStream(index)
    stream = _streams.get((index, handle))
    if stream is None:
        stream = _streams[index, handle] = torch.cuda.current_stream(index)
    status = call(*args, handle)
    for t in tensors:
        if t is not None and t.numel():
            t.record_stream(stream)
    return status


def _check(tensors):
    index, differentiable = tensors[0].get_device(), torch.is_grad_enabled()
    for t in tensors:
        if t.get_device() != index or not t.is_cuda or t.dtype is not torch.float64:
            raise ValueError("same-device CUDA FP64 tensors required")
        if not t.is_contiguous():
            raise ValueError("contiguous tensors required")
        if differentiable and t.requires_grad:
            raise NotImplementedError("manual parameter VJP; double backward/HVP unsupported")


@lru_cache(256)
def _scratch_doubles(name, index, *sizes):
    size = ctypes.c_size_t()
    with torch.cuda.device(index):
        _lib.check(getattr(_lib.library(), name)(*sizes, ctypes.byref(size)), name)
    return (size.value + 7) // 8


def _scratch(name, like, *sizes):
    """Scratch of the size that entry point ``name`` gives for these sizes on ``like``'s device."""
    return like.new_empty((_scratch_doubles(name, like.get_device(), *sizes),))


def _affine_shape(hidden, weight):
    if weight.ndim != 2 or weight.shape[0] < 1 or weight.shape[1] != hidden.shape[1]:
        raise ValueError("expected H[rows,Cin], W[Cout,Cin]")
    return weight.shape


class _PackedActivation:
    def __init__(self, layout):
        self.layout = layout

    def forward(self, value):
        layout = self.layout
        _check((value,))
        layout.check(value)
        out = torch.empty_like(value)
        aux = value.new_empty((layout.points, value.shape[1]))
        _launch("flashns_v8_activation", [layout.dimension, 0, _ptr(value), None, None, _ptr(out), _ptr(aux),
                                          layout.full_points, layout.value_points, value.shape[1]],
                (value, out, aux))
        return out, aux

    def vjp(self, hidden, aux, seed):
        layout = self.layout
        _check((hidden, aux, seed))
        layout.check(hidden)
        layout.check(seed)
        if aux.shape != (layout.points, hidden.shape[1]) or seed.shape != hidden.shape:
            raise ValueError("auxiliary/adjoint shape mismatch")
        out = torch.empty_like(hidden)
        _launch("flashns_v8_activation", [layout.dimension, 1, _ptr(hidden), _ptr(aux), _ptr(seed), _ptr(out), None,
                                          layout.full_points, layout.value_points, hidden.shape[1]],
                (hidden, aux, seed, out))
        return out


class NativeCUDA:
    """Packed-layout hooks (``experiments/pinn_v8/native.py:11-221``)."""

    def __init__(self, build_directory=None):
        _lib.library()
        self.metadata = {"library": str(_lib.LIBRARY), "precision": "FP64", "arch": "sm_100a"}

    def activation_factory(self, layout):
        return _PackedActivation(layout)

    def coordinate_affine(self, layout, coordinates, weight, bias):
        return self._coordinate_affine(layout, coordinates, weight, bias, activation=False)

    def coordinate_affine_activation(self, layout, coordinates, weight, bias):
        return self._coordinate_affine(layout, coordinates, weight, bias, activation=True)

    def _coordinate_affine(self, layout, coordinates, weight, bias, *, activation):
        tensors = (coordinates, weight, bias)
        _check(tensors)
        if coordinates.shape != (layout.points, layout.dimension) or weight.ndim != 2:
            raise ValueError("coordinates must match the physical-coordinate layout")
        channels = weight.shape[0]
        if channels < 1 or weight.shape[1] != layout.dimension or bias.shape != (channels,):
            raise ValueError("expected W[C,dimension], bias[C]")
        out = coordinates.new_empty((layout.rows, channels))
        if activation:
            aux = coordinates.new_empty((layout.points, channels))
            _launch("flashns_v8_coordinate_affine_activation",
                    [layout.dimension, *map(_ptr, tensors), _ptr(out), _ptr(aux), layout.full_points,
                     layout.value_points, channels], (*tensors, out, aux))
            return out, aux
        _launch("flashns_v8_coordinate_affine", [layout.dimension, *map(_ptr, tensors), _ptr(out), layout.full_points,
                                                 layout.value_points, channels], (*tensors, out))
        return out

    def coordinate_wgrad(self, layout, coordinates, derivative):
        tensors = (coordinates, derivative)
        _check(tensors)
        layout.check(derivative)
        channels = derivative.shape[1]
        if coordinates.shape != (layout.points, layout.dimension):
            raise ValueError("expected coordinates[points,dimension], bar_Z[rows,C]")
        partials = derivative.new_empty(((layout.points + 7) // 8, channels, layout.dimension + 1))
        dw = derivative.new_empty((channels, layout.dimension))
        db = derivative.new_empty((channels,))
        _launch("flashns_v8_coordinate_wgrad", [layout.dimension, _ptr(derivative), _ptr(coordinates), _ptr(partials),
                                                _ptr(dw), _ptr(db), layout.full_points, layout.value_points, channels],
                (*tensors, partials, dw, db))
        return dw, db

    def coordinate_activation_wgrad(self, layout, coordinates, hidden, aux, seed):
        tensors = (coordinates, hidden, aux, seed)
        _check(tensors)
        layout.check(hidden)
        layout.check(seed)
        channels = hidden.shape[1]
        if coordinates.shape != (layout.points, layout.dimension) or seed.shape != hidden.shape \
                or aux.shape != (layout.points, channels):
            raise ValueError("expected x[points,dimension], H/bar_H[rows,C], a1[points,C]")
        partials = hidden.new_empty(((layout.points + 7) // 8, channels, layout.dimension + 1))
        dw, db = hidden.new_empty((channels, layout.dimension)), hidden.new_empty((channels,))
        _launch("flashns_v8_coordinate_activation_wgrad",
                [layout.dimension, _ptr(hidden), _ptr(aux), _ptr(seed), _ptr(coordinates), _ptr(partials), _ptr(dw),
                 _ptr(db), layout.full_points, layout.value_points, channels], (*tensors, partials, dw, db))
        return dw, db

    def tail_dgrad_vjp(self, layout, d, weight, hidden, aux, *, backend="F3"):
        if backend not in ("U3", "F3"):
            raise ValueError("packed tail backend must be U3 or F3")
        tensors = (d, weight, hidden, aux)
        _check(tensors)
        layout.check(d)
        layout.check(hidden)
        channels = hidden.shape[1]
        if d.shape != (layout.rows, 3) or weight.shape != (3, channels) or aux.shape != (layout.points, channels):
            raise ValueError("expected D[rows,3], W[3,C], H[rows,C], aux[points,C]")
        out = torch.empty_like(hidden)
        _launch("flashns_v8_tail3", [layout.dimension, int(backend == "F3"), *map(_ptr, tensors), _ptr(out),
                                     layout.full_points, layout.value_points, channels], (*tensors, out))
        if backend == "U3":
            return self.activation_factory(layout).vjp(hidden, aux, out)
        return out

    def seed(self, jets, boundary, pde_weights, boundary_weights, target, loss):
        ni, nb = len(jets), len(boundary)
        for t in (jets, boundary, pde_weights, boundary_weights, target):
            if not t.is_cuda or t.dtype != torch.float64 or t.device != jets.device:
                raise ValueError("same-device CUDA FP64 tensors required")
        if jets.shape != (ni, 10, 3) or boundary.shape != (nb, 3) or boundary.stride(-1) != 1:
            raise ValueError("2-D Q10 interior and contiguous-channel boundary fields required")
        if nb > 1 and boundary.stride(0) < 3:
            raise ValueError("boundary rows must not overlap or broadcast")
        if pde_weights.shape != (ni,) or boundary_weights.shape != (nb, 3) or target.shape != (nb, 3):
            raise ValueError("objective shape mismatch")
        if not all(t.is_contiguous() for t in (jets, pde_weights, boundary_weights, target)):
            raise ValueError("contiguous jet/weight/target storage required")
        di, db = torch.empty_like(jets), boundary.new_empty((nb, 3))
        partial = jets.new_empty(((ni + nb + 127) // 128,))
        boundary_ptr = ctypes.c_void_p(boundary.data_ptr()) if nb else None
        _launch("flashns_v8_loss_seed",
                [_ptr(jets), boundary_ptr, _ptr(pde_weights), _ptr(boundary_weights), _ptr(target), _ptr(di), _ptr(db),
                 _ptr(partial), ni, nb, max(3, boundary.stride(0)) if nb else 3, loss.viscosity,
                 loss.gradient_weight, loss.boundary_weight], (jets, pde_weights, boundary_weights, target, di, db,
                                                               partial))
        return partial.sum(), di, db


    def layer_norm(self, layout, value, gain, bias, *, eps=1e-5):
        """Layer norm over the channels, carried through the jets: ``(out, stats)``.

        The order-0 row of a point is its ordinary layer norm; the other rows are the exact
        Taylor coefficients of the normalized field.  ``stats[rows, 2]`` holds each row's mean
        and reciprocal-deviation coefficients for ``layer_norm_vjp``."""
        _check((value, gain, bias))
        layout.check(value)
        rows, channels = value.shape
        if gain.shape != (channels,) or bias.shape != (channels,):
            raise ValueError("expected gain[C], bias[C]")
        eps = float(eps)
        if not 0.0 < eps <= 1e300:
            raise ValueError("positive finite eps required")
        out, stats = torch.empty_like(value), value.new_empty((rows, 2))
        _launch("flashns_b200_layer_norm", [layout.dimension, *map(_ptr, (value, gain, bias, out, stats)), eps,
                                            layout.full_points, layout.value_points, channels],
                (value, gain, bias))
        return out, stats

    def layer_norm_vjp(self, layout, value, gain, stats, seed, *, skip=None):
        """``(d_value, d_gain, d_bias)`` of ``layer_norm`` at ``seed``; ``skip`` is added to ``d_value``
        (the gradient that reaches ``value`` past the norm, in a residual block)."""
        given = (value, gain, stats, seed) if skip is None else (value, gain, stats, seed, skip)
        _check(given)
        layout.check(value)
        rows, channels = value.shape
        if gain.shape != (channels,) or stats.shape != (rows, 2) or seed.shape != value.shape \
                or (skip is not None and skip.shape != value.shape):
            raise ValueError("expected X/bar_Y[rows,C], gain[C], stats[rows,2]")
        out, dgain, dbias = torch.empty_like(value), torch.empty_like(gain), torch.empty_like(gain)
        scratch = _scratch("flashns_b200_layer_norm_vjp_scratch", value, layout.dimension, layout.full_points,
                           layout.value_points, channels)
        _launch("flashns_b200_layer_norm_vjp",
                [layout.dimension, *map(_ptr, (value, gain, stats, seed, skip, out, dgain, dbias, scratch)),
                 scratch.numel() * 8, layout.full_points, layout.value_points, channels], given)
        return out, dgain, dbias

    def affine(self, layout, hidden, weight, bias, *, residual=None):
        """``H W^T`` with the bias on order-0 rows, plus ``residual``."""
        return self._affine(layout, hidden, weight, bias, residual, activation=False, keep=False)

    def affine_activation(self, layout, hidden, weight, bias, *, residual=None, keep=True):
        """The stable tanh jet of ``H W^T + b``, plus ``residual``: ``(out, activated, aux)`` with what
        ``affine_activation_vjp`` needs, or ``out`` alone when not ``keep``.  Without a residual
        ``activated`` is ``out``."""
        return self._affine(layout, hidden, weight, bias, residual, activation=True, keep=keep)

    def _affine(self, layout, hidden, weight, bias, residual, *, activation, keep):
        given = (hidden, weight, bias) if residual is None else (hidden, weight, bias, residual)
        _check(given)
        layout.check(hidden)
        cout, cin = _affine_shape(hidden, weight)
        if bias.shape != (cout,) or (residual is not None and residual.shape != (layout.rows, cout)):
            raise ValueError("expected H[rows,Cin], W[Cout,Cin], bias[Cout], residual[rows,Cout]")
        out = hidden.new_empty((layout.rows, cout))
        aux = hidden.new_empty((layout.points, cout)) if keep else None
        activated = torch.empty_like(out) if keep and residual is not None else None
        _launch("flashns_b200_affine",
                [layout.dimension, int(activation), *map(_ptr, (hidden, weight, bias, residual, out, activated, aux)),
                 layout.full_points, layout.value_points, cin, cout], given)
        return (out, out if activated is None else activated, aux) if keep else out

    def affine_vjp(self, layout, hidden, weight, seed):
        """``(d_hidden, d_weight, d_bias)`` of ``affine`` at ``seed`` (which is the residual's gradient too)."""
        return self._affine_vjp(layout, hidden, weight, None, None, seed)

    def affine_activation_vjp(self, layout, hidden, weight, activated, aux, seed):
        """``(d_hidden, d_weight, d_bias)`` of ``affine_activation`` at ``seed`` (which is the residual's
        gradient too)."""
        return self._affine_vjp(layout, hidden, weight, activated, aux, seed)

    def _affine_vjp(self, layout, hidden, weight, activated, aux, seed):
        given = (hidden, weight, seed) if activated is None else (hidden, weight, seed, activated, aux)
        _check(given)
        layout.check(hidden)
        cout, cin = _affine_shape(hidden, weight)
        if seed.shape != (hidden.shape[0], cout):
            raise ValueError("expected H[rows,Cin], W[Cout,Cin], bar_Y[rows,Cout]")
        if activated is not None and (activated.shape != seed.shape or aux.shape != (layout.points, cout)):
            raise ValueError("auxiliary/adjoint shape mismatch")
        activation = int(activated is not None)
        out, dw, db = torch.empty_like(hidden), torch.empty_like(weight), weight.new_empty((cout,))
        scratch = _scratch("flashns_b200_affine_vjp_scratch", hidden, layout.dimension, activation,
                           layout.full_points, layout.value_points, cin, cout)
        _launch("flashns_b200_affine_vjp",
                [layout.dimension, activation,
                 *map(_ptr, (hidden, weight, activated, aux, seed, out, dw, db, scratch)), scratch.numel() * 8,
                 layout.full_points, layout.value_points, cin, cout], given)
        return out, dw, db


class Native:
    """Dense ``[B,Q,C]`` hooks (``experiments/cuda_jet_h100/gpu.py``): forward, vjp, dgrad."""

    BACKENDS = ("B1", "F", "F_n32", "U3", "F3")

    def __init__(self, *args, **kwargs):
        _lib.library()

    def forward(self, value, dim):
        q = JetSpec(dim).q
        _check((value,))
        if value.ndim != 3 or value.shape[1] != q:
            raise ValueError("expected canonical full [B,Q,C] jets")
        hidden = torch.empty_like(value)
        aux = value.new_empty((value.shape[0], value.shape[2]))
        _launch("flashns_stable_activation", [dim, False, _ptr(value), None, None, _ptr(hidden), _ptr(aux),
                                              value.shape[0], value.shape[2]], (value, hidden, aux))
        return hidden, aux

    def vjp(self, hidden, aux, adjoint, dim):
        q = JetSpec(dim).q
        _check((hidden, aux, adjoint))
        if hidden.ndim != 3 or hidden.shape[1] != q or adjoint.shape != hidden.shape \
                or aux.shape != (hidden.shape[0], hidden.shape[2]):
            raise ValueError("incompatible full jets, auxiliary state or adjoint")
        out = torch.empty_like(hidden)
        _launch("flashns_stable_activation", [dim, True, _ptr(hidden), _ptr(adjoint), _ptr(aux), _ptr(out), None,
                                              hidden.shape[0], hidden.shape[2]], (hidden, aux, adjoint, out))
        return out

    def dgrad(self, d, weight, hidden, aux, dim, backend="B1"):
        if backend not in self.BACKENDS:
            raise ValueError(f"unknown backend {backend}")
        q = JetSpec(dim).q
        _check((d, weight, hidden, aux))
        if d.ndim != 3 or d.shape[1] != q or weight.ndim != 2 or d.shape[2] != weight.shape[0] \
                or hidden.shape != (d.shape[0], q, weight.shape[1]) or aux.shape != (d.shape[0], weight.shape[1]) \
                or weight.shape[0] == 0:
            raise ValueError("expected D[B,Q,Cout], W[Cout,Cin], H[B,Q,Cin], aux[B,Cin]")
        out = torch.empty_like(hidden)
        tensors = (d, weight, hidden, aux, out)
        if backend in ("U3", "F3") and weight.shape[0] == 3:
            _launch("flashns_stable_tail3", [dim, backend == "F3", *map(_ptr, tensors), d.shape[0], weight.shape[1]],
                    tensors)
            return out if backend == "F3" else self.vjp(hidden, aux, out, dim)
        fused = backend.startswith("F")
        _launch("flashns_stable_dgrad_vjp", [dim, fused, *map(_ptr, tensors), d.shape[0], weight.shape[0],
                                             weight.shape[1]], tensors)
        return out if fused else self.vjp(hidden, aux, out, dim)
