// Hidden affine layer on packed jets with the tanh jet and a residual in its epilogue, and
// its adjoint.
//
//   Z = H W^T, + b on order-0 rows;  A = tanh jet(Z), a1 = sech^2 Z_0;  Y = A (+ R)
// (without the activation Y = Z (+ R)).  Adjoint at G, which is also R's gradient:
//   dZ = VJP of the tanh jet at (A, a1), G;  dH = dZ W;  dW = dZ^T H;  db = sum of order-0 dZ.
#include "flashns_b200.h"
#include "jets_generated.cuh"
#include "layers.cuh"

namespace flashns_b200 {
namespace {

constexpr int kAffThreads = 256;

template <int DIM>
__device__ __forceinline__ void tanh_forward(const double* z, double* h, double& a1) {
  if constexpr (DIM == 2) jet_fwd_2d3(z, h, a1); else jet_fwd_3d3(z, h, a1);
}
template <int DIM>
__device__ __forceinline__ void tanh_vjp(const double* h, double a1, const double* hb, double* zb) {
  if constexpr (DIM == 2) jet_vjp_2d3(h, a1, hb, zb); else jet_vjp_3d3(h, a1, hb, zb);
}

// one thread per (unit, output channel)
template <int DIM, bool ACT>
__global__ void __launch_bounds__(kAffThreads)
    affine_forward(const double* __restrict__ hidden, const double* __restrict__ weight, const double* __restrict__ bias,
                   const double* __restrict__ residual, double* __restrict__ out, double* __restrict__ activated,
                   double* __restrict__ aux, Packed rows, int cin, int cout) {
  constexpr int Q = Jet<DIM>::Q;
  const int64_t total = rows.units<Q>() * cout;
  for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += int64_t(gridDim.x) * blockDim.x) {
    const int64_t u = i / cout;
    const int c = int(i % cout), n = rows.count<Q>(u);
    const bool full = u < rows.full;
    const int64_t row = rows.row<Q>(u);
    double z[Q], h[Q];
#pragma unroll
    for (int s = 0; s < Q; ++s) z[s] = 0.0;
    for (int k = 0; k < cin; ++k) {
      const double w = weight[int64_t(c) * cin + k];
#pragma unroll
      for (int s = 0; s < Q; ++s)
        if (s < n) z[s] += w * hidden[(row + s) * cin + k];
    }
    const double b = bias[c];
#pragma unroll
    for (int s = 0; s < Q; ++s) {
      if (s == 0 || !full) z[s] += b;
      h[s] = z[s];
    }
    if constexpr (ACT) {
      if (full) {
        double a1;
        tanh_forward<DIM>(z, h, a1);
        if (aux) aux[u * cout + c] = a1;
      } else {
#pragma unroll
        for (int s = 0; s < Q; ++s) {
          double a1;
          jet_fwd_2d0(z + s, h + s, a1);
          if (aux && s < n) aux[(rows.full + (u - rows.full) * Q + s) * cout + c] = a1;
        }
      }
    }
#pragma unroll
    for (int s = 0; s < Q; ++s) {
      if (s >= n) continue;
      const int64_t at = (row + s) * cout + c;
      if (activated) activated[at] = h[s];
      out[at] = residual ? h[s] + residual[at] : h[s];
    }
  }
}

// dZ, one thread per (unit, output channel)
template <int DIM>
__global__ void __launch_bounds__(kAffThreads)
    affine_seed(const double* __restrict__ activated, const double* __restrict__ aux, const double* __restrict__ seed,
                double* __restrict__ dz, Packed rows, int cout) {
  constexpr int Q = Jet<DIM>::Q;
  const int64_t total = rows.units<Q>() * cout;
  for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += int64_t(gridDim.x) * blockDim.x) {
    const int64_t u = i / cout;
    const int c = int(i % cout), n = rows.count<Q>(u);
    const int64_t row = rows.row<Q>(u);
    if (u < rows.full) {
      double h[Q], g[Q], z[Q];
#pragma unroll
      for (int s = 0; s < Q; ++s) {
        h[s] = activated[(row + s) * cout + c];
        g[s] = seed[(row + s) * cout + c];
      }
      tanh_vjp<DIM>(h, aux[u * cout + c], g, z);
#pragma unroll
      for (int s = 0; s < Q; ++s) dz[(row + s) * cout + c] = z[s];
    } else {
      for (int s = 0; s < n; ++s)
        dz[(row + s) * cout + c] = seed[(row + s) * cout + c] * aux[(rows.full + (u - rows.full) * Q + s) * cout + c];
    }
  }
}

// dH = dZ W, one thread per element
__global__ void __launch_bounds__(kAffThreads)
    affine_dgrad(const double* __restrict__ dz, const double* __restrict__ weight, double* __restrict__ dh, int64_t rows,
                 int cin, int cout) {
  const int64_t total = rows * cin;
  for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += int64_t(gridDim.x) * blockDim.x) {
    const int64_t r = i / cin;
    const int k = int(i % cin);
    double s = 0.0;
    for (int c = 0; c < cout; ++c) s += dz[r * cout + c] * weight[int64_t(c) * cin + k];
    dh[i] = s;
  }
}

constexpr int kWgTile = 16, kWgParts = 64;

// partials[part][cout][cin + 1]: dW and, in the last column, db of the part's rows
__global__ void __launch_bounds__(kWgTile* kWgTile)
    affine_wgrad(const double* __restrict__ dz, const double* __restrict__ hidden, double* __restrict__ partials,
                 int64_t rows, int64_t full_rows, int q, int cin, int cout) {
  const int c = blockIdx.y * kWgTile + threadIdx.x / kWgTile, k = blockIdx.x * kWgTile + threadIdx.x % kWgTile;
  if (c >= cout || k > cin) return;
  const int64_t per = (rows + gridDim.z - 1) / gridDim.z, first = per * blockIdx.z;
  const int64_t last = first + per < rows ? first + per : rows;
  double s = 0.0;
  if (k < cin) {
    for (int64_t r = first; r < last; ++r) s += dz[r * cout + c] * hidden[r * cin + k];
  } else {
    for (int64_t r = first; r < last; ++r)
      if (r >= full_rows || r % q == 0) s += dz[r * cout + c];
  }
  partials[(int64_t(blockIdx.z) * cout + c) * (cin + 1) + k] = s;
}

__global__ void __launch_bounds__(kAffThreads)
    affine_finish(const double* __restrict__ partials, int parts, double* __restrict__ dw, double* __restrict__ db,
                  int cin, int cout) {
  const int64_t total = int64_t(cout) * (cin + 1);
  for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += int64_t(gridDim.x) * blockDim.x) {
    double s = 0.0;
    for (int p = 0; p < parts; ++p) s += partials[p * total + i];
    const int64_t c = i / (cin + 1);
    const int k = int(i % (cin + 1));
    if (k < cin) dw[c * cin + k] = s;
    else db[c] = s;
  }
}

unsigned grid_for(int64_t count) {
  const int64_t blocks = (count + kAffThreads - 1) / kAffThreads;
  return unsigned(blocks < (1 << 20) ? blocks : (1 << 20));
}

size_t affine_scratch(int64_t count, int cin, int cout, bool act) {
  return (size_t(kWgParts) * cout * (size_t(cin) + 1) + (act ? size_t(count) * cout : 0)) * sizeof(double);
}

}  // namespace
}  // namespace flashns_b200

using namespace flashns_b200;

extern "C" {

int flashns_b200_affine(int dim, int activation, const double* hidden, const double* weight, const double* bias,
                        const double* residual, double* out, double* activated, double* aux, int64_t full_points,
                        int64_t value_points, int cin, int cout, cudaStream_t stream) {
  if (!layer_sizes_ok(dim, full_points, value_points, cin) || !layer_sizes_ok(dim, full_points, value_points, cout) ||
      (activation != 0 && activation != 1) || (!activation && (activated || aux)))
    return int(cudaErrorInvalidValue);
  const Packed rows{full_points, value_points};
  const int64_t count = full_points * (dim == 2 ? 10 : 20) + value_points;
  if (count == 0) return int(cudaSuccess);
  if (!hidden || !weight || !bias || !out) return int(cudaErrorInvalidValue);
  const size_t in = size_t(count) * cin * sizeof(double), bytes = size_t(count) * cout * sizeof(double);
  if (ranges_overlap(out, bytes, hidden, in) || ranges_overlap(out, bytes, residual, bytes) ||
      ranges_overlap(activated, bytes, hidden, in) || ranges_overlap(activated, bytes, residual, bytes) ||
      ranges_overlap(out, bytes, activated, bytes))
    return int(cudaErrorInvalidValue);
  const unsigned grid = grid_for((dim == 2 ? rows.units<10>() : rows.units<20>()) * cout);
  if (dim == 2 && activation) affine_forward<2, true><<<grid, kAffThreads, 0, stream>>>(hidden, weight, bias, residual, out, activated, aux, rows, cin, cout);
  else if (dim == 2) affine_forward<2, false><<<grid, kAffThreads, 0, stream>>>(hidden, weight, bias, residual, out, activated, aux, rows, cin, cout);
  else if (activation) affine_forward<3, true><<<grid, kAffThreads, 0, stream>>>(hidden, weight, bias, residual, out, activated, aux, rows, cin, cout);
  else affine_forward<3, false><<<grid, kAffThreads, 0, stream>>>(hidden, weight, bias, residual, out, activated, aux, rows, cin, cout);
  return int(cudaGetLastError());
}

int flashns_b200_affine_vjp_scratch(int dim, int activation, int64_t full_points, int64_t value_points, int cin,
                                    int cout, size_t* bytes) {
  if (!layer_sizes_ok(dim, full_points, value_points, cin) || !layer_sizes_ok(dim, full_points, value_points, cout) ||
      (activation != 0 && activation != 1) || !bytes)
    return int(cudaErrorInvalidValue);
  const int64_t count = full_points * (dim == 2 ? 10 : 20) + value_points;
  *bytes = count ? affine_scratch(count, cin, cout, activation != 0) : 0;
  return int(cudaSuccess);
}

int flashns_b200_affine_vjp(int dim, int activation, const double* hidden, const double* weight,
                            const double* activated, const double* aux, const double* seed, double* d_hidden,
                            double* d_weight, double* d_bias, double* scratch, size_t scratch_bytes,
                            int64_t full_points, int64_t value_points, int cin, int cout, cudaStream_t stream) {
  if (!layer_sizes_ok(dim, full_points, value_points, cin) || !layer_sizes_ok(dim, full_points, value_points, cout) ||
      (activation != 0 && activation != 1) || !d_weight || !d_bias)
    return int(cudaErrorInvalidValue);
  const Packed rows{full_points, value_points};
  const int q = dim == 2 ? 10 : 20;
  const int64_t count = full_points * q + value_points;
  if (count == 0) {
    cudaError_t e = cudaMemsetAsync(d_weight, 0, size_t(cin) * cout * sizeof(double), stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(d_bias, 0, size_t(cout) * sizeof(double), stream);
    return int(e);
  }
  if (!hidden || !weight || !seed || !d_hidden || !scratch || (activation && (!activated || !aux)))
    return int(cudaErrorInvalidValue);
  const size_t in = size_t(count) * cin * sizeof(double), bytes = size_t(count) * cout * sizeof(double);
  if (scratch_bytes < affine_scratch(count, cin, cout, activation != 0) || ranges_overlap(d_hidden, in, hidden, in) ||
      ranges_overlap(d_hidden, in, seed, bytes) || ranges_overlap(d_hidden, in, activated, bytes) ||
      ranges_overlap(d_hidden, in, scratch, scratch_bytes))
    return int(cudaErrorInvalidValue);
  double* partials = scratch;
  const double* dz = seed;
  if (activation) {
    double* z = scratch + size_t(kWgParts) * cout * (size_t(cin) + 1);
    const unsigned grid = grid_for((dim == 2 ? rows.units<10>() : rows.units<20>()) * cout);
    if (dim == 2) affine_seed<2><<<grid, kAffThreads, 0, stream>>>(activated, aux, seed, z, rows, cout);
    else affine_seed<3><<<grid, kAffThreads, 0, stream>>>(activated, aux, seed, z, rows, cout);
    dz = z;
  }
  affine_dgrad<<<grid_for(count * cin), kAffThreads, 0, stream>>>(dz, weight, d_hidden, count, cin, cout);
  const dim3 grid(unsigned(cin / kWgTile + 1), unsigned((cout + kWgTile - 1) / kWgTile), kWgParts);
  affine_wgrad<<<grid, kWgTile * kWgTile, 0, stream>>>(dz, hidden, partials, count, full_points * q, q, cin, cout);
  affine_finish<<<grid_for(int64_t(cout) * (cin + 1)), kAffThreads, 0, stream>>>(partials, kWgParts, d_weight, d_bias, cin, cout);
  return int(cudaGetLastError());
}

}  // extern "C"
