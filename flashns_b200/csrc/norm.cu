// Layer norm over the channels, propagated through packed jets, and its adjoint.
//
// With * the truncated product of a point's order-3 jets (on value rows: of numbers):
//   mu = mean_c X_c,  D_c = X_c - mu,  v = mean_c D_c * D_c,  r = (v + eps)^(-1/2),
//   Y_c = gain_c (r * D_c) + [order 0] bias_c.
// Adjoint at G, with corr(a, s)_k = sum_j a_j s_(j+k) the transpose of b -> a * b:
//   S = sum_c gain_c corr(D_c, G_c),  M = mean_c gain_c G_c,  w = corr(-r * r * r, S) / C,
//   dX_c = corr(r, gain_c G_c - M) + corr(D_c, w) [+ skip_c],
//   dgain_c = sum over points of <r, corr(D_c, G_c)>,  dbias_c = sum over points of G_(0,c).
// (sum_c D_c = 0, so the mean's share of dX passes through the first term alone.)
#include "flashns_b200.h"
#include "layers.cuh"

namespace flashns_b200 {
namespace {

constexpr int kNormThreads = 128;

// sums of N values over the block's threads, in every thread
template <int N>
__device__ __forceinline__ void block_sums(double (&v)[N], double* shared) {
  lane_sums<N, 16>(v);
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  __syncthreads();  // the previous sums have been read
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) shared[warp * N + i] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    double s = shared[i];
    for (int w = 1; w < warps; ++w) s += shared[w * N + i];
    v[i] = s;
  }
}

// any width: one block per unit, its channels read again for each pass
template <int DIM>
__global__ void __launch_bounds__(kNormThreads)
    norm_forward(const double* __restrict__ x, const double* __restrict__ gain, const double* __restrict__ bias,
                 double* __restrict__ out, double* __restrict__ stats, double eps, Packed rows, int channels) {
  constexpr int Q = Jet<DIM>::Q;
  __shared__ double shared[(kNormThreads / 32) * Q];
  const int64_t units = rows.units<Q>();
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const bool full = u < rows.full;
    const int n = rows.count<Q>(u);
    const int64_t row = rows.row<Q>(u);
    const double* xu = x + row * channels;
    double mean[Q], v[Q], r[Q];
#pragma unroll
    for (int s = 0; s < Q; ++s) mean[s] = v[s] = 0.0;
    for (int c = threadIdx.x; c < channels; c += blockDim.x) {
#pragma unroll
      for (int s = 0; s < Q; ++s)
        if (s < n) mean[s] += xu[int64_t(s) * channels + c];
    }
    block_sums(mean, shared);
#pragma unroll
    for (int s = 0; s < Q; ++s) mean[s] /= channels;
    for (int c = threadIdx.x; c < channels; c += blockDim.x) {
      double d[Q], p[Q];
#pragma unroll
      for (int s = 0; s < Q; ++s) d[s] = s < n ? xu[int64_t(s) * channels + c] - mean[s] : 0.0;
      if (full) {
        Jet<DIM>::square(d, p);
      } else {
#pragma unroll
        for (int s = 0; s < Q; ++s) p[s] = d[s] * d[s];
      }
#pragma unroll
      for (int s = 0; s < Q; ++s) v[s] += p[s];
    }
    block_sums(v, shared);
#pragma unroll
    for (int s = 0; s < Q; ++s) v[s] /= channels;
    if (full) {
      v[0] += eps;
      Jet<DIM>::rsqrt(v, r);
    } else {
#pragma unroll
      for (int s = 0; s < Q; ++s) r[s] = 1.0 / sqrt(v[s] + eps);
    }
    if (threadIdx.x == 0) {
#pragma unroll
      for (int s = 0; s < Q; ++s)
        if (s < n) {
          stats[2 * (row + s)] = mean[s];
          stats[2 * (row + s) + 1] = r[s];
        }
    }
    for (int c = threadIdx.x; c < channels; c += blockDim.x) {
      double d[Q], y[Q];
      const double gc = gain[c], bc = bias[c];
#pragma unroll
      for (int s = 0; s < Q; ++s) d[s] = s < n ? xu[int64_t(s) * channels + c] - mean[s] : 0.0;
      if (full) {
        Jet<DIM>::mul(r, d, y);
      } else {
#pragma unroll
        for (int s = 0; s < Q; ++s) y[s] = r[s] * d[s];
      }
#pragma unroll
      for (int s = 0; s < Q; ++s)
        if (s < n) out[(row + s) * channels + c] = gc * y[s] + (s == 0 || !full ? bc : 0.0);
    }
  }
}

// any width; partials [grid][2][channels]: this block's dgain and dbias
template <int DIM>
__global__ void __launch_bounds__(kNormThreads)
    norm_backward(const double* __restrict__ x, const double* __restrict__ gain, const double* __restrict__ stats,
                  const double* __restrict__ seed, const double* __restrict__ skip, double* __restrict__ dx,
                  double* __restrict__ partials, Packed rows, int channels) {
  constexpr int Q = Jet<DIM>::Q;
  __shared__ double shared[(kNormThreads / 32) * 2 * Q];
  double* mine = partials + int64_t(blockIdx.x) * 2 * channels;
  for (int c = threadIdx.x; c < channels; c += blockDim.x) mine[c] = mine[channels + c] = 0.0;
  const int64_t units = rows.units<Q>();
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const bool full = u < rows.full;
    const int n = rows.count<Q>(u);
    const int64_t row = rows.row<Q>(u);
    double mean[Q], r[Q], sums[2 * Q], w[Q];
#pragma unroll
    for (int s = 0; s < Q; ++s) {
      mean[s] = s < n ? stats[2 * (row + s)] : 0.0;
      r[s] = s < n ? stats[2 * (row + s) + 1] : 0.0;
      sums[s] = sums[Q + s] = 0.0;
    }
    for (int c = threadIdx.x; c < channels; c += blockDim.x) {
      double d[Q], g[Q], p[Q];
      const double gc = gain[c];
      double dgain = 0.0, dbias = 0.0;
#pragma unroll
      for (int s = 0; s < Q; ++s) {
        const int64_t at = (row + s) * channels + c;
        d[s] = s < n ? x[at] - mean[s] : 0.0;
        g[s] = s < n ? seed[at] : 0.0;
      }
      if (full) {
        Jet<DIM>::corr(d, g, p);
        dbias = g[0];
      } else {
#pragma unroll
        for (int s = 0; s < Q; ++s) {
          p[s] = d[s] * g[s];
          dbias += g[s];
        }
      }
#pragma unroll
      for (int s = 0; s < Q; ++s) {
        dgain += r[s] * p[s];
        sums[s] += gc * p[s];
        sums[Q + s] += gc * g[s];
      }
      mine[c] += dgain;
      mine[channels + c] += dbias;
    }
    block_sums(sums, shared);
    if (full) {
      double r2[Q], r3[Q];
      Jet<DIM>::mul(r, r, r2);
      Jet<DIM>::mul(r2, r, r3);
      Jet<DIM>::corr(r3, sums, w);
    } else {
#pragma unroll
      for (int s = 0; s < Q; ++s) w[s] = r[s] * r[s] * r[s] * sums[s];
    }
#pragma unroll
    for (int s = 0; s < Q; ++s) {
      w[s] = -w[s] / channels;
      sums[Q + s] /= channels;
    }
    for (int c = threadIdx.x; c < channels; c += blockDim.x) {
      double d[Q], g[Q], y[Q];
      const double gc = gain[c];
#pragma unroll
      for (int s = 0; s < Q; ++s) {
        const int64_t at = (row + s) * channels + c;
        d[s] = s < n ? x[at] - mean[s] : 0.0;
        g[s] = s < n ? gc * seed[at] - sums[Q + s] : 0.0;
      }
      if (full) {
        Jet<DIM>::corr(r, g, y);
        Jet<DIM>::corr_add(d, w, y);
      } else {
#pragma unroll
        for (int s = 0; s < Q; ++s) y[s] = r[s] * g[s] + d[s] * w[s];
      }
#pragma unroll
      for (int s = 0; s < Q; ++s) {
        if (s >= n) continue;
        const int64_t at = (row + s) * channels + c;
        dx[at] = skip ? y[s] + skip[at] : y[s];
      }
    }
  }
}

// dgain, dbias [channels] each from partials [parts][2][channels], summed in block order
__global__ void __launch_bounds__(kNormThreads)
    norm_finish(const double* __restrict__ partials, int parts, double* __restrict__ dgain, double* __restrict__ dbias,
                int channels) {
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < 2 * channels; i += gridDim.x * blockDim.x) {
    double s = 0.0;
    for (int k = 0; k < parts; ++k) s += partials[int64_t(k) * 2 * channels + i];
    if (i < channels) dgain[i] = s;
    else dbias[i - channels] = s;
  }
}

// blocks of the backward kernel: each keeps one [2][channels] partial
int64_t norm_parts(int dim, Packed rows, int sms) {
  const int64_t units = dim == 2 ? rows.units<10>() : rows.units<20>(), most = int64_t(sms) * 8;
  return units < most ? units : most;
}

}  // namespace
}  // namespace flashns_b200

using namespace flashns_b200;

extern "C" {

int flashns_b200_layer_norm(int dim, const double* value, const double* gain, const double* bias, double* out,
                            double* stats, double eps, int64_t full_points, int64_t value_points, int channels,
                            cudaStream_t stream) {
  if (!layer_sizes_ok(dim, full_points, value_points, channels) || !(eps > 0.0) || eps > 1e300)
    return int(cudaErrorInvalidValue);
  const Packed rows{full_points, value_points};
  const int64_t count = full_points * (dim == 2 ? 10 : 20) + value_points;
  if (count == 0) return int(cudaSuccess);
  if (!value || !gain || !bias || !out || !stats) return int(cudaErrorInvalidValue);
  const size_t bytes = size_t(count) * channels * sizeof(double), small = size_t(channels) * sizeof(double);
  const size_t stat = size_t(count) * 2 * sizeof(double);
  if (ranges_overlap(out, bytes, value, bytes) || ranges_overlap(stats, stat, value, bytes) ||
      ranges_overlap(out, bytes, stats, stat) || ranges_overlap(out, bytes, gain, small) ||
      ranges_overlap(out, bytes, bias, small))
    return int(cudaErrorInvalidValue);
  int sms = 0;
  cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return int(e);
  const unsigned grid = unsigned(norm_parts(dim, rows, sms));
  if (dim == 2) norm_forward<2><<<grid, kNormThreads, 0, stream>>>(value, gain, bias, out, stats, eps, rows, channels);
  else norm_forward<3><<<grid, kNormThreads, 0, stream>>>(value, gain, bias, out, stats, eps, rows, channels);
  return int(cudaGetLastError());
}

int flashns_b200_layer_norm_vjp_scratch(int dim, int64_t full_points, int64_t value_points, int channels,
                                        size_t* bytes) {
  if (!layer_sizes_ok(dim, full_points, value_points, channels) || !bytes) return int(cudaErrorInvalidValue);
  *bytes = 0;
  if (full_points + value_points == 0) return int(cudaSuccess);
  int sms = 0;
  cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return int(e);
  *bytes = size_t(norm_parts(dim, Packed{full_points, value_points}, sms)) * 2 * channels * sizeof(double);
  return int(cudaSuccess);
}

int flashns_b200_layer_norm_vjp(int dim, const double* value, const double* gain, const double* stats,
                                const double* seed, const double* skip, double* d_value, double* d_gain,
                                double* d_bias, double* scratch, size_t scratch_bytes, int64_t full_points,
                                int64_t value_points, int channels, cudaStream_t stream) {
  if (!layer_sizes_ok(dim, full_points, value_points, channels) || !d_gain || !d_bias)
    return int(cudaErrorInvalidValue);
  const Packed rows{full_points, value_points};
  const int64_t count = full_points * (dim == 2 ? 10 : 20) + value_points;
  const size_t small = size_t(channels) * sizeof(double);
  if (count == 0) {
    cudaError_t e = cudaMemsetAsync(d_gain, 0, small, stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(d_bias, 0, small, stream);
    return int(e);
  }
  if (!value || !gain || !stats || !seed || !d_value || !scratch) return int(cudaErrorInvalidValue);
  const size_t bytes = size_t(count) * channels * sizeof(double), stat = size_t(count) * 2 * sizeof(double);
  if (ranges_overlap(d_value, bytes, value, bytes) || ranges_overlap(d_value, bytes, seed, bytes) ||
      ranges_overlap(d_value, bytes, skip, bytes) || ranges_overlap(d_value, bytes, stats, stat) ||
      ranges_overlap(d_value, bytes, scratch, scratch_bytes))
    return int(cudaErrorInvalidValue);
  int sms = 0;
  cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return int(e);
  const int parts = int(norm_parts(dim, rows, sms));
  if (scratch_bytes < size_t(parts) * 2 * small) return int(cudaErrorInvalidValue);
  if (dim == 2) norm_backward<2><<<parts, kNormThreads, 0, stream>>>(value, gain, stats, seed, skip, d_value, scratch, rows, channels);
  else norm_backward<3><<<parts, kNormThreads, 0, stream>>>(value, gain, stats, seed, skip, d_value, scratch, rows, channels);
  e = cudaGetLastError();
  if (e != cudaSuccess) return int(e);
  norm_finish<<<(2 * channels + kNormThreads - 1) / kNormThreads, kNormThreads, 0, stream>>>(scratch, parts, d_gain, d_bias, channels);
  return int(cudaGetLastError());
}

}  // extern "C"
