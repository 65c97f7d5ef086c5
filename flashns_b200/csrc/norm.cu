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
#include <algorithm>
#include <type_traits>

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

// ---------------------------------------------------------------- a unit in registers
// T lanes of a warp, or W whole warps (a block), hold one unit: lane l has channels
// l, l + L, ... (L = T W lanes, K of them), all Q rows each, so every row is read once in
// 8-byte runs of L channels.  The sums over channels are K-term sums in the lane and a halving
// exchange over the lanes (lane_sums), joined over the warps through shared memory.
template <int N, int T, int W>
__device__ __forceinline__ void unit_sums(double (&v)[N], double* shared, int& turn) {
  if constexpr (W == 1) {
    lane_sums<N, T / 2>(v);
  } else {
    // two buffers in turn: one barrier separates a buffer's readers from its next writers
    double* sums = shared + (turn ^= 1) * W * N;
    const int warp = threadIdx.x >> 5;
    int first = 0, limit = N;
    lane_shares<N, 16>(v, first, limit);
#pragma unroll
    for (int i = 0; i < (N + 31) / 32; ++i)
      if (first + i < limit) sums[warp * N + first + i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      double s = sums[i];
#pragma unroll
      for (int w = 1; w < W; ++w) s += sums[w * N + i];
      v[i] = s;
    }
  }
}

template <int T, int W>
constexpr int unit_threads() { return W == 1 ? kNormThreads : 32 * W; }
template <int T, int W>
constexpr int unit_groups() { return W == 1 ? kNormThreads / T : 1; }

template <int DIM, int T, int K, int W>
__global__ void __launch_bounds__(unit_threads<T, W>())
    norm_forward_unit(const double* __restrict__ x, const double* __restrict__ gain, const double* __restrict__ bias,
                      double* __restrict__ out, double* __restrict__ stats, double eps, Packed rows, int channels) {
  constexpr int Q = Jet<DIM>::Q, L = T * W;
  __shared__ double shared[W > 1 ? 2 * W * Q : 1];
  int turn = 0;
  const int lane = W > 1 ? threadIdx.x : threadIdx.x % T;
  const int64_t u = int64_t(blockIdx.x) * unit_groups<T, W>() + (W > 1 ? 0 : threadIdx.x / T);
  const int n = u < rows.units<Q>() ? rows.count<Q>(u) : 0;  // no rows: the lanes only take part in the sums
  const bool full = u < rows.full;
  const int64_t row = rows.row<Q>(u);
  double d[K][Q], sums[Q], r[Q];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int s = 0; s < Q; ++s) {
      const int c = lane + k * L;
      d[k][s] = s < n && c < channels ? x[(row + s) * channels + c] : 0.0;
    }
  const double inv = 1.0 / channels;
#pragma unroll
  for (int s = 0; s < Q; ++s) {
    sums[s] = d[0][s];
#pragma unroll
    for (int k = 1; k < K; ++k) sums[s] += d[k][s];
  }
  unit_sums<Q, T, W>(sums, shared, turn);
  double mean[Q];
#pragma unroll
  for (int s = 0; s < Q; ++s) {
    mean[s] = sums[s] * inv;
    sums[s] = 0.0;
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (lane + k * L < channels) {
      double p[Q];
#pragma unroll
      for (int s = 0; s < Q; ++s) d[k][s] -= mean[s];
      if (full) {
        Jet<DIM>::square(d[k], p);
      } else {
#pragma unroll
        for (int s = 0; s < Q; ++s) p[s] = d[k][s] * d[k][s];
      }
#pragma unroll
      for (int s = 0; s < Q; ++s) sums[s] += p[s];
    }
  }
  unit_sums<Q, T, W>(sums, shared, turn);
#pragma unroll
  for (int s = 0; s < Q; ++s) sums[s] *= inv;
  if (full) {
    sums[0] += eps;
    Jet<DIM>::rsqrt(sums, r);
  } else {
#pragma unroll
    for (int s = 0; s < Q; ++s) r[s] = 1.0 / sqrt(sums[s] + eps);
  }
#pragma unroll
  for (int s = 0; s < Q; ++s)
    if (lane == s % L && s < n) {
      stats[2 * (row + s)] = mean[s];
      stats[2 * (row + s) + 1] = r[s];
    }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = lane + k * L;
    if (c < channels && n > 0) {
      const double gc = gain[c], bc = bias[c];
      double y[Q];
      if (full) {
        Jet<DIM>::mul(r, d[k], y);
      } else {
#pragma unroll
        for (int s = 0; s < Q; ++s) y[s] = r[s] * d[k][s];
      }
#pragma unroll
      for (int s = 0; s < Q; ++s)
        if (s < n) out[(row + s) * channels + c] = gc * y[s] + (s == 0 || !full ? bc : 0.0);
    }
  }
}

template <int DIM, int T, int K, int W>
__global__ void __launch_bounds__(unit_threads<T, W>())
    norm_backward_unit(const double* __restrict__ x, const double* __restrict__ gain, const double* __restrict__ stats,
                       const double* __restrict__ seed, const double* __restrict__ skip, double* __restrict__ dx,
                       double* __restrict__ partials, Packed rows, int channels) {
  constexpr int Q = Jet<DIM>::Q, L = T * W, G = unit_groups<T, W>();
  __shared__ double shared[W > 1 ? 4 * W * Q : 2 * K * kNormThreads];
  int turn = 0;
  const int lane = W > 1 ? threadIdx.x : threadIdx.x % T, group = W > 1 ? 0 : threadIdx.x / T;
  const int64_t units = rows.units<Q>();
  const double inv = 1.0 / channels;
  double gk[K], dgain[K], dbias[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    gk[k] = lane + k * L < channels ? gain[lane + k * L] : 0.0;
    dgain[k] = dbias[k] = 0.0;
  }
  // the block's groups step together, so that a group without a unit still takes part in the shuffles
  for (int64_t u0 = int64_t(blockIdx.x) * G; u0 < units; u0 += int64_t(gridDim.x) * G) {
    const int64_t u = u0 + group;
    const int n = u < units ? rows.count<Q>(u) : 0;
    const bool full = u < rows.full;
    const int64_t row = rows.row<Q>(u);
    double d[K][Q], g[K][Q], r[Q], sums[2 * Q], w[Q];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int s = 0; s < Q; ++s) {
        const int c = lane + k * L;
        const bool ok = s < n && c < channels;
        d[k][s] = ok ? x[(row + s) * channels + c] : 0.0;
        g[k][s] = ok ? seed[(row + s) * channels + c] : 0.0;
      }
#pragma unroll
    for (int s = 0; s < Q; ++s) {
      const double mean = s < n ? stats[2 * (row + s)] : 0.0;
      r[s] = s < n ? stats[2 * (row + s) + 1] : 0.0;
      sums[s] = sums[Q + s] = 0.0;
#pragma unroll
      for (int k = 0; k < K; ++k) d[k][s] = lane + k * L < channels ? d[k][s] - mean : 0.0;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      double p[Q];
      if (full) {
        Jet<DIM>::corr(d[k], g[k], p);
        dbias[k] += g[k][0];
      } else {
#pragma unroll
        for (int s = 0; s < Q; ++s) {
          p[s] = d[k][s] * g[k][s];
          dbias[k] += g[k][s];
        }
      }
#pragma unroll
      for (int s = 0; s < Q; ++s) {
        dgain[k] += r[s] * p[s];
        sums[s] += gk[k] * p[s];
        g[k][s] *= gk[k];
        sums[Q + s] += g[k][s];
      }
    }
    unit_sums<2 * Q, T, W>(sums, shared, turn);
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
      w[s] *= -inv;
      sums[Q + s] *= inv;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = lane + k * L;
      if (c >= channels) continue;
      double y[Q];
#pragma unroll
      for (int s = 0; s < Q; ++s) g[k][s] -= sums[Q + s];
      if (full) {
        Jet<DIM>::corr(r, g[k], y);
        Jet<DIM>::corr_add(d[k], w, y);
      } else {
#pragma unroll
        for (int s = 0; s < Q; ++s) y[s] = r[s] * g[k][s] + d[k][s] * w[s];
      }
#pragma unroll
      for (int s = 0; s < Q; ++s) {
        if (s >= n) continue;
        const int64_t at = (row + s) * channels + c;
        dx[at] = skip ? y[s] + skip[at] : y[s];
      }
    }
    __syncwarp();
  }
  double* mine = partials + int64_t(blockIdx.x) * 2 * channels;
  if constexpr (W > 1) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (lane + k * L < channels) {
        mine[lane + k * L] = dgain[k];
        mine[channels + lane + k * L] = dbias[k];
      }
  } else {  // the block's groups, in order
#pragma unroll
    for (int k = 0; k < K; ++k) {
      shared[(group * K + k) * T + lane] = dgain[k];
      shared[K * kNormThreads + (group * K + k) * T + lane] = dbias[k];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * K * T; i += kNormThreads) {
      const int which = i / (K * T), c = i % (K * T);
      double s = 0.0;
      for (int q = 0; q < G; ++q) s += shared[which * K * kNormThreads + q * K * T + c];
      if (c < channels) mine[which * channels + c] = s;
    }
  }
}

// dgain, dbias [channels] each from partials [parts][2][channels]: 8 strands of parts a value,
// each in order, then the strands in order
constexpr int kFinishStrands = 8, kFinishLanes = 32;
__global__ void __launch_bounds__(kFinishStrands* kFinishLanes)
    norm_finish(const double* __restrict__ partials, int parts, double* __restrict__ dgain, double* __restrict__ dbias,
                int channels) {
  __shared__ double shared[kFinishStrands][kFinishLanes];
  const int lane = threadIdx.x % kFinishLanes, strand = threadIdx.x / kFinishLanes;
  const int64_t i = int64_t(blockIdx.x) * kFinishLanes + lane, n = 2 * int64_t(channels);
  double s = 0.0;
  if (i < n) {
#pragma unroll 8
    for (int k = strand; k < parts; k += kFinishStrands) s += partials[k * n + i];
  }
  shared[strand][lane] = s;
  __syncthreads();
  if (strand == 0 && i < n) {
    for (int k = 1; k < kFinishStrands; ++k) s += shared[k][lane];
    if (i < channels) dgain[i] = s;
    else dbias[i - channels] = s;
  }
}

// How a unit is held at a width: calls f(T, K, W) (as integral constants), or says that no
// register form has it.
template <int V>
using Int = std::integral_constant<int, V>;
template <int DIM, bool BACKWARD, typename F>
bool with_unit(int channels, const F& f) {
  if (channels <= 16) return f(Int<8>{}, Int<2>{}, Int<1>{}), true;
  if (channels <= 32) return f(Int<16>{}, Int<2>{}, Int<1>{}), true;
  if constexpr (DIM == 2) {
    if (channels <= 64) return f(Int<32>{}, Int<2>{}, Int<1>{}), true;
    if (channels <= 128) return f(Int<32>{}, Int<2>{}, Int<2>{}), true;
    if (channels <= 256) return f(Int<32>{}, Int<2>{}, Int<4>{}), true;
  } else {
    if (channels <= 64) return f(Int<32>{}, Int<1>{}, Int<2>{}), true;
    if (channels <= 128) return f(Int<32>{}, Int<1>{}, Int<4>{}), true;
    if (channels <= 256) return f(Int<32>{}, Int<1>{}, Int<8>{}), true;
  }
  return false;
}

// blocks of the backward kernel, each of which keeps one [2][channels] partial: all that are
// resident at once (at most 16 a multiprocessor), or one for each of its units
int64_t norm_parts(int dim, Packed rows, int sms) {
  const int64_t units = dim == 2 ? rows.units<10>() : rows.units<20>(), most = int64_t(sms) * 8;
  return units < most ? units : most;
}

template <int DIM>
cudaError_t launch_norm(const double* x, const double* gain, const double* bias, double* out, double* stats, double eps,
                        Packed rows, int channels, int sms, cudaStream_t stream) {
  const int64_t units = rows.units<Jet<DIM>::Q>();
  const bool done = with_unit<DIM, false>(channels, [&](auto t, auto k, auto w) {
    constexpr int T = t, K = k, W = w, G = unit_groups<T, W>();
    norm_forward_unit<DIM, T, K, W><<<unsigned((units + G - 1) / G), unit_threads<T, W>(), 0, stream>>>(
        x, gain, bias, out, stats, eps, rows, channels);
  });
  if (!done)
    norm_forward<DIM><<<unsigned(norm_parts(DIM, rows, sms)), kNormThreads, 0, stream>>>(x, gain, bias, out, stats, eps,
                                                                                       rows, channels);
  return cudaGetLastError();
}

template <int DIM>
cudaError_t launch_norm_vjp(const double* x, const double* gain, const double* stats, const double* seed,
                            const double* skip, double* dx, double* dgain, double* dbias, double* partials, Packed rows,
                            int channels, int sms, cudaStream_t stream) {
  int64_t parts = norm_parts(DIM, rows, sms);
  const bool done = with_unit<DIM, true>(channels, [&](auto t, auto k, auto w) {
    constexpr int T = t, K = k, W = w, G = unit_groups<T, W>();
    const auto kernel = norm_backward_unit<DIM, T, K, W>;
    const int64_t blocks = (rows.units<Jet<DIM>::Q>() + G - 1) / G;
    int per_sm = 0;
    cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, unit_threads<T, W>(), 0);
    parts = std::min(std::min(parts, blocks), int64_t(sms) * (per_sm > 0 ? per_sm : 1));
    kernel<<<unsigned(parts), unit_threads<T, W>(), 0, stream>>>(x, gain, stats, seed, skip, dx, partials, rows, channels);
  });
  if (!done)
    norm_backward<DIM><<<unsigned(parts), kNormThreads, 0, stream>>>(x, gain, stats, seed, skip, dx, partials, rows, channels);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  norm_finish<<<unsigned((2 * int64_t(channels) + kFinishLanes - 1) / kFinishLanes), kFinishStrands * kFinishLanes, 0,
                stream>>>(partials, int(parts), dgain, dbias, channels);
  return cudaGetLastError();
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
  return int(dim == 2 ? launch_norm<2>(value, gain, bias, out, stats, eps, rows, channels, sms, stream)
                      : launch_norm<3>(value, gain, bias, out, stats, eps, rows, channels, sms, stream));
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
  if (scratch_bytes < size_t(norm_parts(dim, rows, sms)) * 2 * small) return int(cudaErrorInvalidValue);
  const auto launch = dim == 2 ? launch_norm_vjp<2> : launch_norm_vjp<3>;
  return int(launch(value, gain, stats, seed, skip, d_value, d_gain, d_bias, scratch, rows, channels, sms, stream));
}

}  // extern "C"
