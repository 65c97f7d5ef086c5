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

// any width; gain_parts, bias_parts [grid][channels]: this block's dgain and dbias
template <int DIM>
__global__ void __launch_bounds__(kNormThreads)
    norm_backward(const double* __restrict__ x, const double* __restrict__ gain, const double* __restrict__ stats,
                  const double* __restrict__ seed, const double* __restrict__ skip, double* __restrict__ dx,
                  double* __restrict__ gain_parts, double* __restrict__ bias_parts, Packed rows, int channels) {
  constexpr int Q = Jet<DIM>::Q;
  __shared__ double shared[(kNormThreads / 32) * 2 * Q];
  double *gains = gain_parts + int64_t(blockIdx.x) * channels, *biases = bias_parts + int64_t(blockIdx.x) * channels;
  for (int c = threadIdx.x; c < channels; c += blockDim.x) gains[c] = biases[c] = 0.0;
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
      gains[c] += dgain;
      biases[c] += dbias;
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

// ---------------------------------------------------------------- streamed units
// A group of W warps takes one unit at a time (T < 32 lanes of a warp: one each of several
// units, so that narrow layers fill their warps); lane l has channels l and l + T W (K of
// them).  HBM bounds the sizes that matter, but only while a unit costs few instructions: a
// value is 16 to 32 bytes and some 50 multiply-adds.  So
//   - a group copies its next unit, one contiguous run, into shared memory (cp.async, 16 bytes
//     where the width is even and the tensors aligned) while it works on this one; rows past
//     the last are copied as zeros, so no pass tests for them;
//   - a width that the lanes cover exactly is a constant, which leaves no address arithmetic in
//     the copies and passes (16,384 + 4,096 points, 64 wide: the adjoint 63 us against 86);
//   - sums over channels are a halving exchange over the lanes (each ends with its own few),
//     then shared memory joins the warps and hands all sums to all lanes.
// Blocks are persistent, one a multiprocessor; each has as many groups as its shared memory
// and registers hold.
//
// Measured: 16,384 + 4,096 points, 64 wide: 35 us (0.75 of the copy bandwidth; launch and first
// loads are 4), the adjoint with a skip 61 (0.87); 3-D 32,768 + 8,192 points, 128 wide: 259
// (0.81); the 3-D adjoint at 4,099 + 1,031 points, 100 wide: 66 (0.46): its 8 warps, for which
// there are registers, wait for one another's sums and on latency (0.44 instructions a cycle
// and scheduler), and each forms r * r * r and w for its point.
constexpr int kUnitMostLanes = 256;  // lanes of the widest group
constexpr size_t kUnitSmem = 226 * 1024;
template <int DIM, bool BACKWARD>
constexpr int unit_k() { return DIM == 3 && BACKWARD ? 1 : 2; }  // channels a lane
template <int DIM, bool BACKWARD>
constexpr int unit_warps() { return BACKWARD ? 8 : DIM == 2 ? 16 : 10; }  // most warps of a block
template <bool BACKWARD>
constexpr int unit_slots() { return BACKWARD ? 5 : 2; }  // X (and G) twice; skip

__device__ __forceinline__ void copy8(double* smem, const double* gmem, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;\n" ::"r"(smem_u32(smem)), "l"(gmem), "r"(valid ? 8 : 0));
}

template <int DIM, bool BACKWARD, int T, int W, bool EXACT>
struct Place {
  static constexpr int kDim = DIM;
  static constexpr bool kExact = EXACT;
  static constexpr int Q = Jet<DIM>::Q, K = unit_k<DIM, BACKWARD>(), L = T * W, N = BACKWARD ? 2 * Q : Q;
  static constexpr int kUnits = W > 1 ? 1 : 32 / T;         // units of a set, the group's step
  static constexpr int kThreads = 32 * W;                   // of a group
  static constexpr int kSlot = Q * K * kThreads;            // doubles of one set's values, at most
  static constexpr int kSums = (W > 1 ? 2 * W : kUnits) * N;  // one buffer of sums
  static constexpr int kStats = BACKWARD ? kUnits * 2 * Q : 0;
  static constexpr int kDoubles = unit_slots<BACKWARD>() * kSlot + 2 * kSums + 2 * kStats;
  static constexpr int kGroups = int(kUnitSmem / sizeof(double) / kDoubles) < unit_warps<DIM, BACKWARD>() / W
                                     ? int(kUnitSmem / sizeof(double) / kDoubles)
                                     : unit_warps<DIM, BACKWARD>() / W;
  static constexpr int kBlock = kGroups * kThreads;
  int group, sub, lane, in_group;
  __device__ Place()
      : group(threadIdx.x / kThreads), sub(W > 1 ? 0 : threadIdx.x % 32 / T), lane(threadIdx.x % L),
        in_group(threadIdx.x % kThreads) {}
  __device__ __forceinline__ void sync() const {
    if constexpr (W == 1) __syncwarp(); else named_sync(1 + group, kThreads);
  }
  __device__ __forceinline__ bool has(int k, int channels) const { return EXACT || lane + k * L < channels; }
  // the set's values (a contiguous run; rows past the last as zeros) into `slot`
  __device__ __forceinline__ void copy(double* slot, const double* __restrict__ from, int64_t set, int64_t total,
                                       int channels, bool vec) const {
    const int width = EXACT ? K * L : channels, values = kUnits * Q * width;
    const int64_t left = total * width - set * values;
    const double* src = from + set * values;
    if (EXACT && left >= values) {
      const unsigned to = smem_u32(slot + 2 * in_group);
#pragma unroll
      for (int i = 0; i < kSlot; i += 2 * kThreads)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to + 8u * i), "l"(src + 2 * in_group + i));
    } else if ((EXACT || vec) && (left >= values || left % 2 == 0)) {
      // rolled up: unrolled, every copy's address is kept in registers
#pragma unroll 2
      for (int i = 2 * in_group; i < values; i += 2 * kThreads) cp_async16(slot + i, i < left ? src + i : from, i < left);
    } else {
#pragma unroll 2
      for (int i = in_group; i < values; i += kThreads) copy8(slot + i, i < left ? src + i : from, i < left);
    }
  }
  // v: this lane's part of N sums; all of them in every lane of the unit
  __device__ __forceinline__ void sum(double (&v)[N], double* sums) const {
    int first = 0, limit = N;
    lane_shares<N, T / 2>(v, first, limit);
    double* mine = sums + (W > 1 ? in_group / 32 : sub) * N;
#pragma unroll
    for (int i = 0; i < (N + T - 1) / T + 1; ++i)
      if (first + i < limit) mine[first + i] = v[i];
    sync();
    if constexpr (W > 1) {  // every warp joins the warps' sums, a few a lane, into its own copy
      double* own = sums + W * N + in_group / 32 * N;
#pragma unroll
      for (int i = threadIdx.x % 32; i < N; i += 32) {
        double s = sums[i];
#pragma unroll
        for (int w = 1; w < W; ++w) s += sums[w * N + i];
        own[i] = s;
      }
      __syncwarp();
      mine = own;
    }
    const double2* all = reinterpret_cast<const double2*>(mine);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) v[2 * i] = all[i].x, v[2 * i + 1] = all[i].y;
    if constexpr (W > 1) __syncwarp();  // read before the next sums' copy
  }
  // rows row .. row + n - 1 of channel c
  __device__ __forceinline__ static void store(double* __restrict__ out, const double (&y)[Q], int64_t row, int n, int c,
                                               int channels) {
    if constexpr (EXACT) channels = K * L;
    double* to = out + row * channels + c;
    if (n == Q) {
#pragma unroll
      for (int s = 0; s < Q; ++s) to[int64_t(s) * channels] = y[s];
    } else {
#pragma unroll
      for (int s = 0; s < Q; ++s)
        if (s < n) to[int64_t(s) * channels] = y[s];
    }
  }
};

template <typename At>
__global__ void __launch_bounds__(At::kBlock, 1)
    norm_forward_unit(const double* __restrict__ x, const double* __restrict__ gain, const double* __restrict__ bias,
                      double* __restrict__ out, double* __restrict__ stats, double eps, Packed rows, int channels, bool vec) {
  constexpr int DIM = At::kDim, Q = At::Q, K = At::K, L = At::L;
  extern __shared__ __align__(16) double smem[];
  const At at;
  double* buffers = smem + at.group * At::kDoubles;
  double* sums_at = buffers + 2 * At::kSlot;
  const int width = At::kExact ? K * L : channels;
  const int64_t total = rows.full * Q + rows.value, units = rows.units<Q>(), sets = (units + At::kUnits - 1) / At::kUnits;
  const int64_t stride = int64_t(gridDim.x) * At::kGroups;
  const double inv = 1.0 / channels;
  double gk[K], bk[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = at.lane + k * L;
    gk[k] = c < channels ? gain[c] : 0.0;
    bk[k] = c < channels ? bias[c] : 0.0;
  }
  auto load = [&](int64_t set, int stage) {
    if (set < sets) at.copy(buffers + stage * At::kSlot, x, set, total, channels, vec);
    cp_async_commit();
  };
  int stage = 0;
  const int64_t first = blockIdx.x + int64_t(at.group) * gridDim.x;  // few units: one a block
  load(first, 0);
  for (int64_t set = first; set < sets; set += stride, stage ^= 1) {
    const int64_t u = set * At::kUnits + at.sub;
    const int n = u < units ? rows.count<Q>(u) : 0;  // no rows: the lanes only take part in the sums
    const bool full = u < rows.full;
    const int64_t row = rows.row<Q>(u);
    const double* xs = buffers + stage * At::kSlot + at.sub * Q * width + at.lane;
    double sums[Q], mean[Q], r[Q];
#pragma unroll
    for (int s = 0; s < Q; ++s) sums[s] = 0.0;
    cp_async_wait<0>();
    at.sync();  // the other lanes' copies; and the other stage has been read out
    load(set + stride, stage ^ 1);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!at.has(k, channels)) continue;
#pragma unroll
      for (int s = 0; s < Q; ++s) sums[s] += xs[k * L + s * width];
    }
    __syncwarp();
    at.sum(sums, sums_at);
#pragma unroll
    for (int s = 0; s < Q; ++s) {
      mean[s] = sums[s] * inv;
      sums[s] = 0.0;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!at.has(k, channels)) continue;
      double d[Q], p[Q];
#pragma unroll
      for (int s = 0; s < Q; ++s) d[s] = xs[k * L + s * width] - mean[s];
      if (full) {
        Jet<DIM>::square(d, p);
      } else {
#pragma unroll
        for (int s = 0; s < Q; ++s) p[s] = d[s] * d[s];
      }
#pragma unroll
      for (int s = 0; s < Q; ++s) sums[s] += p[s];
    }
    __syncwarp();
    at.sum(sums, sums_at + At::kSums);
#pragma unroll
    for (int s = 0; s < Q; ++s) sums[s] *= inv;
    if (full) {
      sums[0] += eps;
      Jet<DIM>::rsqrt(sums, r);
    } else {
#pragma unroll
      for (int s = 0; s < Q; ++s) r[s] = 1.0 / sqrt(sums[s] + eps);
    }
    if (at.lane == 0) {
      double* st = stats + 2 * row;
#pragma unroll
      for (int s = 0; s < Q; ++s)
        if (s < n) {
          st[2 * s] = mean[s];
          st[2 * s + 1] = r[s];
        }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = at.lane + k * L;
      if (!at.has(k, channels)) continue;
      double d[Q], y[Q];
#pragma unroll
      for (int s = 0; s < Q; ++s) d[s] = xs[k * L + s * width] - mean[s];
      if (full) {
        Jet<DIM>::mul(r, d, y);
#pragma unroll
        for (int s = 0; s < Q; ++s) y[s] = s == 0 ? gk[k] * y[s] + bk[k] : gk[k] * y[s];
      } else {
#pragma unroll
        for (int s = 0; s < Q; ++s) y[s] = gk[k] * (r[s] * d[s]) + bk[k];
      }
      At::store(out, y, row, n, c, channels);
    }
    __syncwarp();
  }
  cp_async_wait<0>();
}

template <typename At>
__global__ void __launch_bounds__(At::kBlock, 1)
    norm_backward_unit(const double* __restrict__ x, const double* __restrict__ gain, const double* __restrict__ stats,
                       const double* __restrict__ seed, const double* __restrict__ skip, double* __restrict__ dx,
                       double* __restrict__ gain_parts, double* __restrict__ bias_parts, Packed rows, int channels,
                       bool vec) {
  constexpr int DIM = At::kDim, Q = At::Q, K = At::K, L = At::L, TH = At::kThreads;
  extern __shared__ __align__(16) double smem[];
  const At at;
  double* buffers = smem + at.group * At::kDoubles;  // [2][X, G], skip
  double* sums_at = buffers + 5 * At::kSlot;
  const int width = At::kExact ? K * L : channels;
  double* stats_at = sums_at + 2 * At::kSums;  // [2][unit][Q] of (mean, r)
  const int64_t units = rows.units<Q>(), sets = (units + At::kUnits - 1) / At::kUnits;
  const int64_t stride = int64_t(gridDim.x) * At::kGroups, all_rows = rows.full * Q + rows.value;
  const double inv = 1.0 / channels;
  double gk[K], dgain[K], dbias[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    gk[k] = at.lane + k * L < channels ? gain[at.lane + k * L] : 0.0;
    dgain[k] = dbias[k] = 0.0;
  }
  auto load = [&](int64_t set, int stage) {
    if (set < sets) {
      double* slot = buffers + 2 * stage * At::kSlot;
      at.copy(slot, x, set, all_rows, channels, vec);
      at.copy(slot + At::kSlot, seed, set, all_rows, channels, vec);
#pragma unroll
      for (int i = 0; i < (At::kStats + TH - 1) / TH; ++i) {
        const int e = at.in_group + i * TH;
        const int64_t j = set * At::kStats + e;
        if (e < At::kStats) copy8(stats_at + stage * At::kStats + e, j < 2 * all_rows ? stats + j : stats, j < 2 * all_rows);
      }
    }
    cp_async_commit();
  };
  int stage = 0;
  const int64_t first = blockIdx.x + int64_t(at.group) * gridDim.x;
  load(first, 0);
  for (int64_t set = first; set < sets; set += stride, stage ^= 1) {
    const int64_t u = set * At::kUnits + at.sub;
    const int n = u < units ? rows.count<Q>(u) : 0;
    const bool full = u < rows.full;
    const int64_t row = rows.row<Q>(u);
    const double* xs = buffers + 2 * stage * At::kSlot + at.sub * Q * width + at.lane;
    const double *gs = xs + At::kSlot, *es = buffers + 4 * At::kSlot + at.sub * Q * width + at.lane;
    const double2* st = reinterpret_cast<const double2*>(stats_at + stage * At::kStats + at.sub * 2 * Q);
    double r[Q], sums[2 * Q], w[Q];
    cp_async_wait<0>();  // X, G and stats of this unit
    at.sync();           // the other lanes' copies; and the slots loaded next have been read out
    if (skip) at.copy(buffers + 4 * At::kSlot, skip, set, all_rows, channels, vec);
    cp_async_commit();
    load(set + stride, stage ^ 1);
#pragma unroll
    for (int s = 0; s < 2 * Q; ++s) sums[s] = 0.0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!at.has(k, channels)) continue;
      double d[Q], g[Q], p[Q];
#pragma unroll
      for (int s = 0; s < Q; ++s) {
        d[s] = xs[k * L + s * width] - st[s].x;
        g[s] = gs[k * L + s * width];
      }
      if (full) {
        Jet<DIM>::corr(d, g, p);
        dbias[k] += g[0];
      } else {
#pragma unroll
        for (int s = 0; s < Q; ++s) {
          p[s] = d[s] * g[s];
          dbias[k] += g[s];
        }
      }
#pragma unroll
      for (int s = 0; s < Q; ++s) {
        dgain[k] += st[s].y * p[s];
        sums[s] += gk[k] * p[s];
        sums[Q + s] += gk[k] * g[s];
      }
    }
    __syncwarp();
    cp_async_wait<1>();  // skip, which the sums' barrier shows to the other lanes
    at.sum(sums, sums_at + stage * At::kSums);
#pragma unroll
    for (int s = 0; s < Q; ++s) r[s] = st[s].y;
    if (full) {
      double r2[Q], r3[Q];
      Jet<DIM>::square(r, r2);
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
      const int c = at.lane + k * L;
      if (!at.has(k, channels)) continue;
      double d[Q], g[Q], y[Q];
#pragma unroll
      for (int s = 0; s < Q; ++s) {
        d[s] = xs[k * L + s * width] - st[s].x;
        g[s] = gk[k] * gs[k * L + s * width] - sums[Q + s];
      }
      if (full) {
        Jet<DIM>::corr(r, g, y);
        Jet<DIM>::corr_add(d, w, y);
      } else {
#pragma unroll
        for (int s = 0; s < Q; ++s) y[s] = r[s] * g[s] + d[s] * w[s];
      }
      if (skip) {
#pragma unroll
        for (int s = 0; s < Q; ++s) y[s] += es[k * L + s * width];
      }
      At::store(dx, y, row, n, c, channels);
    }
    __syncwarp();
  }
  cp_async_wait<0>();
  pdl_trigger();
  // the block's lanes that share a channel, in order
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = (threadIdx.x / L * K + k) * L + threadIdx.x % L;
    smem[i] = dgain[k];
    smem[K * At::kBlock + i] = dbias[k];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * K * L; i += At::kBlock) {
    const int which = i / (K * L), c = i % (K * L);
    double s = 0.0;
    for (int q = 0; q < At::kBlock / L; ++q) s += smem[which * K * At::kBlock + q * K * L + c];
    if (c < channels) (which ? bias_parts : gain_parts)[int64_t(blockIdx.x) * channels + c] = s;
  }
}

// dgain, dbias [channels] each from their [parts][channels]: 32 strands of parts a value, each in
// order, then the strands in order
constexpr int kFinishStrands = 32, kFinishLanes = 32;
__global__ void __launch_bounds__(kFinishStrands* kFinishLanes)
    norm_finish(const double* __restrict__ gain_parts, const double* __restrict__ bias_parts, int parts,
                double* __restrict__ dgain, double* __restrict__ dbias, int channels) {
  __shared__ double shared[kFinishStrands][kFinishLanes];
  const int lane = threadIdx.x % kFinishLanes, strand = threadIdx.x / kFinishLanes;
  const int64_t i = int64_t(blockIdx.x) * kFinishLanes + lane, c = i < channels ? i : i - channels;
  const bool live = i < 2 * int64_t(channels);
  const double* from = (i < channels ? gain_parts : bias_parts) + c;
  double s = 0.0;
  pdl_wait();
  if (live) {
#pragma unroll 8
    for (int k = strand; k < parts; k += kFinishStrands) s += from[int64_t(k) * channels];
  }
  shared[strand][lane] = s;
  __syncthreads();
  if (strand == 0 && live) {
    for (int k = 1; k < kFinishStrands; ++k) s += shared[k][lane];
    (i < channels ? dgain : dbias)[c] = s;
  }
}

template <int V>
using Int = std::integral_constant<int, V>;
template <typename A>
struct Type { using type = A; };
// How many lanes share a unit of `channels`: calls f(Type<Place<...>>) with the fewest whose K
// channels each cover them; false where none do.  Exact: they cover no more, and the tensors
// are aligned.
template <int DIM, bool BACKWARD, typename F>
bool with_lanes(int channels, bool aligned, const F& f) {
  constexpr int K = unit_k<DIM, BACKWARD>();
  const int lanes = (channels + K - 1) / K;
  const auto call = [&](auto t, auto w) {
    if (aligned && channels == K * t * w) f(Type<Place<DIM, BACKWARD, t, w, true>>{});
    else f(Type<Place<DIM, BACKWARD, t, w, false>>{});
    return true;
  };
  if (lanes <= 8) return call(Int<8>{}, Int<1>{});
  if (lanes <= 16) return call(Int<16>{}, Int<1>{});
  if (lanes <= 32) return call(Int<32>{}, Int<1>{});
  if (lanes <= 64) return call(Int<32>{}, Int<2>{});
  if (lanes <= 128) return call(Int<32>{}, Int<4>{});
  return lanes <= kUnitMostLanes && call(Int<32>{}, Int<8>{});
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// blocks of the adjoint, each of which keeps a [channels] of dgain and of dbias: one a multiprocessor
// where units are streamed, eight of the small ones elsewhere; at most one a unit
template <int DIM>
int64_t norm_parts(Packed rows, int channels, int sms) {
  const bool streamed = with_lanes<DIM, true>(channels, false, [](auto) {});
  return std::min(rows.units<Jet<DIM>::Q>(), int64_t(sms) * (streamed ? 1 : 8));
}
int64_t norm_parts(int dim, Packed rows, int channels, int sms) {
  return dim == 2 ? norm_parts<2>(rows, channels, sms) : norm_parts<3>(rows, channels, sms);
}

template <int DIM>
cudaError_t launch_norm(const double* x, const double* gain, const double* bias, double* out, double* stats, double eps,
                        Packed rows, int channels, int sms, cudaStream_t stream) {
  const int64_t units = rows.units<Jet<DIM>::Q>();
  cudaError_t e = cudaSuccess;
  const bool done = with_lanes<DIM, false>(channels, aligned16(x), [&](auto place) {
    using At = typename decltype(place)::type;
    const auto kernel = norm_forward_unit<At>;
    const int smem = int(sizeof(double)) * At::kGroups * At::kDoubles;
    // a per-device attribute: set on every call, so that each device gets it
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess)
      kernel<<<unsigned(std::min<int64_t>(units, sms)), At::kBlock, smem, stream>>>(x, gain, bias, out, stats, eps, rows,
                                                                                   channels, aligned16(x) && channels % 2 == 0);
  });
  if (!done)
    norm_forward<DIM><<<unsigned(std::min(units, int64_t(sms) * 8)), kNormThreads, 0, stream>>>(x, gain, bias, out, stats,
                                                                                              eps, rows, channels);
  return e != cudaSuccess ? e : cudaGetLastError();
}

template <int DIM>
cudaError_t launch_norm_vjp(const double* x, const double* gain, const double* stats, const double* seed,
                            const double* skip, double* dx, double* dgain, double* dbias, double* partials, Packed rows,
                            int channels, int sms, cudaStream_t stream) {
  const int parts = int(norm_parts<DIM>(rows, channels, sms));
  double *gain_parts = dgain, *bias_parts = dbias;  // a single block's sums are the gradients
  if (parts > 1) gain_parts = partials, bias_parts = partials + int64_t(parts) * channels;
  cudaError_t e = cudaSuccess;
  const bool aligned = aligned16(x) && aligned16(seed) && aligned16(skip);
  const bool done = with_lanes<DIM, true>(channels, aligned, [&](auto place) {
    using At = typename decltype(place)::type;
    const auto kernel = norm_backward_unit<At>;
    const int smem = int(sizeof(double)) * At::kGroups * At::kDoubles;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess)
      kernel<<<parts, At::kBlock, smem, stream>>>(x, gain, stats, seed, skip, dx, gain_parts, bias_parts, rows, channels,
                                                  aligned && channels % 2 == 0);
  });
  if (!done)
    norm_backward<DIM><<<parts, kNormThreads, 0, stream>>>(x, gain, stats, seed, skip, dx, gain_parts, bias_parts, rows,
                                                         channels);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess || parts == 1) return e;
  const unsigned blocks = unsigned((2 * int64_t(channels) + kFinishLanes - 1) / kFinishLanes);
  return launch_dependent(norm_finish, blocks, kFinishStrands * kFinishLanes, 0, stream, gain_parts, bias_parts, parts,
                          dgain, dbias, channels);
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
  if (outputs_overlap({{out, bytes}, {stats, stat}}, {{value, bytes}, {gain, small}, {bias, small}}))
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
  *bytes = size_t(norm_parts(dim, Packed{full_points, value_points}, channels, sms)) * 2 * channels * sizeof(double);
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
  if (outputs_overlap({{d_value, bytes}, {d_gain, small}, {d_bias, small}, {scratch, scratch_bytes}},
                      {{value, bytes}, {gain, small}, {stats, stat}, {seed, bytes}, {skip, bytes}}))
    return int(cudaErrorInvalidValue);
  int sms = 0;
  cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return int(e);
  if (scratch_bytes < size_t(norm_parts(dim, rows, channels, sms)) * 2 * small) return int(cudaErrorInvalidValue);
  const auto launch = dim == 2 ? launch_norm_vjp<2> : launch_norm_vjp<3>;
  return int(launch(value, gain, stats, seed, skip, d_value, d_gain, d_bias, scratch, rows, channels, sms, stream));
}

}  // extern "C"
