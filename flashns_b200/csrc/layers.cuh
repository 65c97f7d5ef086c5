// What the layer operators (norm.cu, affine.cu) share: packed units, jet products by
// dimension, fixed-order sums over lanes, argument checks.
#pragma once
#include <cuda.h>

#include <climits>
#include <cstddef>
#include <cstdint>
#include <initializer_list>
#include <mutex>

#include "common.cuh"
#include "products_generated.cuh"

namespace flashns_b200 {

// A unit is Q consecutive packed rows: the jet of one full point, or up to Q value rows
// (each a point of its own).  Both load and store alike.
struct Packed {
  int64_t full, value;  // points
  template <int Q>
  __host__ __device__ int64_t units() const { return full + (value + Q - 1) / Q; }
  template <int Q>
  __host__ __device__ int64_t row(int64_t u) const { return u * Q; }  // full points' rows come first
  template <int Q>
  __host__ __device__ int count(int64_t u) const {  // live rows of unit u
    if (u < full) return Q;
    const int64_t left = value - (u - full) * Q;
    return int(left < Q ? left : Q);
  }
};

template <int DIM>
struct Jet {
  static constexpr int Q = Basis<DIM>::Q;
  static __device__ __forceinline__ void square(const double* d, double* v) {
    if constexpr (DIM == 2) jet_square_2d3(d, v); else jet_square_3d3(d, v);
  }
  static __device__ __forceinline__ void mul(const double* a, const double* b, double* out) {
    if constexpr (DIM == 2) jet_mul_2d3(a, b, out); else jet_mul_3d3(a, b, out);
  }
  static __device__ __forceinline__ void corr(const double* a, const double* s, double* out) {
    if constexpr (DIM == 2) jet_corr_2d3(a, s, out); else jet_corr_3d3(a, s, out);
  }
  static __device__ __forceinline__ void corr_add(const double* a, const double* s, double* out) {
    if constexpr (DIM == 2) jet_corr_add_2d3(a, s, out); else jet_corr_add_3d3(a, s, out);
  }
  static __device__ __forceinline__ void rsqrt(const double* v, double* r) {
    if constexpr (DIM == 2) jet_rsqrt_2d3(v, r); else jet_rsqrt_3d3(v, r);
  }
};

// Sums of N values over 2 * O lanes, left in every lane.  Each step halves the values a lane
// carries (it keeps one half and gives the other away), so N values over 32 lanes take about
// 2 N shuffles in place of 5 N; the way back hands the sums out.  Every lane gets the same
// bits, in an order fixed by the lane numbers.
template <int N, int O>
__device__ __forceinline__ void lane_sums(double* v) {
  if constexpr (O == 0) {
    return;
  } else if constexpr (N == 1) {
    v[0] += __shfl_xor_sync(0xffffffffu, v[0], O);
    lane_sums<1, O / 2>(v);
  } else {
    constexpr int H = (N + 1) / 2;
    const bool up = (threadIdx.x & O) != 0;
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const double lo = v[i], hi = i + H < N ? v[i + H] : 0.0;
      v[i] = (up ? hi : lo) + __shfl_xor_sync(0xffffffffu, up ? lo : hi, O);
    }
    lane_sums<H, O / 2>(v);
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const double other = __shfl_xor_sync(0xffffffffu, v[i], O), mine = v[i];
      v[i] = up ? other : mine;
      if (i + H < N) v[i + H] = up ? mine : other;
    }
  }
}

// The first half of lane_sums: every lane ends with its own few of the N sums, v[0 ..] being
// the sums first, first + 1, ... below limit (call with first = 0, limit = N).
template <int N, int O>
__device__ __forceinline__ void lane_shares(double* v, int& first, int& limit) {
  if constexpr (O > 0) {
    constexpr int H = (N + 1) / 2;
    const bool up = (threadIdx.x & O) != 0;
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const double lo = v[i], hi = i + H < N ? v[i + H] : 0.0;
      v[i] = (up ? hi : lo) + __shfl_xor_sync(0xffffffffu, up ? lo : hi, O);
    }
    if (up) first += H;
    else limit = limit < first + H ? limit : first + H;
    lane_shares<H, O / 2>(v, first, limit);
  }
}

inline bool layer_sizes_ok(int dim, int64_t full, int64_t value, int widest) {
  if ((dim != 2 && dim != 3) || full < 0 || value < 0 || widest < 1) return false;
  const int64_t q = dim == 2 ? 10 : 20;
  // rows <= full * q + value, padded by one unit; offsets in bytes stay in 64 bits
  if (full > (INT64_MAX - value - q) / q) return false;
  return full * q + value + q <= INT64_MAX / int64_t(sizeof(double)) / widest / 2;
}

inline bool ranges_overlap(const void* a, size_t na, const void* b, size_t nb) {
  const auto pa = reinterpret_cast<uintptr_t>(a), pb = reinterpret_cast<uintptr_t>(b);
  return a && b && na && nb && (pa <= pb ? pb - pa < na : pa - pb < nb);
}

struct Span {
  const void* at;  // null: no such tensor
  size_t bytes;
};
// whether an output (or the scratch) lies over an input or another output
inline bool outputs_overlap(std::initializer_list<Span> outputs, std::initializer_list<Span> inputs) {
  for (const Span* o = outputs.begin(); o != outputs.end(); ++o) {
    for (const Span& i : inputs)
      if (ranges_overlap(o->at, o->bytes, i.at, i.bytes)) return true;
    for (const Span* other = outputs.begin(); other != o; ++other)
      if (ranges_overlap(o->at, o->bytes, other->at, other->bytes)) return true;
  }
  return false;
}

inline cudaError_t sm_count(int* sms) {
  int device = 0;
  const cudaError_t e = cudaGetDevice(&device);
  return e != cudaSuccess ? e : cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device);
}

// Tensor map of [rows][cols] row-major FP64 read or written in boxes of box_rows x box_cols;
// what a box holds past the matrix reads as zeros and is not written.  base and the rows on
// 16-byte boundaries.  swizzle: 16-byte piece c of a box's 128-byte row r lies at c ^ (r & 7).
inline cudaError_t matrix_map(CUtensorMap* map, const double* base, int64_t rows, int cols, int box_cols, int box_rows,
                              bool swizzle = false) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode encode = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {  // through the runtime, without a link against the driver library
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      encode = reinterpret_cast<Encode>(p);
  });
  if (!encode) return cudaErrorNotSupported;
  const cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)}, pitch[1] = {cuuint64_t(cols) * sizeof(double)};
  const cuuint32_t box[2] = {cuuint32_t(box_cols), cuuint32_t(box_rows)}, step[2] = {1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT64, 2, const_cast<double*>(base), dims, pitch, box, step,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// Launch that may start while the stream's previous kernel drains; the kernel waits
// (pdl_wait) before it reads what that one wrote.
template <typename... P, typename... A>
cudaError_t launch_dependent(void (*kernel)(P...), unsigned grid, unsigned threads, size_t smem, cudaStream_t stream,
                             A... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(grid);
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, static_cast<P>(args)...);
}

}  // namespace flashns_b200
