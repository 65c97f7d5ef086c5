// Hidden affine layer on packed jets with the tanh jet and a residual in its epilogue, and
// its adjoint.
//
//   Z = H W^T, + b on order-0 rows;  A = tanh jet(Z), a1 = sech^2 Z_0;  Y = A (+ R)
// (without the activation Y = Z (+ R)).  Adjoint at G, which is also R's gradient:
//   dZ = VJP of the tanh jet at (A, a1), G;  dH = dZ W;  dW = dZ^T H;  db = sum of order-0 dZ.
#include <algorithm>

#include "flashns_b200.h"
#include "jets_generated.cuh"
#include "layers.cuh"

namespace flashns_b200 {
// set by a kernel whose bounded wait on a copy gave up (read with eval.cu's word)
__device__ int g_affine_fault = 0;
cudaError_t affine_fault(int* fault, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(fault, g_affine_fault, sizeof(int));
  if (e == cudaSuccess && clear) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_affine_fault, &zero, sizeof(int));
  }
  return e;
}
namespace {

constexpr int kAffThreads = 256;

// Polls after which a wait on a copy gives up: on a tile, and on what a tile's outputs need
// besides.  Fewer than kMbarSpins only where a test makes the waits give up.
struct Polls {
  unsigned tile, late;
};
thread_local Polls t_polls{kMbarSpins, kMbarSpins};

// A wait that gives up sets the fault word and then, bounded too, lets the copy land: a late one
// would write into the place's next use, or into another block's memory.  False in the whole
// warp if any of its lanes gave up (call it with the whole warp).
__device__ __forceinline__ bool wait_copy(uint64_t* bar, unsigned phase, unsigned polls) {
  const bool ok = mbar_wait(bar, phase, polls);
  if (__all_sync(0xffffffffu, ok)) return true;
  if (!ok) atomicExch(&g_affine_fault, 1);
  mbar_wait(bar, phase);
  __syncwarp();
  return false;
}

template <int DIM>
__device__ __forceinline__ void tanh_forward(const double* z, double* h, double& a1) {
  if constexpr (DIM == 2) jet_fwd_2d3(z, h, a1); else jet_fwd_3d3(z, h, a1);
}
template <int DIM>
__device__ __forceinline__ void tanh_vjp(const double* h, double a1, const double* hb, double* zb) {
  if constexpr (DIM == 2) jet_vjp_2d3(h, a1, hb, zb); else jet_vjp_3d3(h, a1, hb, zb);
}

// ---------------------------------------------------------------- forward
// Z^T = W H^T on the FP64 tensor pipe (DMMA m16n8k8): MMA M = output channels, N = packed
// rows, K = input channels.  A warp owns 16 channels of 4 units; column 2t + e of its n8 tile
// j is row 2j + e of unit t, so a thread's accumulators hold all Q rows of one unit for two
// channels and the tanh jet, bias and residual run from registers.  Row g of the M tile is
// channel 2g (g < 8) or 2(g - 8) + 1, which makes a thread's two channels neighbours: the
// residual and the outputs move as 16-byte pairs.
//
// This form is for layers whose whole tiles do not fit (below), odd input widths, unaligned
// tensors, and value rows alone.  A CTA keeps a block of 64 output channels' W in shared memory
// (wider inputs than 256 stream it) and runs NG groups of GW warps that share it: each streams
// its own tiles (GW units x 32 input channels a stage, NS stages of cp.async).  Left to
// themselves the groups fall into step, sharing the one FP64 datapath evenly, and then wait for
// memory together, so they take turns on it (Turns: 64 -> 64 with tanh and residual at 16,384 +
// 4,096 points takes 89 us in a ring of four, 95 with two turns at a time).  Rows are padded to
// 36 doubles, W's to 2 (mod 8), and a 3-D unit by 8 more: every fragment load is free of bank
// conflicts.
constexpr int kFwKC = 32, kFwLD = kFwKC + 4, kFwCB = 64;

template <int DIM>
constexpr int fw_unit_stride() { return Jet<DIM>::Q * kFwLD + (DIM == 3 ? 8 : 0); }
template <int DIM, int NG, int GW, int NS, bool STREAM>
size_t fw_smem(int cin) {
  const size_t ld = STREAM ? kFwKC + 2 : (size_t(cin) + kFwKC - 1) / kFwKC * kFwKC + 2;
  return sizeof(double) * (size_t(NG) * NS * GW * fw_unit_stride<DIM>() + kFwCB * ld * (STREAM ? NG * NS : 1));
}

// hides a loop-invariant stride, so that its multiples are formed where they are used and not
// kept in registers through the MMAs
__device__ __forceinline__ int64_t opaque(int64_t v) {
  asm volatile("mov.b64 %0, %0;" : "+l"(v));
  return v;
}
__device__ __forceinline__ void prefetch_line(const void* gmem) { asm volatile("prefetch.global.L2 [%0];\n" ::"l"(gmem)); }
__device__ __forceinline__ void cp_async8(void* smem, const void* gmem, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;\n" ::"r"(smem_u32(smem)), "l"(gmem), "r"(valid ? 8 : 0));
}

// Weights of output channels c0 .. c0 + 63 and input channels k0 .. k0 + width - 1 into dst
// [64][ld], zero past the ends: w is [cout][cin], or with `across` [cin][cout] (the adjoint's
// product with W instead of its transpose).
__device__ __forceinline__ void load_weight(double* dst, int ld, const double* __restrict__ w, int c0, int k0, int width,
                                            int cin, int cout, bool vec, bool across, int tid, int threads) {
  if (across) {
    for (int e = tid; e < kFwCB * width; e += threads) {
      const int r = e % kFwCB, k = k0 + e / kFwCB;
      const bool ok = c0 + r < cout && k < cin;
      cp_async8(dst + r * ld + k - k0, ok ? w + int64_t(k) * cout + c0 + r : w, ok);
    }
  } else if (vec) {
    const int half = width / 2;
    for (int e = tid; e < kFwCB * half; e += threads) {
      const int r = e / half, k = k0 + 2 * (e % half);
      const bool ok = c0 + r < cout && k < cin;
      cp_async16(dst + r * ld + k - k0, ok ? w + int64_t(c0 + r) * cin + k : w, ok);
    }
  } else {
    for (int e = tid; e < kFwCB * width; e += threads) {
      const int r = e / width, k = k0 + e % width;
      const bool ok = c0 + r < cout && k < cin;
      cp_async8(dst + r * ld + k - k0, ok ? w + int64_t(c0 + r) * cin + k : w, ok);
    }
  }
}

// Bias and tanh jet of unit u, channels c and c + 1: the accumulators' rows into h0, h1; a1 is
// stored here.
template <int DIM, bool ACT>
__device__ __forceinline__ void forward_jets(const double (&acc)[Jet<DIM>::Q / 2][4], double b0, double b1, int64_t u,
                                             int c, const Packed& rows, int cout, double* __restrict__ aux, bool two,
                                             double (&h0)[Jet<DIM>::Q], double (&h1)[Jet<DIM>::Q]) {
  constexpr int Q = Jet<DIM>::Q;
  const bool full = u < rows.full;
#pragma unroll
  for (int s = 0; s < Q; ++s) {
    h0[s] = acc[s >> 1][s & 1] + (s == 0 || !full ? b0 : 0.0);
    h1[s] = acc[s >> 1][2 + (s & 1)] + (s == 0 || !full ? b1 : 0.0);
  }
  if constexpr (ACT) {
    double a0, a1;
    if (full) {
      tanh_forward<DIM>(h0, h0, a0);
      tanh_forward<DIM>(h1, h1, a1);
      if (aux) {
        aux[u * cout + c] = a0;
        if (two) aux[u * cout + c + 1] = a1;
      }
    } else {
      const int n = rows.count<Q>(u);
      double* ax = aux ? aux + (rows.full + (u - rows.full) * Q) * cout + c : nullptr;
#pragma unroll
      for (int s = 0; s < Q; ++s) {
        jet_fwd_2d0(h0 + s, h0 + s, a0);
        jet_fwd_2d0(h1 + s, h1 + s, a1);
        if (ax && s < n) {
          ax[int64_t(s) * cout] = a0;
          if (two) ax[int64_t(s) * cout + 1] = a1;
        }
      }
    }
  }
}

// h0, h1 of unit u to `activated`, and with the residual to `out`
template <int DIM>
__device__ __forceinline__ void forward_store(double (&h0)[Jet<DIM>::Q], double (&h1)[Jet<DIM>::Q], int64_t u, int c,
                                              const Packed& rows, int cout, const double* __restrict__ residual,
                                              double* __restrict__ out, double* __restrict__ activated, bool vec, bool two) {
  constexpr int Q = Jet<DIM>::Q;
  const int n = rows.count<Q>(u);
  const int64_t at = rows.row<Q>(u) * cout + c;
  const bool whole = vec && n == Q;
  if (whole) {
    const int64_t step = opaque(cout);
    if (activated) {
      double* to = activated + at;
#pragma unroll
      for (int s = 0; s < Q; ++s, to += step) *reinterpret_cast<double2*>(to) = make_double2(h0[s], h1[s]);
    }
    if (residual) {
      const double* from = residual + at;
#pragma unroll
      for (int half = 0; half < Q; half += 10) {  // ten rows requested at once
        double2 r[10];
#pragma unroll
        for (int s = 0; s < 10; ++s, from += step) r[s] = *reinterpret_cast<const double2*>(from);
#pragma unroll
        for (int s = 0; s < 10; ++s) h0[half + s] += r[s].x, h1[half + s] += r[s].y;
      }
    }
    double* to = out + at;
#pragma unroll
    for (int s = 0; s < Q; ++s, to += step) *reinterpret_cast<double2*>(to) = make_double2(h0[s], h1[s]);
    return;
  }
#pragma unroll
  for (int s = 0; s < Q; ++s) {
    if (s >= n) continue;
    const int64_t i = at + int64_t(s) * cout;
    if (activated) activated[i] = h0[s];
    out[i] = residual ? h0[s] + residual[i] : h0[s];
    if (two) {
      if (activated) activated[i + 1] = h1[s];
      out[i + 1] = residual ? h1[s] + residual[i + 1] : h1[s];
    }
  }
}

// eight input channels of a tile: A rows ap and ap + ldw, B columns of n8 tile j at row 2 j
template <int NT>
__device__ __forceinline__ void forward_step(double (&acc)[NT][4], const double* ap, int ldw, const double* bp,
                                             int ld = kFwLD) {
  const double a[4] = {ap[0], ap[ldw], ap[4], ap[ldw + 4]};
#pragma unroll
  for (int j = 0; j < NT; ++j) mma_m16n8k8(acc[j], a, bp[2 * j * ld], bp[2 * j * ld + 4]);
}

// The groups' turns on the tensor pipe: group g runs a tile's MMAs between take and pass, after
// group g - 1 (group 0 after the last).  Turn barrier g counts group g syncing and its
// predecessor arriving; the last group opens the ring with one arrival, and a group whose
// predecessor arrived once more than it synced closes with one more sync (tiles are dealt in
// turn, so the groups' counts differ by at most one).
template <int NG, int THREADS, bool TURNS = true>
struct Turns {
  int g;
  __device__ explicit Turns(int group) : g(group) {
    if (TURNS && g == NG - 1) named_arrive(1 + NG, 2 * THREADS);
  }
  __device__ void take() const { named_sync(1 + NG + g, 2 * THREADS); }
  __device__ void pass() const { named_arrive(1 + NG + (g + 1) % NG, 2 * THREADS); }
  // tiles of this group and of its predecessor
  __device__ void close(int64_t mine, int64_t before) const {
    if (before + (g == 0) > mine) named_sync(1 + NG + g, 2 * THREADS);
  }
};

// Ten value rows from `row` on, channels c and c + 1, where there are no full points: two rows a
// round, the accumulators moving up, so that the loop holds four tanhs and not twenty (the
// unrolled form waits for instructions).
template <bool ACT>
__device__ __forceinline__ void forward_values(double (&acc)[5][4], double b0, double b1, int64_t row, int64_t total, int c,
                                               int cout, const double* __restrict__ residual, double* __restrict__ out,
                                               double* __restrict__ activated, double* __restrict__ aux, bool vec) {
  const bool two = c + 1 < cout;
  int64_t at = row * cout + c;
#pragma unroll 1
  for (int j = 0; j < 5; ++j, row += 2, at += 2 * int64_t(cout)) {
    double h[4] = {acc[0][0] + b0, acc[0][2] + b1, acc[0][1] + b0, acc[0][3] + b1}, a[4];  // (row, channel)
#pragma unroll
    for (int i = 0; i + 1 < 5; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = acc[i + 1][e];
    double2 r[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      r[e] = make_double2(0.0, 0.0);
      if (residual && row + e < total) {
        const double* from = residual + at + e * int64_t(cout);
        if (vec) r[e] = *reinterpret_cast<const double2*>(from);
        else r[e] = make_double2(from[0], two ? from[1] : 0.0);
      }
    }
    if constexpr (ACT) {
#pragma unroll
      for (int i = 0; i < 4; ++i) jet_fwd_2d0(h + i, h + i, a[i]);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (row + e >= total) break;
      const int64_t i = at + e * int64_t(cout);
      const double y0 = residual ? h[2 * e] + r[e].x : h[2 * e], y1 = residual ? h[2 * e + 1] + r[e].y : h[2 * e + 1];
      if (vec) {
        if (activated) *reinterpret_cast<double2*>(activated + i) = make_double2(h[2 * e], h[2 * e + 1]);
        if (ACT && aux) *reinterpret_cast<double2*>(aux + i) = make_double2(a[2 * e], a[2 * e + 1]);
        *reinterpret_cast<double2*>(out + i) = make_double2(y0, y1);
      } else {
        if (activated) activated[i] = h[2 * e];
        if (ACT && aux) aux[i] = a[2 * e];
        out[i] = y0;
        if (two) {
          if (activated) activated[i + 1] = h[2 * e + 1];
          if (ACT && aux) aux[i + 1] = a[2 * e + 1];
          out[i + 1] = y1;
        }
      }
    }
  }
}

template <int DIM, bool ACT, int NG, int GW, int NS, bool STREAM, bool VALUES, bool TURNS>
__global__ void __launch_bounds__(NG* GW * 32, 1)
    affine_forward(const double* __restrict__ hidden, const double* __restrict__ weight, const double* __restrict__ bias,
                   const double* __restrict__ residual, double* __restrict__ out, double* __restrict__ activated,
                   double* __restrict__ aux, Packed rows, int cin, int cout, bool vec_in, bool vec_out, bool across) {
  constexpr int Q = Jet<DIM>::Q, NT = Q / 2, US = fw_unit_stride<DIM>(), KC = kFwKC;
  constexpr int GT = 32 * GW, UT = GW, RT = UT * Q;  // a group's threads; units and rows of its tile
  extern __shared__ __align__(128) double smem[];
  const int tid = threadIdx.x, group = tid / GT, gt = tid % GT, wc = (gt >> 5) & 3, wr = gt >> 7;
  const int lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int blocks = (cout + kFwCB - 1) / kFwCB, cb = blockIdx.x % blocks, c0 = cb * kFwCB;
  const int64_t per = gridDim.x / blocks, units = rows.units<Q>(), total = rows.full * Q + rows.value;
  const int64_t tiles = (units + UT - 1) / UT, first = blockIdx.x / blocks + group * per;
  const auto count = [&](int64_t from) { return from < tiles ? (tiles - 1 - from) / (per * NG) + 1 : 0; };
  const int64_t mine = count(first);
  const int nk = (cin + KC - 1) / KC, ldw = STREAM ? KC + 2 : nk * KC + 2;
  double* ring = smem + group * NS * UT * US;
  double* sw = smem + NG * NS * UT * US + (STREAM ? group * NS * kFwCB * ldw : 0);
  const int64_t tile_step = per * NG;
  auto load_chunk = [&](int64_t r0, int k0, int stage) {
    double* dst = ring + stage * UT * US;
    if (vec_in) {  // 16 lanes a row, rows sub, sub + 2, ... of each unit
      const int unit = (gt >> 4) % UT, sub = (gt >> 4) / UT, k = 2 * (gt & 15);
      const int64_t r = r0 + unit * Q + sub, step = opaque(2 * int64_t(cin));
      const double* src = hidden + r * cin + k0 + k;
      double* to = dst + unit * US + sub * kFwLD + k;
      if (r0 + RT <= total && k0 + k < cin) {  // cin even: covers k + 1
#pragma unroll
        for (int i = 0; i < Q / 2; ++i, src += step) cp_async16(to + 2 * i * kFwLD, src, true);
      } else {
        for (int i = 0; i < Q / 2; ++i, src += step) {
          const bool ok = r + 2 * i < total && k0 + k < cin;
          cp_async16(to + 2 * i * kFwLD, ok ? src : hidden, ok);
        }
      }
    } else {
      for (int e = gt; e < RT * KC; e += GT) {
        const int r = e / KC, k = e % KC;
        const bool ok = r0 + r < total && k0 + k < cin;
        cp_async8(dst + r / Q * US + r % Q * kFwLD + k, ok ? hidden + (r0 + r) * cin + k0 + k : hidden, ok);
      }
    }
    if constexpr (STREAM)
      load_weight(sw + stage * kFwCB * ldw, ldw, weight, c0, k0, KC, cin, cout, vec_in, across, gt, GT);
  };
  // the next chunk to load: its tile, K chunk and stage
  int64_t load_tile = first;
  int load_kc = 0, load_stage = 0;

  auto load = [&] {
    if (load_tile < tiles) load_chunk(load_tile * RT, load_kc * KC, load_stage);
    cp_async_commit();
    load_stage = load_stage + 1 == NS ? 0 : load_stage + 1;
    if (++load_kc == nk) load_kc = 0, load_tile += tile_step;
  };

  if constexpr (!STREAM) load_weight(sw, ldw, weight, c0, 0, nk * KC, cin, cout, vec_in, across, tid, NG * GT);
  cp_async_commit();
#pragma unroll
  for (int s = 0; s < NS - 1; ++s) load();
  cp_async_wait<NS - 1>();
  __syncthreads();  // W is there for every group

  const int ch = wc * 16 + 2 * g, c = c0 + ch;  // this thread's channels c, c + 1
  const double b0 = bias && c < cout ? bias[c] : 0.0, b1 = bias && c + 1 < cout ? bias[c + 1] : 0.0;
  double acc[NT][4];
  const Turns<NG, GT, TURNS> turns(group);
  int stage = 0;
  for (int64_t tile = first; tile < tiles; tile += tile_step) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0.0;
    if (residual) {  // the tile's residual towards L2, for the epilogue
      const int width = cout - c0 < kFwCB ? cout - c0 : kFwCB;
      for (int e = gt; e < RT * (kFwCB / 16); e += GT) {
        const int64_t r = tile * RT + e / (kFwCB / 16);
        const int k = e % (kFwCB / 16) * 16;
        if (r < total && k < width) prefetch_line(residual + r * cout + c0 + k);
      }
    }
    for (int kc = 0; kc < nk; ++kc) {
      cp_async_wait<NS - 2>();
      named_sync(1 + group, GT);  // the chunk is there, the stage loaded next is read out
      load();
      if (TURNS && kc == 0) turns.take();
      const double* bp = ring + stage * UT * US + (wr * 4 + (g >> 1)) * US + (g & 1) * kFwLD + t;
      const double* ap = sw + (STREAM ? stage * kFwCB * ldw : kc * KC) + ch * ldw + t;
      const int left = cin - kc * KC;
      if (left >= KC) {
#pragma unroll
        for (int k = 0; k < KC / 8; ++k) forward_step<NT>(acc, ap + 8 * k, ldw, bp + 8 * k);
      } else {
#pragma unroll 1
        for (int k = 0; k < (left + 7) / 8; ++k) forward_step<NT>(acc, ap + 8 * k, ldw, bp + 8 * k);
      }
      stage = stage + 1 == NS ? 0 : stage + 1;
    }
    if (TURNS) turns.pass();
    const int64_t u = tile * UT + wr * 4 + t;
    if constexpr (VALUES) {
      if (u * Q < total && c < cout)
        forward_values<ACT>(acc, b0, b1, u * Q, total, c, cout, residual, out, activated, aux, vec_out);
    } else {
      const bool live = u < units && c < cout;
      double h0[Q], h1[Q];
      if (live) {
        forward_jets<DIM, ACT>(acc, b0, b1, u, c, rows, cout, aux, c + 1 < cout, h0, h1);
        forward_store<DIM>(h0, h1, u, c, rows, cout, residual, out, activated, vec_out, c + 1 < cout);
      }
    }
    __syncwarp();
  }
  if (TURNS) turns.close(mine, count(blockIdx.x / blocks + (group + NG - 1) % NG * per));
  cp_async_wait<0>();
}

// ---------------------------------------------------------------- forward, resident tiles
// The same product where W's block and two whole tiles fit in shared memory (cin <= 112 for up
// to 64 outputs, 128 for more): two groups of 8 warps, WC of them across channels (16 each) and 8 / WC across rows (40 each, as
// four blocks of 10; a 3-D unit is two blocks).  A group waits for its whole tile before it
// takes its turn, runs MMAs and tanh jets in one stretch, hands the turn on, and only then
// loads its next tile and stores: between take and pass there is no barrier and no memory
// access, and the partner's turn covers the group's.  The jets stay inside the turn because
// DMMA and DFMA share one datapath with DMMA first: outside it they crawl behind the partner's
// MMAs (16,384 + 4,096 points, 64 -> 64 with residual: 110 us against 88, both with outputs
// stored by threads; 76 with the boxes below).  A tile is one TMA box of 36 columns for each 32
// (the 4 more are the padding that frees the fragment loads of bank conflicts).  At that size a
// turn is 6,500 cycles of MMAs (5,120 at the full rate) and 1,250 of jets.
constexpr int kTileGroup = 256, kTileSmem = 227 * 1024;
constexpr int tile_rows(int wc) { return 320 / wc; }
__host__ __device__ constexpr int tile_planes(int cin) { return (cin + kFwKC - 1) / kFwKC; }
__host__ __device__ constexpr int tile_ldw(int cin) { return (cin + 7) / 8 * 8 + 2; }  // 2 (mod 8)
// a tile's rows: whole planes of 32 channels, then the rest, to 8, with its own padding (12, 20,
// 28 or 36 doubles are all 4 or 12 (mod 16))
__host__ __device__ constexpr int tail_ld(int cin) { return cin % kFwKC ? (cin % kFwKC + 7) / 8 * 8 + 4 : 0; }
__host__ __device__ constexpr int tile_width(int cin) { return cin / kFwKC * kFwLD + tail_ld(cin); }
constexpr size_t tile_smem(int wc, int cin) {
  return sizeof(double) * (2 * size_t(tile_rows(wc)) * tile_width(cin) + size_t(16 * wc) * tile_ldw(cin) + 18);  // 18 barriers
}

// rows r0 .. r0 + count - 1 (zeros from `total` on) and columns 0 .. cin8 - 1 (zeros past cin)
// of src into dst [count][ld]: one row a warp
__device__ __forceinline__ void load_rows(double* dst, int ld, const double* __restrict__ src, int64_t r0, int count,
                                          int64_t total, int cin, bool vec, int warp, int warps, int lane) {
  const int cin8 = (cin + 7) / 8 * 8;
  for (int r = warp; r < count; r += warps) {
    const bool live = r0 + r < total;
    const double* row = live ? src + (r0 + r) * cin : src;
    if (vec) {
      for (int k = 2 * lane; k < cin8; k += 64) cp_async16(dst + r * ld + k, k < cin ? row + k : src, live && k < cin);
    } else {
      for (int k = lane; k < cin8; k += 32) cp_async8(dst + r * ld + k, k < cin ? row + k : src, live && k < cin);
    }
  }
}

struct TileMaps {
  CUtensorMap planes, tail, out, activated, residual;
};

// How a tile's outputs leave and its residual comes.  A warp's 40 rows x 16 channels go through
// a box in shared memory, in and out by TMA: the same bytes as loads and stores of the threads
// keep the load/store unit busy for 1,400 cycles a tile (5,000 with the residual and a second
// output), in which the partner's fragment loads, and with them its MMAs, hardly advance.  The
// boxes have room of their own, or lie in the tile that has been read, whose successor (and the
// residual) then arrives a little later.  Where neither has the room for a group's eight boxes,
// threads load and store: with more than 64 outputs, layers of 82 to 112 inputs (dH: of 74 to
// 96 outputs); in 3-D with a residual, which never takes the tile's place, layers from 74 inputs on
// (82 with more than 64 outputs).
enum Leave { kByThreads, kInTile, kOwnBoxes };
constexpr int kBoxDoubles = 40 * 16, kBoxesBytes = 8 * kBoxDoubles * 8;  // a warp's; a group's

// pairs (h0, h1) of rows row + s, channels 2 g, 2 g + 1, into a warp's box, or onto what is there
template <int Q>
__device__ __forceinline__ void box_pairs(double* box, const double (&h0)[Q], const double (&h1)[Q], int row, int g,
                                          bool onto) {
  const auto at = [&](int r) { return reinterpret_cast<double2*>(box + r * 16 + ((g ^ (r & 7)) << 1)); };
  if (onto) {
#pragma unroll
    for (int half = 0; half < Q; half += 5) {  // loads first: the stores could not pass them
      double2 v[5];
#pragma unroll
      for (int s = 0; s < 5; ++s) v[s] = *at(row + half + s);
#pragma unroll
      for (int s = 0; s < 5; ++s) *at(row + half + s) = make_double2(h0[half + s] + v[s].x, h1[half + s] + v[s].y);
    }
  } else {
#pragma unroll
    for (int s = 0; s < Q; ++s) *at(row + s) = make_double2(h0[s], h1[s]);
  }
}
// one channel's rows
template <int Q>
__device__ __forceinline__ void box_single(double* box, const double (&z)[Q], int row, int channel, bool onto) {
  const auto at = [&](int r) -> double& { return box[r * 16 + (((channel >> 1) ^ (r & 7)) << 1) + (channel & 1)]; };
  if (onto) {
#pragma unroll
    for (int half = 0; half < Q; half += 10) {  // loads first: the stores could not pass them
      double v[10];
#pragma unroll
      for (int s = 0; s < 10; ++s) v[s] = at(row + half + s);
#pragma unroll
      for (int s = 0; s < 10; ++s) at(row + half + s) = z[half + s] + v[s];
    }
  } else {
#pragma unroll
    for (int s = 0; s < Q; ++s) at(row + s) = z[s];
  }
}
// a warp's box from columns x .., rows y ..
__device__ __forceinline__ void fetch_box(const CUtensorMap* map, double* box, int x, int y, uint64_t* bar, int lane) {
  if (lane == 0) {
    fence_proxy_async();
    mbar_arrive_expect_tx(bar, kBoxDoubles * sizeof(double));
    tma_load_2d(box, map, x, y, bar);
  }
}
// a warp's box to columns x .., rows y ..; back when the box may be written again
__device__ __forceinline__ void send_box(const CUtensorMap* map, const double* box, int x, int y, int lane) {
  fence_proxy_async();
  __syncwarp();
  if (lane == 0) {
    tma_store_2d(map, x, y, box);
    bulk_commit();
    bulk_wait_read();
  }
  __syncwarp();
}

// A 3-D unit's two blocks lie with neighbouring threads, each with ten rows of two channels;
// they trade, and each goes on with one channel's twenty rows.
__device__ __forceinline__ void trade_blocks(const double (&acc)[5][4], int t, double (&z)[20]) {
#pragma unroll
  for (int s = 0; s < 10; ++s) {
    const double first = acc[s >> 1][s & 1], second = acc[s >> 1][2 + (s & 1)];
    const double got = __shfl_xor_sync(0xffffffffu, t & 1 ? first : second, 1);
    z[s] = t & 1 ? got : first;
    z[10 + s] = t & 1 ? second : got;
  }
}

template <int DIM, bool ACT, int WC>
__global__ void __launch_bounds__(2 * kTileGroup, 1)
    affine_forward_tile(const __grid_constant__ TileMaps maps, const double* __restrict__ weight,
                        const double* __restrict__ bias, const double* __restrict__ residual, double* __restrict__ out,
                        double* __restrict__ activated, double* __restrict__ aux, Packed rows, int cin, int cout,
                        bool vec_w, bool vec_out, Leave leave, Polls polls) {
  constexpr int Q = Jet<DIM>::Q, NT = 5, RT = tile_rows(WC), CB = 16 * WC, LD = kFwLD, PLANE = RT * LD;
  extern __shared__ __align__(128) double smem[];
  const int tid = threadIdx.x, group = tid / kTileGroup, gt = tid % kTileGroup, warp = gt >> 5, wc = warp % WC, wr = warp / WC;
  const int lane = tid & 31, g = lane >> 2, t = lane & 3;
  if (smem_u32(smem) & 127) {  // TMA destinations need it: refuse, never fault
    if (tid == 0) atomicExch(&g_affine_fault, 2);
    return;
  }
  const int blocks = (cout + CB - 1) / CB, c0 = blockIdx.x % blocks * CB;
  const int64_t per = gridDim.x / blocks, total = rows.full * Q + rows.value;
  const int64_t tiles = (total + RT - 1) / RT, first = blockIdx.x / blocks + group * per;
  const auto count = [&](int64_t from) { return from < tiles ? (tiles - 1 - from) / (2 * per) + 1 : 0; };
  const int planes = cin / kFwKC, ldt = tail_ld(cin), ldw = tile_ldw(cin), size = RT * tile_width(cin);
  double *tile_at = smem + group * size, *sw = smem + 2 * size;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sw + CB * ldw);
  uint64_t* bar_box = bars + 2 + (tid >> 5);
  double* box = leave == kOwnBoxes ? sw + CB * ldw + 18 : tile_at;
  box += (1024 - (smem_u32(box) & 1023)) % 1024 / 8;
  box += ((leave == kOwnBoxes ? group * 8 : 0) + warp) * kBoxDoubles;
  auto load = [&](int64_t tile) {  // by one thread, once every warp has read the last tile
    fence_proxy_async();
    mbar_arrive_expect_tx(bars + group, unsigned(size * sizeof(double)));
    for (int k = 0; k < planes; ++k) tma_load_2d(tile_at + k * PLANE, &maps.planes, k * kFwKC, int(tile * RT), bars + group);
    if (ldt) tma_load_2d(tile_at + planes * PLANE, &maps.tail, planes * kFwKC, int(tile * RT), bars + group);
  };

  if (gt == 0) mbar_init(bars + group, 1);
  if (lane == 0) mbar_init(bar_box, 1);
  __syncthreads();
  if (gt == 0 && first < tiles) load(first);
  load_rows(sw, ldw, weight, c0, CB, cout, cin, vec_w, tid >> 5, 16, lane);
  cp_async_commit();
  cp_async_wait<0>();
  __syncthreads();

  const int ch = wc * 16 + 2 * g, c = c0 + ch;  // this thread's channels c, c + 1
  const double b0 = c < cout ? bias[c] : 0.0, b1 = c + 1 < cout ? bias[c + 1] : 0.0;
  const int brow = wr * 40 + (g >> 1) * 10 + (g & 1);
  const double *ap = sw + ch * ldw + t, *bp = tile_at + brow * LD + t;
  const Turns<2, kTileGroup> turns(group);
  unsigned phase = 0;
  // a copy's wait gave up: in this warp; in this group, which keeps the turns and does no more work
  bool late = false, dead = false;
  for (int64_t tile = first; tile < tiles; tile += 2 * per) {
    double acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0.0;
    const int x = c0 + wc * 16, y = int(tile * RT) + wr * 40;  // this warp's box
    const bool fetched = residual && leave == kOwnBoxes && x < cout && !late && !dead;
    if (fetched) fetch_box(&maps.residual, box, x, y, bar_box, lane);
    if (residual && leave != kOwnBoxes) {  // towards L2, for this tile's epilogue
      const int64_t r0 = tile * RT, left = total - r0;
      if (vec_out && blocks == 1) {
        if (gt == 0) prefetch_l2(residual + r0 * cout, unsigned((left < RT ? left : RT) * cout * sizeof(double)));
      } else {
        const int width = cout - c0 < CB ? cout - c0 : CB;
        for (int e = gt; e < RT * WC; e += kTileGroup)
          if (e / WC < left && e % WC * 16 < width) prefetch_line(residual + (r0 + e / WC) * cout + c0 + e % WC * 16);
      }
    }
    if (!dead) {
      const bool ok = wait_copy(bars + group, phase, polls.tile);
      dead = named_sync_or(1 + group, kTileGroup, late || !ok);
      if (dead && fetched) mbar_wait(bar_box, phase);  // no box is under way when the block ends
    }
    turns.take();
    if (!dead && c0 + wc * 16 < cout) {
      for (int p = 0; p < planes; ++p) {
#pragma unroll
        for (int k = 0; k < 4; ++k) forward_step<NT>(acc, ap + p * kFwKC + 8 * k, ldw, bp + p * PLANE + 8 * k);
      }
      const double* tail = tile_at + planes * PLANE + brow * ldt + t;
#pragma unroll 1
      for (int k = 0; k < ldt / 8; ++k) forward_step<NT>(acc, ap + planes * kFwKC + 8 * k, ldw, tail + 8 * k, ldt);
    }
    const bool more = tile + 2 * per < tiles && !dead;
    if constexpr (DIM == 2) {
      const int64_t u = tile * (RT / Q) + wr * 4 + t;
      const bool live = !dead && u * Q < total && c < cout;
      double h0[Q], h1[Q];
      if (live) forward_jets<DIM, ACT>(acc, b0, b1, u, c, rows, cout, aux, c + 1 < cout, h0, h1);
      __syncwarp();
      turns.pass();
      named_sync(1 + group, kTileGroup);  // every warp has read the tile
      if (gt == 0 && more && leave != kInTile) load(tile + 2 * per);
      if (leave == kByThreads) {
        if (live) forward_store<DIM>(h0, h1, u, c, rows, cout, residual, out, activated, vec_out, c + 1 < cout);
      } else {
        if (x < cout && !dead) {
          if (residual) {
            if (leave == kInTile) fetch_box(&maps.residual, box, x, y, bar_box, lane);
            late = !wait_copy(bar_box, phase, polls.late);
          }
          if (!late) {
            box_pairs(box, h0, h1, t * 10, g, residual != nullptr);
            send_box(&maps.out, box, x, y, lane);
          }
          if (!late && activated) {
            box_pairs(box, h0, h1, t * 10, g, false);
            send_box(&maps.activated, box, x, y, lane);
          }
        }
      }
    } else {
      const int64_t u = tile * (RT / Q) + wr * 2 + (t >> 1), row = u * Q;
      const int cc = c + (t & 1);
      const bool live = !dead && row < total && cc < cout, full = u < rows.full;
      const int n = live ? rows.count<Q>(u) : 0;
      double z[Q];
      trade_blocks(acc, t, z);
      if (live) {
        const double b = t & 1 ? b1 : b0;
#pragma unroll
        for (int s = 0; s < Q; ++s) z[s] += s == 0 || !full ? b : 0.0;
        if constexpr (ACT) {
          double a1;
          if (full) {
            tanh_forward<DIM>(z, z, a1);
            if (aux) aux[u * cout + cc] = a1;
          } else {
            double* ax = aux ? aux + (rows.full + (u - rows.full) * Q) * cout + cc : nullptr;
#pragma unroll
            for (int s = 0; s < Q; ++s) {
              jet_fwd_2d0(z + s, z + s, a1);
              if (ax && s < n) ax[int64_t(s) * cout] = a1;
            }
          }
        }
      }
      __syncwarp();
      turns.pass();
      named_sync(1 + group, kTileGroup);
      if (gt == 0 && more && leave != kInTile) load(tile + 2 * per);
      if (leave == kByThreads) {
        if (live) {
          const int64_t step = opaque(cout);
          double* to = out + row * cout + cc;
          if (activated) {
            double* also = activated + row * cout + cc;
#pragma unroll
            for (int s = 0; s < Q; ++s, also += step)
              if (s < n) *also = z[s];
          }
          if (residual) {
            const double* from = residual + row * cout + cc;
#pragma unroll
            for (int half = 0; half < Q; half += 10) {  // ten rows requested at once
              double r[10];
#pragma unroll
              for (int s = 0; s < 10; ++s, from += step) r[s] = half + s < n ? *from : 0.0;
#pragma unroll
              for (int s = 0; s < 10; ++s) z[half + s] += r[s];
            }
          }
#pragma unroll
          for (int s = 0; s < Q; ++s, to += step)
            if (s < n) *to = z[s];
        }
      } else if (x < cout && !dead) {
        const int r0 = (t >> 1) * 20, channel = 2 * g + (t & 1);
        if (residual) {
          if (leave == kInTile) fetch_box(&maps.residual, box, x, y, bar_box, lane);
          late = !wait_copy(bar_box, phase, polls.late);
        }
        if (!late) {
          box_single(box, z, r0, channel, residual != nullptr);
          send_box(&maps.out, box, x, y, lane);
        }
        if (!late && activated) {
          box_single(box, z, r0, channel, false);
          send_box(&maps.activated, box, x, y, lane);
        }
      }
    }
    phase ^= 1;
    __syncwarp();
    if (leave == kInTile) {
      dead = named_sync_or(1 + group, kTileGroup, late) || dead;  // every box has left the tile's place
      if (gt == 0 && more && !dead) load(tile + 2 * per);
    }
  }
  if (lane == 0) bulk_wait();
  turns.close(count(first), count(blockIdx.x / blocks + (1 - group) * per));
}

constexpr int64_t kMostWeights = int64_t(1) << 40;  // what scratch sizes multiply stays in 64 bits
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <int DIM, bool ACT, int NG, int GW, int NS, bool STREAM, bool VALUES = false, bool TURNS = true>
cudaError_t launch_forward(const double* hidden, const double* weight, const double* bias, const double* residual,
                           double* out, double* activated, double* aux, Packed rows, int cin, int cout,
                           bool across, cudaStream_t stream) {
  const auto kernel = affine_forward<DIM, ACT, NG, GW, NS, STREAM, VALUES, TURNS>;
  const size_t smem = fw_smem<DIM, NG, GW, NS, STREAM>(cin);
  int sms = 0;
  cudaError_t e = sm_count(&sms);
  // a per-device attribute: set on every call, so that each device gets it
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
  if (e != cudaSuccess) return e;
  const int64_t blocks = (int64_t(cout) + kFwCB - 1) / kFwCB;
  const int64_t tiles = (rows.units<Jet<DIM>::Q>() + GW - 1) / GW;
  const int64_t most = sms / blocks > 0 ? sms / blocks : 1, per = tiles < most ? tiles : most;
  const bool vec_in = cin % 2 == 0 && aligned16(hidden) && aligned16(weight);
  const bool vec_out = cout % 2 == 0 && aligned16(out) && aligned16(residual) && aligned16(activated) && aligned16(aux);
  kernel<<<unsigned(per * blocks), NG * GW * 32, smem, stream>>>(hidden, weight, bias, residual, out, activated, aux,
                                                                 rows, cin, cout, vec_in, vec_out, across);
  return cudaGetLastError();
}

template <int DIM, bool ACT, int WC>
cudaError_t launch_forward_tile(const double* hidden, const double* weight, const double* bias, const double* residual,
                                double* out, double* activated, double* aux, Packed rows, int cin, int cout,
                                bool, cudaStream_t stream) {
  const auto kernel = affine_forward_tile<DIM, ACT, WC>;
  size_t smem = tile_smem(WC, cin);
  const int64_t blocks = (int64_t(cout) + 16 * WC - 1) / (16 * WC), total = rows.full * Jet<DIM>::Q + rows.value;
  const int64_t tiles = (total + tile_rows(WC) - 1) / tile_rows(WC);
  int sms = 0;
  TileMaps maps{};
  cudaError_t e = sm_count(&sms);
  if (e == cudaSuccess && cin >= kFwKC) e = matrix_map(&maps.planes, hidden, total, cin, kFwLD, tile_rows(WC));
  if (e == cudaSuccess && cin % kFwKC) e = matrix_map(&maps.tail, hidden, total, cin, tail_ld(cin), tile_rows(WC));
  const bool vec_out = cout % 2 == 0 && aligned16(out) && aligned16(residual) && aligned16(activated) && aligned16(aux);
  const size_t boxes = smem + 2 * kBoxesBytes + 1024;
  // a 3-D tile's residual in the tile's place comes too late for its next tile (100 -> 60 at
  // 8,193 + 2,049 points: 112 us, by threads 105)
  const bool late = DIM == 3 && residual;
  const Leave leave = !vec_out                                                              ? kByThreads
                      : boxes <= kTileSmem                                                  ? kOwnBoxes
                      : !late && sizeof(double) * tile_rows(WC) * tile_width(cin) >= kBoxesBytes + 1024 ? kInTile
                                                                                            : kByThreads;
  if (leave == kOwnBoxes) smem = boxes;
  if (e == cudaSuccess && leave != kByThreads) e = matrix_map(&maps.out, out, total, cout, 16, 40, true);
  if (e == cudaSuccess && leave != kByThreads && activated) e = matrix_map(&maps.activated, activated, total, cout, 16, 40, true);
  if (e == cudaSuccess && leave != kByThreads && residual) e = matrix_map(&maps.residual, residual, total, cout, 16, 40, true);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
  if (e != cudaSuccess) return e;
  const int64_t most = sms / blocks > 0 ? sms / blocks : 1, per = tiles < most ? tiles : most;
  kernel<<<unsigned(per * blocks), 2 * kTileGroup, smem, stream>>>(maps, weight, bias, residual, out, activated, aux, rows,
                                                                  cin, cout, aligned16(weight), vec_out, leave, t_polls);
  return cudaGetLastError();
}

// W's block beside as many groups and stages as 227 KB hold
template <int DIM, bool ACT, typename... Args>
cudaError_t forward(int cin, int cout, bool values, bool boxes, Args... args) {
  // tanhs of value rows alone (a point a row: the dimension does not matter) go with the small
  // groups, without turns: 40,401 rows 64 -> 64 take 29 us, in whole tiles 35
  if constexpr (ACT) {
    if (values) {
      if (cin <= 160) return launch_forward<2, true, 4, 4, 3, false, true, false>(args...);
      if (cin <= 256) return launch_forward<2, true, 4, 4, 2, false, true, false>(args...);
      return launch_forward<2, true, 4, 4, 2, true, true, false>(args...);
    }
  }
  if (boxes && cout <= 64 && tile_smem(4, cin) <= kTileSmem) return launch_forward_tile<DIM, ACT, 4>(args...);
  if (boxes && cout > 64 && tile_smem(8, cin) <= kTileSmem) return launch_forward_tile<DIM, ACT, 8>(args...);
  if constexpr (DIM == 2) {
    if (cin <= 160) return launch_forward<2, ACT, 4, 4, 3, false>(args...);
    if (cin <= 256) return launch_forward<2, ACT, 4, 4, 2, false>(args...);
    return launch_forward<2, ACT, 4, 4, 2, true>(args...);
  } else {
    if (cin <= 160) return launch_forward<3, ACT, 3, 4, 2, false>(args...);
    if (cin <= 256) return launch_forward<3, ACT, 2, 4, 2, false>(args...);
    return launch_forward<3, ACT, 2, 4, 2, true>(args...);
  }
}

// ---------------------------------------------------------------- adjoint
// dZ, one thread per (unit, output channel): widths that the tiles below do not hold
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

// dZ = VJP(A, a1; G) and dH = dZ W in one pass; FUSED (both widths <= 64): dW += dZ^T H too.
//
// Two groups of 8 warps, tiles of 320 / WC rows and 16 WC input channels, W resident.  Inside
// its turn a group runs FP64 work alone: its tile's dZ, in G's place in shared memory (a thread
// takes a unit's whole jet of one output channel); dH^T = W^T dZ^T from there, with a thread's
// two input channels side by side (the pair of a row of W is one 16-byte load, and dH leaves as
// 16-byte pairs); then dW = dZ^T H, whose accumulators stay in registers over all of the CTA's
// tiles.  The partner's turn (12,000 cycles and more) covers what moves data: G and A in by
// TMA boxes (unfused, A and a1 go to registers), dH out.  H takes A's place once the VJP has
// read it, behind the MMAs of dH.  Outside the turn the VJP took 15,000 cycles behind the
// partner's MMAs; inside, a turn of the 2-D 64 -> 64 layer is 14,150 cycles, 11,700 without a
// VJP, 10,240 for the MMAs alone at the full rate (16,384 + 4,096 points: 117 us, against 144).
// Unfused, dZ also goes to global memory, for affine_wgrad_tile.
constexpr size_t back_smem(int wc, bool fused, int cin, int cout) {
  const int other = cin > cout ? cin : cout;  // H and A share their place
  return sizeof(double) * (2 * size_t(tile_rows(wc)) * kFwLD * (tile_planes(cout) + (fused ? tile_planes(other) : 0)) +
                           size_t((cout + 7) / 8 * 8) * (16 * wc + 4) + 4);
}

// The turn passes this many 8-row steps of dW (fused) or 8-channel steps of dH before a group's
// last MMAs: the partner's VJP begins behind them.
constexpr int kEarlyRows = 6, kEarlySteps = 6;

struct BackMaps {
  CUtensorMap seed, activated, hidden, dh;
};

template <int DIM, bool ACT, int WC, bool FUSED>
__global__ void __launch_bounds__(2 * kTileGroup, 1)
    affine_backward_tile(const __grid_constant__ BackMaps maps, const double* __restrict__ hidden,
                         const double* __restrict__ weight, const double* __restrict__ activated,
                         const double* __restrict__ aux, const double* __restrict__ seed, double* __restrict__ dz,
                         double* __restrict__ dh, double* __restrict__ dw_parts, double* __restrict__ db_parts, Packed rows,
                         int cin, int cout, bool boxes, bool vec_out, bool vec_w, Leave leave, Polls polls) {
  constexpr int Q = Jet<DIM>::Q, RT = tile_rows(WC), CB = 16 * WC, LD = kFwLD, PLANE = RT * LD, LDW = CB + 4;
  constexpr int NT = RT * WC / 64, UT = RT / Q, PAIRS = UT * CB / kTileGroup;  // n8 tiles a warp; jets a thread
  constexpr bool SWAP = FUSED && ACT;  // A first, then H in its place
  static_assert(NT == 5 && PAIRS * kTileGroup == UT * CB && RT % 8 == 0, "");
  extern __shared__ __align__(128) double smem[];
  const int tid = threadIdx.x, group = tid / kTileGroup, gt = tid % kTileGroup, warp = gt >> 5, wc = warp % WC, wr = warp / WC;
  const int lane = tid & 31, g = lane >> 2, t = lane & 3;
  if (smem_u32(smem) & 127) {
    if (tid == 0) atomicExch(&g_affine_fault, 2);
    return;
  }
  const int blocks = (cin + CB - 1) / CB, i0 = blockIdx.x % blocks * CB;
  const int64_t per = gridDim.x / blocks, total = rows.full * Q + rows.value, units = rows.units<Q>();
  const int64_t tiles = (total + RT - 1) / RT, first = blockIdx.x / blocks + group * per;
  const auto count = [&](int64_t from) { return from < tiles ? (tiles - 1 - from) / (2 * per) + 1 : 0; };
  const int pz = tile_planes(cout), ph = FUSED ? tile_planes(cin) : 0, c8 = (cout + 7) / 8 * 8;
  const int px = FUSED ? (pz > ph ? pz : ph) : 0;  // planes of the place that A and H share
  double *z_at = smem + group * (pz + px) * PLANE, *h_at = z_at + pz * PLANE, *sw = smem + 2 * (pz + px) * PLANE;
  uint64_t *bar = reinterpret_cast<uint64_t*>(sw + c8 * LDW) + 2 * group, *bar_h = bar + 1;
  double* box = leave == kOwnBoxes ? sw + c8 * LDW + 4 : z_at;  // this warp's 40 rows x 16 channels
  box += (1024 - (smem_u32(box) & 1023)) % 1024 / 8;
  box += ((leave == kOwnBoxes ? group * 8 : 0) + warp) * kBoxDoubles;

  // a tile's planes of a [total][width] matrix, by TMA (one thread, after bar's expect) or by all
  auto copy = [&](double* to, const CUtensorMap* map, const double* from, int64_t tile, int planes, int width, uint64_t* b) {
    if (boxes) {
      for (int p = 0; p < planes; ++p) tma_load_2d(to + p * PLANE, map, p * kFwKC, int(tile * RT), b);
    } else {
#pragma unroll 1
      for (int e = gt; e < RT * planes * kFwKC; e += kTileGroup) {
        const int r = e / (planes * kFwKC), k = e % (planes * kFwKC);
        const bool ok = tile * RT + r < total && k < width;
        cp_async8(to + k / kFwKC * PLANE + r * LD + k % kFwKC, ok ? from + (tile * RT + r) * width + k : from, ok);
      }
    }
  };
  // This thread's jets: channel cz of the tile's units ul(i).
  const int cz = gt % CB;
  const bool has_z = cz < cout;
  double* const z_mine = z_at + cz / kFwKC * PLANE + cz % kFwKC;
  const double* const a_mine = h_at + cz / kFwKC * PLANE + cz % kFwKC;
  const auto ul = [&](int i) { return gt / CB + i * (kTileGroup / CB); };
  double kept[ACT && !FUSED ? PAIRS : 1][Q], a1[PAIRS], db = 0.0;
  auto request = [&](int64_t tile) {  // once every warp has read the last tile's dZ and H
    if (!boxes || gt == 0) {
      if (boxes) {
        fence_proxy_async();
        mbar_arrive_expect_tx(bar, unsigned((pz + (SWAP ? pz : ph)) * PLANE * sizeof(double)));
      }
      copy(z_at, &maps.seed, seed, tile, pz, cout, bar);
      if (SWAP) copy(h_at, &maps.activated, activated, tile, pz, cout, bar);
      else if (FUSED) copy(h_at, &maps.hidden, hidden, tile, ph, cin, bar);
      if (SWAP && boxes) {
        const int64_t left = total - tile * RT;
        prefetch_l2(hidden + tile * RT * cin, unsigned((left < RT ? left : RT) * cin * sizeof(double)));
      }
    }
    cp_async_commit();
    if constexpr (ACT) {
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        const int64_t u = tile * UT + ul(i);
        const bool live = has_z && u < units, full = live && u < rows.full;
        a1[i] = full ? aux[u * cout + cz] : 0.0;
        if constexpr (!FUSED) {
          const int n = live ? rows.count<Q>(u) : 0;
          const int64_t step = opaque(cout);
          const double* from = full ? activated + rows.row<Q>(u) * cout + cz  // value rows: their a1
                                    : aux + (rows.full + (u - rows.full) * Q) * cout + cz;
#pragma unroll
          for (int s = 0; s < Q; ++s, from += step) kept[i][s] = s < n ? *from : 0.0;
        }
      }
    }
  };
  auto form = [&](int64_t tile) {
    if (!has_z) return;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      const int64_t u = tile * UT + ul(i);
      double* at = z_mine + ul(i) * Q * LD;
      double z[Q];
      if constexpr (ACT) {
        double gz[Q], h[Q];
#pragma unroll
        for (int s = 0; s < Q; ++s) {
          gz[s] = at[s * LD];
          h[s] = FUSED ? a_mine[(ul(i) * Q + s) * LD] : kept[FUSED ? 0 : i][s];
        }
        if (u < rows.full) {
          tanh_vjp<DIM>(h, a1[i], gz, z);
        } else {
          const int n = u < units ? rows.count<Q>(u) : 0;
          const double* from = aux + (rows.full + (u - rows.full) * Q) * cout + cz;
#pragma unroll
          for (int s = 0; s < Q; ++s) z[s] = gz[s] * (FUSED ? (s < n ? from[int64_t(s) * cout] : 0.0) : h[s]);
        }
#pragma unroll
        for (int s = 0; s < Q; ++s) at[s * LD] = z[s];
      } else {
#pragma unroll
        for (int s = 0; s < Q; ++s) z[s] = at[s * LD];
      }
      db += z[0];
      if (u >= rows.full) {
#pragma unroll
        for (int s = 1; s < Q; ++s) db += z[s];
      }
    }
  };
  auto store_dz = [&](int64_t tile) {  // unfused: for affine_wgrad_tile
    if (!ACT || FUSED || i0 != 0) return;
    const int64_t left = total - tile * RT;
    const int n = left < RT ? int(left) : RT;
    double* to = dz + tile * RT * cout;  // dz is 16-byte aligned, RT even
    if (cout % 2 == 0) {
      for (int r = warp; r < n; r += kTileGroup / 32)
        for (int c = 2 * lane; c < cout; c += 64)
          *reinterpret_cast<double2*>(to + r * cout + c) =
              *reinterpret_cast<const double2*>(z_at + c / kFwKC * PLANE + r * LD + c % kFwKC);
    } else {
      for (int r = warp; r < n; r += kTileGroup / 32)
        for (int c = lane; c < cout; c += 32) to[r * cout + c] = z_at[c / kFwKC * PLANE + r * LD + c % kFwKC];
    }
  };

  if (gt == 0) {
    mbar_init(bar, 1);
    mbar_init(bar_h, 1);
  }
  __syncthreads();
  if (first < tiles) request(first);
  for (int c = tid >> 5; c < c8; c += 2 * kTileGroup / 32) {  // W rows c, columns i0 .. i0 + CB - 1
    const double* from = weight + int64_t(c) * cin + i0;
    if (vec_w) {
      for (int i = 2 * lane; i < CB; i += 64) {
        const bool ok = c < cout && i0 + i < cin;
        cp_async16(sw + c * LDW + i, ok ? from + i : weight, ok);
      }
    } else {
      for (int i = lane; i < CB; i += 32) {
        const bool ok = c < cout && i0 + i < cin;
        cp_async8(sw + c * LDW + i, ok ? from + i : weight, ok);
      }
    }
  }
  cp_async_commit();
  cp_async_wait<0>();
  __syncthreads();

  const int ci = i0 + wc * 16 + 2 * g;  // this thread's input channels ci, ci + 1
  const double* ap = sw + t * LDW + wc * 16 + 2 * g;
  const double* bp = z_at + (wr * 40 + g) * LD + t;
  // dW: output channels 16 (warp % 4) .., input channels 32 (warp / 4) ..
  constexpr int WN = FUSED ? 4 : 1;
  double wacc[WN][4];
#pragma unroll
  for (int j = 0; j < WN; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) wacc[j][e] = 0.0;
  const int wz = warp % 4 * 16, wh = warp / 4;
  const bool has_w = FUSED && wz < cout && wh < ph, has_h = i0 + wc * 16 < cin;
  const double* wa = z_at + wz / kFwKC * PLANE + t * LD + wz % kFwKC + g;
  const double* wb = h_at + wh * PLANE + t * LD + g;
  const Turns<2, kTileGroup> turns(group);
  const int early = c8 / 8 > kEarlySteps ? c8 / 8 - kEarlySteps : 0;
  unsigned phase = 0;
  // a copy's wait gave up: in this warp (H's); in this group, which keeps the turns and does no more work
  bool late = false, dead = false;
  for (int64_t tile = first; tile < tiles; tile += 2 * per) {
    double acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0.0;
    cp_async_wait<0>();
    if (!dead) dead = named_sync_or(1 + group, kTileGroup, boxes && !wait_copy(bar, phase, polls.tile));
    turns.take();
    if (!dead) form(tile);
    if constexpr (ACT) {
      named_sync(1 + group, kTileGroup);  // dZ is there, A has been read
      if (SWAP && !dead && (!boxes || gt == 0)) {
        if (boxes) {
          fence_proxy_async();
          mbar_arrive_expect_tx(bar_h, unsigned(ph * PLANE * sizeof(double)));
        }
        copy(h_at, &maps.hidden, hidden, tile, ph, cin, bar_h);
        cp_async_commit();
      }
    }
    if (!dead && has_h) {
      for (int p = 0; p < pz; ++p) {
        const double *a_at = ap + p * kFwKC * LDW, *b_at = bp + p * PLANE;
        const int left = c8 / 8 - 4 * p;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (k >= left) break;
          if (!FUSED && 4 * p + k == early) turns.pass();
          const double2 lo = *reinterpret_cast<const double2*>(a_at + 8 * k * LDW);
          const double2 hi = *reinterpret_cast<const double2*>(a_at + (8 * k + 4) * LDW);
          const double a[4] = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
          for (int j = 0; j < NT; ++j) mma_m16n8k8(acc[j], a, b_at[8 * j * LD + 8 * k], b_at[8 * j * LD + 8 * k + 4]);
        }
      }
    }
    if (SWAP) {
      if (!boxes) {
        cp_async_wait<0>();
        named_sync(1 + group, kTileGroup);
      } else if (!dead) {
        late = !wait_copy(bar_h, phase, polls.late);
      }
    }
    if (!FUSED && !(!dead && has_h)) turns.pass();
    if (FUSED && !(!dead && !late && has_w)) turns.pass();
    if (!dead && !late && has_w) {
#pragma unroll
      for (int r = 0; r < RT; r += 8) {
        if (r == RT - 8 * kEarlyRows) turns.pass();
        const double a[4] = {wa[r * LD], wa[r * LD + 8], wa[(r + 4) * LD], wa[(r + 4) * LD + 8]};
#pragma unroll
        for (int j = 0; j < WN; ++j) mma_m16n8k8(wacc[j], a, wb[r * LD + 8 * j], wb[(r + 4) * LD + 8 * j]);
      }
    }
    phase ^= 1;
    // every warp has read dZ and H
    if constexpr (SWAP) dead = named_sync_or(1 + group, kTileGroup, late) || dead;
    else named_sync(1 + group, kTileGroup);
    const int64_t next = tile + 2 * per;
    if (leave == kByThreads) {
      if (!dead) store_dz(tile);
      if (ACT && !FUSED) named_sync(1 + group, kTileGroup);  // dZ has been read for global memory
      if (next < tiles && !dead) request(next);
      if (!dead && ci < cin) {
        const bool two = ci + 1 < cin;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int64_t r = tile * RT + wr * 40 + 8 * j + 2 * t + e;
            if (r >= total) continue;
            double* to = dh + r * cin + ci;
            if (vec_out) {
              *reinterpret_cast<double2*>(to) = make_double2(acc[j][e], acc[j][2 + e]);
            } else {
              to[0] = acc[j][e];
              if (two) to[1] = acc[j][2 + e];
            }
          }
      }
    } else {
      const int y = int(tile * RT) + wr * 40;
      if (!dead) store_dz(tile);
      if (ACT && !FUSED) named_sync(1 + group, kTileGroup);  // dZ has been read for global memory
      if (leave == kOwnBoxes && next < tiles && !dead) request(next);
      if (!dead && i0 + wc * 16 < cin) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = 8 * j + 2 * t + e;
            *reinterpret_cast<double2*>(box + r * 16 + ((g ^ (r & 7)) << 1)) = make_double2(acc[j][e], acc[j][2 + e]);
          }
        send_box(&maps.dh, box, i0 + wc * 16, y, lane);
      }
      if (leave == kInTile) {
        named_sync(1 + group, kTileGroup);  // every box has left
        if (next < tiles && !dead) request(next);
      }
    }
  }
  if (lane == 0) bulk_wait();
  turns.close(count(first), count(blockIdx.x / blocks + (1 - group) * per));
  cp_async_wait<0>();
  __syncthreads();
  double* sums = smem;
  if (i0 == 0) {  // this CTA's [cout] of db
    sums[tid] = db;
    __syncthreads();
    if (tid < cout) {
      double s = 0.0;
      for (int k = tid; k < 2 * kTileGroup; k += CB) s += sums[k];
      db_parts[blockIdx.x / blocks * cout + tid] = s;
    }
    __syncthreads();
  }
  if constexpr (FUSED) {  // and [cout][cin] of dW: the groups' shares in order
    if (group == 1) {
#pragma unroll
      for (int j = 0; j < WN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sums[(wz + g + 8 * (e >> 1)) * CB + wh * 32 + 8 * j + 2 * t + (e & 1)] = wacc[j][e];
    }
    __syncthreads();
    double* mine = dw_parts + int64_t(blockIdx.x) * cout * cin;
    if (group == 0) {
#pragma unroll
      for (int j = 0; j < WN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = wz + g + 8 * (e >> 1), i = wh * 32 + 8 * j + 2 * t + (e & 1);
          if (c < cout && i < cin) mine[c * cin + i] = wacc[j][e] + sums[c * CB + i];
        }
    }
  }
}

// dW = dZ^T H, and db unless db_parts is null: a CTA's block of 16 MT (16 / WI) output x 32 WI input channels over its
// share of the rows, accumulators in registers throughout; 32-row stages of both operands by
// TMA boxes (or cp.async), two ahead of the MMAs.  dw_parts [share][cout][cin], db_parts
// [share][cout].
constexpr int kWgRows = 32, kWgStages = 3, kWgThreads = 512;
constexpr int wg_cout(int mt, int wi) { return 16 * mt * (16 / wi); }
constexpr size_t wg_smem(int mt, int wi) {
  return sizeof(double) * (size_t(kWgStages) * kWgRows * kFwLD * (wg_cout(mt, wi) / kFwKC + wi) + 2 * kWgStages);
}

template <int MT, int WI>
__global__ void __launch_bounds__(kWgThreads, 1)
    affine_wgrad_tile(const __grid_constant__ CUtensorMap dz_map, const __grid_constant__ CUtensorMap hidden_map,
                      const double* __restrict__ dz, const double* __restrict__ hidden,
                      double* __restrict__ dw_parts, double* __restrict__ db_parts,
                      int64_t total, int64_t full_rows, int q, int cin, int cout, bool boxes, Polls polls) {
  constexpr int CZ = wg_cout(MT, WI), CI = 32 * WI, PZ = CZ / kFwKC, P = PZ + WI, LD = kFwLD, PLANE = kWgRows * LD;
  extern __shared__ __align__(128) double smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  if (smem_u32(smem) & 127) {
    if (tid == 0) atomicExch(&g_affine_fault, 2);
    return;
  }
  const int bi = (cin + CI - 1) / CI, blocks = bi * ((cout + CZ - 1) / CZ), block = blockIdx.x % blocks;
  const int c0 = block / bi * CZ, i0 = block % bi * CI;
  const int64_t share = blockIdx.x / blocks, shares = gridDim.x / blocks, tiles = (total + kWgRows - 1) / kWgRows;
  const int64_t mine = share < tiles ? (tiles - 1 - share) / shares + 1 : 0;
  uint64_t *bars = reinterpret_cast<uint64_t*>(smem + kWgStages * P * PLANE), *empty = bars + kWgStages;
  auto load = [&](int64_t k, int stage) {  // the k-th of this CTA's tiles
    if (k >= mine) {
      if (!boxes) cp_async_commit();
      return;
    }
    const int64_t r0 = (share + k * shares) * kWgRows;
    double* to = smem + stage * P * PLANE;
    if (boxes) {
      if (tid != 0) return;
      fence_proxy_async();
      mbar_arrive_expect_tx(bars + stage, unsigned(P * PLANE * sizeof(double)));
      for (int p = 0; p < P; ++p)
        tma_load_2d(to + p * PLANE, p < PZ ? &dz_map : &hidden_map, p < PZ ? c0 + p * kFwKC : i0 + (p - PZ) * kFwKC, int(r0),
                    bars + stage);
    } else {
      for (int e = tid; e < P * kWgRows * kFwKC; e += kWgThreads) {
        const int p = e / (kWgRows * kFwKC), r = e / kFwKC % kWgRows, k = e % kFwKC;
        const bool z = p < PZ;
        const int c = z ? c0 + p * kFwKC + k : i0 + (p - PZ) * kFwKC + k, width = z ? cout : cin;
        const bool ok = r0 + r < total && c < width;
        const double* from = z ? dz : hidden;
        cp_async8(to + p * PLANE + r * LD + k, ok ? from + (r0 + r) * width + c : from, ok);
      }
      cp_async_commit();
    }
  };
  if (tid == 0)
    for (int s = 0; s < kWgStages; ++s) {
      mbar_init(bars + s, 1);
      mbar_init(empty + s, kWgThreads / 32);
    }
  __syncthreads();
  load(0, 0);
  load(1, 1);
  const int wz = warp / WI * 16 * MT, wh = warp % WI;
  const bool live = c0 + wz < cout && i0 + wh * 32 < cin;
  double acc[MT][4][4], db = 0.0;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[m][j][e] = 0.0;
  int stage = 0;
  unsigned phase = 0;
  for (int64_t k = 0; k < mine; ++k) {
    const int ahead = stage == 0 ? 2 : stage - 1;  // tile k - 1's stage, tile k + 2's next
    if (boxes) {
      // the warps meet only at the stages: a warp that is done with one starts on the next
      bool ok = mbar_wait(bars + stage, phase, polls.tile);
      if (tid == 0 && k + 2 < mine) {
        ok = ok && (k == 0 || mbar_wait(empty + ahead, unsigned((k - 1) / kWgStages) & 1, polls.late));
        if (ok) load(k + 2, ahead);
      }
      if (!__all_sync(0xffffffffu, ok)) {  // a wait gave up; the other warps' will too
        if (lane == 0) atomicExch(&g_affine_fault, 1);
        // The first warp, whose lane 0 asks for the tiles, stays (waits bounded too) until those
        // under way have landed: the block's memory is another's when it has ended.
        if (warp == 0) {
          const bool asked = __shfl_sync(0xffffffffu, ok, 0);  // for tile k + 2 as well
          const int64_t end = mine < k + 2 + asked ? mine : k + 2 + asked;
          for (int64_t n = k; n < end; ++n) mbar_wait(bars + n % kWgStages, unsigned(n / kWgStages) & 1);
        }
        return;
      }
    } else {
      cp_async_wait<1>();
      __syncthreads();
      load(k + 2, ahead);
    }
    const double* at = smem + stage * P * PLANE;
    if (live) {
      const double* za = at + wz / kFwKC * PLANE + t * LD + wz % kFwKC + g;
      const double* hb = at + (PZ + wh) * PLANE + t * LD + g;
#pragma unroll
      for (int r = 0; r < kWgRows; r += 8) {
        double a[MT][4], b[4][2];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) a[m][e] = za[16 * m + (r + 4 * (e >> 1)) * LD + 8 * (e & 1)];
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j][0] = hb[r * LD + 8 * j], b[j][1] = hb[(r + 4) * LD + 8 * j];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int j = 0; j < 4; ++j) mma_m16n8k8(acc[m][j], a[m], b[j][0], b[j][1]);
      }
    }
    if (db_parts && i0 == 0 && tid < CZ) {
      const int64_t r0 = (share + k * shares) * kWgRows;
      const double* z = at + tid / kFwKC * PLANE + tid % kFwKC;
      // order-0 rows: every q-th of the full points', every value row
      const int skip = int((q - r0 % q) % q);
      for (int r = r0 + skip < full_rows ? skip : int(full_rows > r0 ? full_rows - r0 : 0); r < kWgRows;
           r += r0 + r + q < full_rows ? q : r0 + r < full_rows ? int(full_rows - r0) - r : 1)
        db += z[r * LD];
    }
    __syncwarp();
    if (boxes && lane == 0) mbar_arrive(empty + stage);
    if (++stage == kWgStages) stage = 0, phase ^= 1;
  }
  if (!boxes) cp_async_wait<0>();
  double* to = dw_parts + share * cout * cin;
  if (live) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = c0 + wz + 16 * m + g + 8 * (e >> 1), i = i0 + wh * 32 + 8 * j + 2 * t + (e & 1);
          if (c < cout && i < cin) to[int64_t(c) * cin + i] = acc[m][j][e];
        }
  }
  if (db_parts && i0 == 0 && tid < CZ && c0 + tid < cout) db_parts[share * cout + c0 + tid] = db;
}

// dW [nw] and db [cout] from dw_parts [parts][nw] and db_parts [bias_parts][cout]: 16 strands of
// parts a value, each in order, then the strands in order
constexpr int kFinStrands = 16, kFinLanes = 32;
__global__ void __launch_bounds__(kFinStrands* kFinLanes)
    affine_finish(const double* __restrict__ dw_parts, int parts, const double* __restrict__ db_parts, int bias_parts,
                  double* __restrict__ dw, double* __restrict__ db, int64_t nw, int cout) {
  __shared__ double shared[kFinStrands][kFinLanes];
  const int lane = threadIdx.x % kFinLanes, strand = threadIdx.x / kFinLanes;
  const int64_t i = int64_t(blockIdx.x) * kFinLanes + lane;
  const bool bias = i >= nw, live = i < nw + cout;
  const double* from = bias ? db_parts + (i - nw) : dw_parts + i;
  const int64_t stride = bias ? cout : nw;
  const int n = bias ? bias_parts : parts;
  double s = 0.0;
  pdl_wait();
  if (live) {
#pragma unroll 10
    for (int k = strand; k < n; k += kFinStrands) s += from[k * stride];
  }
  shared[strand][lane] = s;
  __syncthreads();
  if (strand == 0 && live) {
    for (int k = 1; k < kFinStrands; ++k) s += shared[k][lane];
    if (bias) db[i - nw] = s;
    else dw[i] = s;
  }
}

unsigned grid_for(int64_t count) {
  const int64_t blocks = (count + kAffThreads - 1) / kAffThreads;
  return unsigned(blocks < (1 << 20) ? blocks : (1 << 20));
}

// What an adjoint call runs and the scratch that takes: dZ (unless it is the seed, or fused),
// then the partials of dW and db.
struct BackPlan {
  bool fused, tiled;         // one kernel for everything; dZ and dH in one kernel
  int64_t parts, bias_parts; // partials of dW and db
  int64_t dz, dw, doubles;   // scratch: dZ, then dW's partials, then db's
};
BackPlan back_plan(int64_t count, int cin, int cout, bool act, int sms) {
  BackPlan p;
  p.fused = cin <= 64 && cout <= 64;
  p.tiled = cout <= 128;
  p.dz = 0;
  if (p.fused) {
    p.parts = p.bias_parts = std::min<int64_t>((count + tile_rows(4) - 1) / tile_rows(4), sms);
  } else {
    const int mt = cin <= 64 || cout <= 64 ? 1 : 2, wi = cin <= 64 ? 2 : 4;
    const int64_t blocks = ((int64_t(cin) + 32 * wi - 1) / (32 * wi)) * ((int64_t(cout) + wg_cout(mt, wi) - 1) / wg_cout(mt, wi));
    p.parts = std::min<int64_t>((count + kWgRows - 1) / kWgRows, std::max<int64_t>(sms / blocks, 1));
    const int64_t across = (int64_t(cin) + 127) / 128;
    p.bias_parts = p.tiled ? std::min<int64_t>((count + tile_rows(8) - 1) / tile_rows(8), std::max<int64_t>(sms / across, 1))
                           : p.parts;
    if (act) p.dz = (count * cout + 15) / 16 * 16;
  }
  p.dw = p.parts * cout * cin;
  p.doubles = p.dz + p.dw + p.bias_parts * cout;
  return p;
}

template <int DIM, bool ACT, int WC, bool FUSED>
cudaError_t launch_backward_tile(const double* hidden, const double* weight, const double* activated, const double* aux,
                                 const double* seed, double* dz, double* dh, double* dw_parts, double* db_parts, int64_t per,
                                 Packed rows, int cin, int cout, cudaStream_t stream) {
  const auto kernel = affine_backward_tile<DIM, ACT, WC, FUSED>;
  size_t smem = back_smem(WC, FUSED, cin, cout);
  const int64_t total = rows.full * Jet<DIM>::Q + rows.value, blocks = (int64_t(cin) + 16 * WC - 1) / (16 * WC);
  const bool boxes = cout % 2 == 0 && aligned16(seed) && total < INT_MAX - 1024 &&
                     (!FUSED || (cin % 2 == 0 && aligned16(hidden) && aligned16(activated)));
  BackMaps maps{};
  cudaError_t e = cudaSuccess;
  if (boxes) e = matrix_map(&maps.seed, seed, total, cout, kFwLD, tile_rows(WC));
  if (e == cudaSuccess && boxes && FUSED) e = matrix_map(&maps.hidden, hidden, total, cin, kFwLD, tile_rows(WC));
  if (e == cudaSuccess && boxes && FUSED && ACT) e = matrix_map(&maps.activated, activated, total, cout, kFwLD, tile_rows(WC));
  const bool vec_out = cin % 2 == 0 && aligned16(dh);
  const int planes = tile_planes(cout) + (FUSED ? std::max(tile_planes(cin), tile_planes(cout)) : 0);
  const size_t own = smem + 2 * kBoxesBytes + 1024;
  const Leave leave = !vec_out || total >= INT_MAX - 1024                                            ? kByThreads
                      : own <= kTileSmem                                                             ? kOwnBoxes
                      : sizeof(double) * planes * tile_rows(WC) * kFwLD >= size_t(kBoxesBytes) + 1024 ? kInTile
                                                                                                     : kByThreads;
  if (leave == kOwnBoxes) smem = own;
  if (e == cudaSuccess && leave != kByThreads) e = matrix_map(&maps.dh, dh, total, cin, 16, 40, true);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
  if (e != cudaSuccess) return e;
  kernel<<<unsigned(per * blocks), 2 * kTileGroup, smem, stream>>>(maps, hidden, weight, activated, aux, seed, dz, dh,
                                                                  dw_parts, db_parts, rows, cin, cout, boxes, vec_out,
                                                                  cin % 2 == 0 && aligned16(weight), leave, t_polls);
  return cudaGetLastError();
}

template <int MT, int WI>
cudaError_t launch_wgrad(const double* dz, const double* hidden, double* dw_parts, double* db_parts, int64_t parts,
                         int64_t total, int64_t full_rows, int q, int cin, int cout, cudaStream_t stream) {
  const auto kernel = affine_wgrad_tile<MT, WI>;
  const size_t smem = wg_smem(MT, WI);
  const int64_t blocks = ((int64_t(cin) + 32 * WI - 1) / (32 * WI)) * ((int64_t(cout) + wg_cout(MT, WI) - 1) / wg_cout(MT, WI));
  const bool boxes = cin % 2 == 0 && cout % 2 == 0 && aligned16(dz) && aligned16(hidden) && total < INT_MAX - 1024;
  CUtensorMap dz_map{}, hidden_map{};
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
  if (e == cudaSuccess && boxes) e = matrix_map(&dz_map, dz, total, cout, kFwLD, kWgRows);
  if (e == cudaSuccess && boxes) e = matrix_map(&hidden_map, hidden, total, cin, kFwLD, kWgRows);
  if (e != cudaSuccess) return e;
  kernel<<<unsigned(parts * blocks), kWgThreads, smem, stream>>>(dz_map, hidden_map, dz, hidden, dw_parts, db_parts, total,
                                                                full_rows, q, cin, cout, boxes, t_polls);
  return cudaGetLastError();
}

template <int DIM, bool ACT>
cudaError_t backward(const double* hidden, const double* weight, const double* activated, const double* aux,
                     const double* seed, double* dh, double* dw, double* db, double* scratch, const BackPlan& plan,
                     Packed rows, int cin, int cout, cudaStream_t stream) {
  constexpr int Q = Jet<DIM>::Q;
  const int64_t total = rows.full * Q + rows.value;
  const bool whole = plan.parts == 1 && plan.bias_parts == 1;  // a single share is the gradient
  double *dz = plan.dz ? scratch : nullptr, *dw_parts = whole ? dw : scratch + plan.dz;
  double* db_parts = whole ? db : scratch + plan.dz + plan.dw;
  cudaError_t e = cudaSuccess;
  if (plan.fused) {
    e = launch_backward_tile<DIM, ACT, 4, true>(hidden, weight, activated, aux, seed, dz, dh, dw_parts, db_parts, plan.parts,
                                                rows, cin, cout, stream);
  } else {
    const double* z = ACT ? dz : seed;
    if (plan.tiled) {
      e = launch_backward_tile<DIM, ACT, 8, false>(hidden, weight, activated, aux, seed, dz, dh, dw_parts, db_parts,
                                                   plan.bias_parts, rows, cin, cout, stream);
    } else {
      if constexpr (ACT) {
        affine_seed<DIM><<<grid_for(rows.units<Q>() * cout), kAffThreads, 0, stream>>>(activated, aux, seed, dz, rows, cout);
        e = cudaGetLastError();
      }
      // dH = dZ W: the forward product over the output channels, with W read across
      if (e == cudaSuccess)
        e = forward<DIM, false>(cout, cin, false, false, z, weight, static_cast<const double*>(nullptr),
                                static_cast<const double*>(nullptr), dh, static_cast<double*>(nullptr),
                                static_cast<double*>(nullptr), rows, cout, cin, true, stream);
    }
    if (e != cudaSuccess) return e;
    const auto wgrad = cin <= 64 ? launch_wgrad<1, 2> : cout <= 64 ? launch_wgrad<1, 4> : launch_wgrad<2, 4>;
    e = wgrad(z, hidden, dw_parts, plan.tiled ? nullptr : db_parts, plan.parts, total, rows.full * Q, Q, cin, cout, stream);
  }
  if (e != cudaSuccess || whole) return e;
  const int64_t nw = int64_t(cin) * cout;
  return launch_dependent(affine_finish, unsigned((nw + cout + kFinLanes - 1) / kFinLanes), kFinStrands * kFinLanes, 0, stream,
                          dw_parts, int(plan.parts), db_parts, int(plan.bias_parts), dw, db, nw, cout);
}

}  // namespace
}  // namespace flashns_b200

using namespace flashns_b200;

extern "C" {

int flashns_b200_layer_wait_polls(unsigned tile, unsigned late) {
  if (tile > kMbarSpins || late > kMbarSpins) return int(cudaErrorInvalidValue);
  t_polls = {tile, late};
  return int(cudaSuccess);
}

int flashns_b200_affine(int dim, int activation, const double* hidden, const double* weight, const double* bias,
                        const double* residual, double* out, double* activated, double* aux, int64_t full_points,
                        int64_t value_points, int cin, int cout, cudaStream_t stream) {
  if (!layer_sizes_ok(dim, full_points, value_points, cin) || !layer_sizes_ok(dim, full_points, value_points, cout) ||
      int64_t(cin) * cout > kMostWeights || (activation != 0 && activation != 1) || (!activation && (activated || aux)))
    return int(cudaErrorInvalidValue);
  const Packed rows{full_points, value_points};
  const int64_t count = full_points * (dim == 2 ? 10 : 20) + value_points;
  if (count == 0) return int(cudaSuccess);
  if (!hidden || !weight || !bias || !out) return int(cudaErrorInvalidValue);
  const size_t in = size_t(count) * cin * sizeof(double), bytes = size_t(count) * cout * sizeof(double);
  const size_t weights = size_t(cin) * cout * sizeof(double), small = size_t(cout) * sizeof(double);
  if (outputs_overlap({{out, bytes}, {activated, bytes}, {aux, size_t(full_points + value_points) * small}},
                      {{hidden, in}, {weight, weights}, {bias, small}, {residual, bytes}}))
    return int(cudaErrorInvalidValue);
  // TMA boxes: rows on 16-byte boundaries, row numbers that fit their 32-bit coordinate
  const bool boxes = cin % 2 == 0 && aligned16(hidden) && count < INT_MAX - 1024;
  const auto run = [&](auto launch) { return int(launch(cin, cout, full_points == 0, boxes, hidden, weight, bias, residual, out, activated, aux, rows, cin, cout, false, stream)); };
  if (dim == 2) return activation ? run([](auto... a) { return forward<2, true>(a...); }) : run([](auto... a) { return forward<2, false>(a...); });
  return activation ? run([](auto... a) { return forward<3, true>(a...); }) : run([](auto... a) { return forward<3, false>(a...); });
}

int flashns_b200_affine_vjp_scratch(int dim, int activation, int64_t full_points, int64_t value_points, int cin,
                                    int cout, size_t* bytes) {
  if (!layer_sizes_ok(dim, full_points, value_points, cin) || !layer_sizes_ok(dim, full_points, value_points, cout) ||
      int64_t(cin) * cout > kMostWeights || (activation != 0 && activation != 1) || !bytes)
    return int(cudaErrorInvalidValue);
  const int64_t count = full_points * (dim == 2 ? 10 : 20) + value_points;
  *bytes = 0;
  if (count == 0) return int(cudaSuccess);
  int sms = 0;
  const cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return int(e);
  *bytes = size_t(back_plan(count, cin, cout, activation != 0, sms).doubles) * sizeof(double);
  return int(cudaSuccess);
}

int flashns_b200_affine_vjp(int dim, int activation, const double* hidden, const double* weight,
                            const double* activated, const double* aux, const double* seed, double* d_hidden,
                            double* d_weight, double* d_bias, double* scratch, size_t scratch_bytes,
                            int64_t full_points, int64_t value_points, int cin, int cout, cudaStream_t stream) {
  if (!layer_sizes_ok(dim, full_points, value_points, cin) || !layer_sizes_ok(dim, full_points, value_points, cout) ||
      int64_t(cin) * cout > kMostWeights || (activation != 0 && activation != 1) || !d_weight || !d_bias)
    return int(cudaErrorInvalidValue);
  const Packed rows{full_points, value_points};
  const int q = dim == 2 ? 10 : 20;
  const int64_t count = full_points * q + value_points;
  if (count == 0) {
    cudaError_t e = cudaMemsetAsync(d_weight, 0, size_t(cin) * cout * sizeof(double), stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(d_bias, 0, size_t(cout) * sizeof(double), stream);
    return int(e);
  }
  if (!hidden || !weight || !seed || !d_hidden || !scratch || !aligned16(scratch) || (activation && (!activated || !aux)))
    return int(cudaErrorInvalidValue);
  const size_t in = size_t(count) * cin * sizeof(double), bytes = size_t(count) * cout * sizeof(double);
  const size_t weights = size_t(cin) * cout * sizeof(double), small = size_t(cout) * sizeof(double);
  if (outputs_overlap({{d_hidden, in}, {d_weight, weights}, {d_bias, small}, {scratch, scratch_bytes}},
                      {{hidden, in}, {weight, weights}, {seed, bytes}, {activation ? activated : nullptr, bytes},
                       {activation ? aux : nullptr, size_t(full_points + value_points) * small}}))
    return int(cudaErrorInvalidValue);
  // at least one share of dW and db, whatever the device
  if (scratch_bytes < weights + small) return int(cudaErrorInvalidValue);
  int sms = 0;
  const cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return int(e);
  const BackPlan plan = back_plan(count, cin, cout, activation != 0, sms);
  if (scratch_bytes < size_t(plan.doubles) * sizeof(double)) return int(cudaErrorInvalidValue);
  const auto run = dim == 2 ? (activation ? backward<2, true> : backward<2, false>)
                            : (activation ? backward<3, true> : backward<3, false>);
  return int(run(hidden, weight, activated, aux, seed, d_hidden, d_weight, d_bias, scratch, plan, rows, cin, cout,
                 stream));
}

}  // extern "C"
