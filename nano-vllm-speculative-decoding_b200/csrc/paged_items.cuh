// The item sequence of the paged attention kernels and how a persistent grid shares it: used by the bf16 cache's kernel
// (verify_attention.cu) and the 8-bit cache's (verify_attention_fp8.cu).
//
// An item is a (row, KV head); its keys are cut into 128-key tiles, and the items' tiles form one sequence that is
// split into equal contiguous shares, one per CTA.  Args holds the row metadata (cu_seqlens_q, cu_seqlens_k,
// context_lens, q_per_seq, R, block_tables, W, block_size, Hkv, err); the CTA's Smem its share (x_begin, x_end,
// row_tile0, b_start, r0).
#pragma once

#include "common.cuh"
#include "sm100.cuh"

#include <cudaTypedefs.h>

namespace specdec {
namespace attention {

using namespace sm100;

constexpr int kHeadDim = 128;
constexpr int kKeysPerTile = 128;
constexpr int kCols = 32;              // packed query columns (group x positions)
constexpr float kNegBig = -1.0e30f;    // start value of the running maxima (finite: no -inf arithmetic)

// One piece of a split item: O^T columns (unnormalised, relative to the piece's running maxima) then the maxima m
// and the sums l of the 32 columns.
constexpr int kPartialFloats = kCols * kHeadDim + 2 * kCols;

// Workspace: two piece slots per SM (a size fixed per device), then R * Hkv arrival counters (256-byte padded).
// The counters sit at the same offset for calls of every shape, so a workspace zeroed once stays valid: every
// call leaves the counters it used at zero, and no call's pieces overlap another call's counters.
inline long long partial_bytes(int sm_count) { return 2LL * sm_count * kPartialFloats * 4; }
inline long long counters_bytes(long long R, int Hkv) { return (R * Hkv * 4 + 255) / 256 * 256; }
inline long long workspace_bytes(long long R, int Hkv, int sm_count) {
  return partial_bytes(sm_count) + counters_bytes(R, Hkv);
}
static_assert((kPartialFloats * 4 * 2) % 256 == 0, "counters stay 256-byte aligned");

// The driver's tensor-map encoder (one entry point for every device), looked up on first use; the initialisation
// of a function-local static is thread-safe.
inline PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = []() -> PFN_cuTensorMapEncodeTiled_v12000 {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    return nullptr;
  }();
  return fn;
}

// Max over the warp's 32 lanes in one instruction (sm_100a redux.sync on f32).
__device__ __forceinline__ float warp_max_redux(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// Sum over the 32 lanes of 16 columns held by every lane; lane j ends with column (j & 15)'s sum; v is consumed.
__device__ __forceinline__ float column_reduce16(float (&v)[16], int lane) {
#pragma unroll
  for (int c = 0; c < 16; ++c) v[c] += __shfl_xor_sync(0xffffffffu, v[c], 16);
#pragma unroll
  for (int w = 8; w >= 1; w >>= 1) {
    const bool upper = (lane & w) != 0;
#pragma unroll
    for (int c = 0; c < w; ++c) {
      const float send = upper ? v[c] : v[c + w];
      const float keep = upper ? v[c + w] : v[c];
      v[c] = keep + __shfl_xor_sync(0xffffffffu, send, w);
    }
  }
  return v[0];
}

// A row's queries and keys; nt = 0 when the row has no work (no queries, or metadata that the kernel rejects).
struct RowInfo {
  int q_start, ql, L, nt;
};

// kStrict: query rows outside the T of the call are rejected too, and a row of queries without a key is an item of no
// tiles (its output is the kernel's to clear), not an error.
template <int QMAX, bool kStrict = false, typename Args>
__device__ __forceinline__ RowInfo row_info(const Args& a, int b, bool report) {
  RowInfo r;
  if (a.cu_seqlens_q) {
    r.q_start = a.cu_seqlens_q[b];
    r.ql = a.cu_seqlens_q[b + 1] - r.q_start;
    r.L = a.cu_seqlens_k[b + 1] - a.cu_seqlens_k[b];
  } else {
    r.q_start = b * a.q_per_seq;
    r.ql = a.q_per_seq;
    r.L = a.context_lens[b];
  }
  r.nt = 0;
  if (r.ql > 0) {
    if constexpr (kStrict) {
      if (r.q_start < 0 || r.ql > a.T - r.q_start) r.L = -1;
      if (r.ql <= QMAX && r.L == 0) return r;
    }
    if (r.ql > QMAX || r.L <= 0 || r.L > a.W * a.block_size) {   // inconsistent metadata: report, never read
      if (report) atomicCAS(a.err, 0, 2);
    } else {
      r.nt = (r.L + kKeysPerTile - 1) / kKeysPerTile;
    }
  }
  return r;
}

// The item sequence: items (row b, KV head h) in row-major order, item (b, h) holding the sequence's tiles
// [A, A + r.nt).  Each role of a CTA walks it from the item holding x_begin to the one holding x_end - 1.
template <int QMAX, bool kStrict = false>
struct Walk {
  int b, h;
  long long A;
  RowInfo r;
  template <typename Args, typename Smem>
  __device__ __forceinline__ void start(const Args& a, const Smem& S) {
    b = S.b_start;
    r = RowInfo{S.r0[0], S.r0[1], S.r0[2], S.r0[3]};   // found by the prologue
    h = (int)(S.x_begin - S.row_tile0) / r.nt;        // within the row: nt * Hkv tiles, 32 bits
    A = S.row_tile0 + (long long)h * r.nt;
  }
  template <typename Args>
  __device__ __forceinline__ void next(const Args& a) {
    A += r.nt;
    if (++h == a.Hkv) {
      h = 0;
      do {
        ++b;
        r = b < a.R ? row_info<QMAX, kStrict>(a, b, false) : RowInfo{0, 0, 0, 1};
      } while (r.nt == 0);
    }
  }
  // this CTA's tiles of the item: item-local [t0, t1)
  __device__ __forceinline__ int t0(long long x_begin) const { return (int)(x_begin > A ? x_begin - A : 0); }
  __device__ __forceinline__ int t1(long long x_end) const {
    return (int)(x_end < A + r.nt ? x_end - A : (long long)r.nt);
  }
};

// Tile-by-tile cursor over the CTA's share: the segment (item piece) index n of the current tile and whether the
// tile is the segment's first / last.
template <int QMAX, bool kStrict = false>
struct Cursor {
  Walk<QMAX, kStrict> w;
  int n, left;
  bool first;
  template <typename Args, typename Smem>
  __device__ __forceinline__ void start(const Args& a, const Smem& S) {
    w.start(a, S);
    n = 0;
    left = w.t1(S.x_end) - w.t0(S.x_begin);
    first = true;
  }
  __device__ __forceinline__ bool last() const { return left == 1; }
  template <typename Args>
  __device__ __forceinline__ void advance(const Args& a, long long x_begin, long long x_end) {
    if (--left == 0) {
      w.next(a);
      ++n;
      left = w.t1(x_end) - w.t0(x_begin);
      first = true;
    } else {
      first = false;
    }
  }
};

// x * y / z for y and z up to the grid (< 256): in 32 bits where the product fits, as it does below 2^24 tiles.
__device__ __forceinline__ long long mul_div(long long x, long long y, long long z) {
  return x < (1LL << 24) ? (long long)((unsigned)x * (unsigned)y / (unsigned)z) : x * y / z;
}
// ceil(x * y / z) for y up to the grid (< 256) and x up to z: the same.
__device__ __forceinline__ long long mul_ceil_div(long long x, long long y, long long z) {
  return z < (1LL << 24) ? (long long)(((unsigned)x * (unsigned)y + (unsigned)z - 1u) / (unsigned)z) : (x * y + z - 1) / z;
}
__device__ __forceinline__ long long ceil_div(long long x, long long y) { return (x + y - 1) / y; }

// This CTA's share [xb, xe) of the tile sequence, split evenly over Ge = min(grid, T) CTAs, and the row holding its
// first tile: two passes of 32 rows at a time over the row metadata, by one warp.
struct Share {
  long long T, Ge, xb, xe, row0;
  int bstart;
  RowInfo r0;
};
template <int QMAX, bool kStrict = false, typename Args>
__device__ __forceinline__ Share find_share(const Args& a, int lane) {
  long long row_tiles = 0;
  for (int b0 = 0; b0 < a.R; b0 += 32) {
    const int b = b0 + lane;
    const int nt = b < a.R ? row_info<QMAX, kStrict>(a, b, true).nt : 0;
    row_tiles += __reduce_add_sync(0xffffffffu, (unsigned)nt);
  }
  const long long T = row_tiles * a.Hkv;
  const long long Ge = T < (long long)gridDim.x ? T : (long long)gridDim.x;
  const long long c = blockIdx.x;
  long long xb = 0, xe = 0, row0 = 0;
  int bstart = 0;
  RowInfo r0{0, 0, 0, 1};
  if (c < Ge) {
    xb = mul_div(T, c, Ge);
    xe = mul_div(T, c + 1, Ge);
    long long pre = 0;
    for (int b0 = 0; b0 < a.R; b0 += 32) {
      const int b = b0 + lane;
      const RowInfo ri = b < a.R ? row_info<QMAX, kStrict>(a, b, false) : RowInfo{0, 0, 0, 0};
      const long long v = (long long)ri.nt * a.Hkv;
      long long inc = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      const long long first = pre + inc - v;
      const unsigned hit = __ballot_sync(0xffffffffu, v > 0 && xb >= first && xb < first + v);
      if (hit) {
        const int src = __ffs(hit) - 1;
        bstart = b0 + src;
        row0 = __shfl_sync(0xffffffffu, first, src);
        r0.q_start = __shfl_sync(0xffffffffu, ri.q_start, src);
        r0.ql = __shfl_sync(0xffffffffu, ri.ql, src);
        r0.L = __shfl_sync(0xffffffffu, ri.L, src);
        r0.nt = __shfl_sync(0xffffffffu, ri.nt, src);
        break;
      }
      pre += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
  return Share{T, Ge, xb, xe, row0, bstart, r0};
}

}  // namespace attention
}  // namespace specdec
