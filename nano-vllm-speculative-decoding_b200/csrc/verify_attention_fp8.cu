// Verify / decode attention over the 8-bit paged cache (e4m3 codes, a scale per group of slots and KV head) for sm_100a.
//
// Reference behaviour: Attention.forward, verify and decode branches (nanovllm/layers/attention.py:59-77), over keys and
// values that are code * scale:
//   o = sum_j p_j vs_j v_j,  p = softmax_j(softmax_scale * ks_j * (q . k_j)),
// causal (bottom-right aligned) or over the whole context; a query that sees no key gives zeros.
//
// What bounds it: HBM.  A 128-key tile of one head is 2 * 16 KB of codes (half the bf16 cache's) and 64 B of scales for
// 4 * 128 * 128 * 32 FLOP, 128 FLOP a byte.  The cache's layout keeps a head's rows of a block together, so a tile is one
// contiguous 16 KB.
//
// Design.  The item sequence, its split over a persistent grid and the merge of split items are the bf16 kernel's
// (paged_items.cuh, verify_attention.cu).  What differs is how 8-bit codes meet the tensor core without being widened in
// shared memory (widening a tile would cost a read of 32 KB and a write of 64 KB of shared memory a tile, more than the
// 748 ns that HBM leaves it):  the MMAs are kind::f8f6f4 with the cache's codes as the A operand straight from the TMA's
// tile, and the other operand, which is 16-bit by nature, goes in as a sum of 8-bit parts side by side in N:
//   S^T[128 keys x 2*32] = K . [q1 | q2]^T   q = 2^e (q1 + q2 / 16), both e4m3: bf16's 8 bits are 4 + 4, so the split is
//                                            exact down to 2^-14 of the item's largest query element (beyond: an absolute
//                                            2^-22 of it), e from that element
//   O^T[128 dims x 3*32] += V^T . [p1 | p2 | p3]^T   p = p1 + p2 / 8 + p3 / 64, all e5m2: 3 bits each, what is left over
//                                            taken 8 times, so that each part has e5m2's whole range: off by 2^-9 of p (what
//                                            bf16 gives) or, below 2^-21 of the column's running maximum, 2^-30 of that
// N-wise parts read A once; stacked along K they would read it 2 and 3 times, and A's reads of shared memory are what an
// MMA with so few columns costs.  The parts' sums are taken in fp32 after TMEM.  (Parts on one scale cost 1 % less, 354 for
// 357 us at 16k contexts, 424 for 430 sustained, and lost what is below 2^-24 of the maximum: 1 % of a row of 262,144 keys,
// one of them e^17 times as likely as each other, in one piece.  The denominator sums p itself.  Taking the leftovers 8 times
// only for long rows, behind a branch: 432 us.)
// The scales never touch the codes: ks_j multiplies the score, and vs_j goes into the exponent: with t_j = s_j + log2 vs_j
// the running maximum is over t, the tensor core gets p'_j = 2^(t_j - m) (so the largest contribution keeps every bit
// whatever the scales' spread), and the denominator sums p'_j / vs_j.  (fp32's range bounds the spread: a key whose vs is
// 2^-110 of another's can be missing from the denominator, where it counts 2^-23 of that other's weight or, only past 2^110,
// more.)
//   warp 0       TMA producer: K tiles and the scales  warps 4-11   softmax over keys (a TMEM lane is a key; two groups of
//   warp 1       TMEM allocator, MMA issuer                          16 columns each), P parts, O rescale, epilogue
//   warp 2       prologue                              warps 12-15  query parts of the next items; rows without keys
//   warp 3       TMA producer: the V tiles
// Softmax: online per column with lazy rescaling (O is rescaled when a column's maximum grows by more than 2^8; p' reaches
// 2^15 then, in e5m2's range), masked by key index.  V rows past the context are zeroed in shared memory.
// A softmax step takes a pair of tiles: its fixed costs (score load, the vote on the maxima, the proxy fence, the
// hand-over: some 700 clocks that two warps a scheduler cannot hide) are paid once for 256 keys, and a warp has two
// independent tiles' arithmetic to interleave (16k contexts: 379 -> 362 us; one tile ahead in software instead: 595 us).
// The MMA warp runs converged with a predicated leader lane: issued from a divergent lane an MMA cost about 100 clocks,
// more than its execution (429 -> 376 us).  Rings deeper than this lost time (5 stages of K and V: 15 % at 3k contexts).
// Measured (32 query and 8 KV heads, in a graph): 64 rows of 1 to 8 queries on 16k contexts 355 to 367 us (2144 MB, 0.90 to
// 0.93 of the copy rate; the bf16 kernel on its cache 630 to 674 us) where the SMs hold 1.9 GHz; called for seconds on end
// the GPU reaches its 1000 W and the clock falls to 1.5 to 1.7 GHz: 424 to 432 us (0.77), a pair's 2700 clocks being the
// softmax's chain then.  64 draft blocks of 7 on 3k 88 to 92 us (95 sustained), 32 rows on 1k 30 us, one token on 1000 keys
// 13 us: what an item costs beside its tiles (query parts, first wait, pieces and their merge).  Four of the softmax's
// registers spill; their reloads are in its loop, some 6 a pair of tiles, 0.6 % of the instructions executed.  At one clock
// and without gain: a warp each for the score and the PV MMAs (the softmax then waits for P's buffer itself: 371 against
// 354 us), and 8 columns a group for items of at most 16 (352 against 347 us: the chain is latency, not columns).
#include "paged_items.cuh"
#include "specdec_b200.h"

#include <cuda_fp8.h>
#include <math.h>

namespace specdec {
namespace attention_fp8 {

using namespace attention;

constexpr int kSubKeys = 32;                          // an item's last tile loads in 32-key sub-boxes
constexpr int kStages = 4;                            // K ring and V ring depth (tiles): 128 KB in flight
// Scale ring depth.  A tile's scales arrive on its K tile's barrier.  The entry of tile g is written again for tile
// g + 16, which K's producer reaches after S of tile g + 12 is done: at least six pairs on, and a pair's scores go out
// after P of the pair two before it.
constexpr int kScaleStages = 16;
static_assert(kScaleStages >= kStages + 4, "a scale entry must outlive the softmax's reads");
constexpr int kGroups = 2, kGroupCols = kCols / kGroups;   // softmax warpgroups, 16 columns each
constexpr int kSoftmaxWarp = 4, kSoftmaxThreads = kGroups * 128, kSoftmaxWarps = kSoftmaxThreads / 32;
constexpr int kQueryWarp = kSoftmaxWarp + kSoftmaxWarps;
constexpr int kThreads = kQueryWarp * 32 + 128;
// The softmax holds a pair of tiles in registers: the other warpgroups (0: producers and MMA, 3: queries) hand theirs over.
// The shares must fit what the block is launched with, which the host checks.
constexpr int kSoftmaxRegs = 168, kProducerRegs = 72;
constexpr int kLaunchRegs = (kSoftmaxRegs * kSoftmaxThreads + kProducerRegs * 256 + kThreads - 1) / kThreads;
constexpr int kBarMerge = 1 + kGroups, kBarQuery = 2 + kGroups;   // named barriers: 1 .. kGroups are the groups'
constexpr int kTileBytes = kKeysPerTile * kHeadDim;   // 16 KB of codes
constexpr int kQParts = 2, kPParts = 3;
constexpr int kQBytes = kQParts * kCols * kHeadDim;   // 8 KB, double-buffered by item
constexpr int kPPartBytes = kKeysPerTile * kCols;     // 4 KB
constexpr int kPBytes = kPParts * kPPartBytes;        // 12 KB a tile; a pair's 24 KB double-buffered
constexpr uint32_t kTmemCols = 512;                   // two pairs of S (2 x 64 columns), then O0 and O1 of 96
constexpr uint32_t kTmemSTile = 64, kTmemSPair = 128, kTmemO = 256, kTmemOStride = 128;
constexpr float kPBias = 7.0f;                        // p' is kept 2^7 up: its range is [2^-24, 2^8] of the maximum
constexpr float kMinScale = 7.888609052210118e-31f;   // 2^-100, the store's smallest scale

constexpr int kErrTimeoutQ = 11, kErrTimeoutK = 12, kErrTimeoutV = 13, kErrTimeoutS = 14, kErrTimeoutP = 15,
              kErrTimeoutO = 16, kErrTimeoutEmpty = 17, kErrPage = 5;

struct Args {
  const __nv_bfloat16* q;    // [T, H, D]
  long long q_row_stride;
  const float *k_scale, *v_scale;
  const int* cu_seqlens_q;   // [R + 1] or null (decode mode)
  const int* cu_seqlens_k;
  const int* context_lens;   // [R] (decode mode)
  int q_per_seq, R, T;
  const int* block_tables;   // [R, W]
  int W, block_size, group;
  int num_blocks;
  int H, Hkv;
  float scale_log2;          // softmax_scale * log2(e)
  int causal;
  __nv_bfloat16* out;
  long long out_row_stride;
  int* counters;
  float* partial;
  int* err;
};

struct Smem {
  uint64_t q_full[2], q_empty[2];
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t s_full[2], p_full[2], o_done[2], o_free[2];
  alignas(16) float scales[kScaleStages][2][kKeysPerTile / 16];   // [ring][K, V][group of the tile]
  alignas(16) float red_max[2][32][4];   // [pair parity][column][warp] maxima
  alignas(16) float red_sum[32][4];
  unsigned red_q[4];
  float q_scale[4];          // by item & 3: the item's 2^e
  uint32_t tmem_base;
  int abort;
  long long total_tiles, x_begin, x_end, row_tile0;
  int b_start, active;
  int r0[4];
  int page0;                 // page of the share's first tile
  int last_piece;
};

constexpr int kOffQ = 0;
constexpr int kOffK = kOffQ + 2 * kQBytes;
constexpr int kOffV = kOffK + kStages * kTileBytes;
constexpr int kOffP = kOffV + kStages * kTileBytes;
constexpr int kOffCtl = kOffP + 4 * kPBytes;
constexpr int kSmemBytes = kOffCtl + (int)sizeof(Smem) + 1024;   // + alignment slack
static_assert(kSmemBytes <= 232448, "shared memory above the sm_100 per-CTA limit");

__device__ __forceinline__ float2 decode_e4m3x2(unsigned pair) {
  return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(pair & 0xffffu), __NV_E4M3)));
}
__device__ __forceinline__ unsigned encode_e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ unsigned half2_bits(__half2 h) { return *reinterpret_cast<unsigned*>(&h); }
__device__ __forceinline__ __half2 bits_half2(unsigned u) { return *reinterpret_cast<__half2*>(&u); }

// The page of a row's key, block 0 in place of an id outside the cache.
__device__ __forceinline__ int page_of(const Args& a, const int* table, int key0) {
  int page = table[key0 / a.block_size];
  if (page < 0 || page >= a.num_blocks) {
    atomicCAS(a.err, 0, kErrPage);
    page = 0;
  }
  return page;
}

// Pair-by-pair cursor over the CTA's share: the segment (item piece) number n, whether the pair is its first or last, and
// whether it has a second tile (a piece of an odd number of tiles ends in a single).
template <int QMAX>
struct PairCursor {
  Walk<QMAX, true> w;
  int n, left;
  bool first;
  __device__ __forceinline__ void start(const Args& a, const Smem& S) {
    w.start(a, S);
    n = 0;
    left = w.t1(S.x_end) - w.t0(S.x_begin);
    first = true;
  }
  __device__ __forceinline__ bool two() const { return left >= 2; }
  __device__ __forceinline__ bool last() const { return left <= 2; }
  __device__ __forceinline__ void advance(const Args& a, long long x_begin, long long x_end) {
    first = last();
    left -= 2;
    if (left <= 0) {
      w.next(a);
      ++n;
      left = w.t1(x_end) - w.t0(x_begin);
    }
  }
};

template <int G>
__global__ void __launch_bounds__(kThreads, 1)
    verify_attention_fp8_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                                const __grid_constant__ CUtensorMap kmap32, const __grid_constant__ CUtensorMap vmap32,
                                const Args a) {
  constexpr int QMAX = kCols / G;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* sQ = base + kOffQ;
  unsigned char* sK = base + kOffK;
  unsigned char* sV = base + kOffV;
  unsigned char* sP = base + kOffP;
  Smem& S = *reinterpret_cast<Smem*>(base + kOffCtl);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&S.q_full[i], 4);     // one elected arrival per query warp
      mbar_init(&S.q_empty[i], 1);
      mbar_init(&S.s_full[i], 1);
      mbar_init(&S.p_full[i], kSoftmaxWarps);     // one elected arrival per softmax warp
      mbar_init(&S.o_done[i], 1);
      mbar_init(&S.o_free[i], kSoftmaxWarps);
    }
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&S.k_full[s], 1);
      mbar_init(&S.k_empty[s], 1);
      mbar_init(&S.v_full[s], 1);
      mbar_init(&S.v_empty[s], 1);
    }
    S.abort = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&S.tmem_base, kTmemCols);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
    prefetch_tensormap(&kmap32);
    prefetch_tensormap(&vmap32);
  }
  if (warp == 2) {
    const Share share = find_share<QMAX, true>(a, lane);
    if (lane == 0) {
      int page0 = 0;
      if (share.xe > share.xb) {       // the share's first tile: its page, and its codes into L2 ahead of the loads
        const int h = (int)(share.xb - share.row0) / share.r0.nt;
        const int key0 = (int)(share.xb - share.row0 - (long long)h * share.r0.nt) * kKeysPerTile;
        page0 = page_of(a, a.block_tables + (long long)share.bstart * a.W, key0);
        tma_prefetch_3d(&kmap, 0, key0 % a.block_size, page0 * a.Hkv + h);
        tma_prefetch_3d(&vmap, 0, key0 % a.block_size, page0 * a.Hkv + h);
      }
      S.total_tiles = share.T;
      S.active = (int)share.Ge;
      S.x_begin = share.xb;
      S.x_end = share.xe;
      S.row_tile0 = share.row0;
      S.b_start = share.bstart;
      S.r0[0] = share.r0.q_start;
      S.r0[1] = share.r0.ql;
      S.r0[2] = share.r0.L;
      S.r0[3] = share.r0.nt;
      S.page0 = page0;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // an early (programmatic dependent) launch ran the prologue while the preceding kernel finished
  griddep_wait();
  const uint32_t tmem = S.tmem_base;
  volatile int* abort = &S.abort;
  const long long x_begin = S.x_begin, x_end = S.x_end;
  const int ntiles = (int)(x_end - x_begin);
  const bool softmax = warp >= kSoftmaxWarp && warp < kQueryWarp;

  if (!softmax) registers_down<kProducerRegs>();
  if (warp == 0 || warp == 3) {
    // ------------------------------------------------------------------ TMA producers: K with both scales, V
    const bool is_k = warp == 0;
    if (lane == 0 && ntiles > 0) {
      uint64_t* full = is_k ? S.k_full : S.v_full;
      uint64_t* empty = is_k ? S.k_empty : S.v_empty;
      unsigned char* ring = is_k ? sK : sV;
      const CUtensorMap* map = is_k ? &kmap : &vmap;
      const CUtensorMap* map32 = is_k ? &kmap32 : &vmap32;
      const int per_tile = kKeysPerTile / a.group, per_block = a.block_size / a.group;
      const uint32_t scale_bytes = per_tile * 4;
      Walk<QMAX, true> wk;
      wk.start(a, S);
      bool ok = true;
      int g = 0;
      for (; ok && wk.A < x_end; wk.next(a)) {
        const int* table = a.block_tables + (long long)wk.b * a.W;
        const int t1 = wk.t1(x_end);
        for (int t = wk.t0(x_begin); t < t1; ++t, ++g) {
          const int stage = g % kStages;
          const uint32_t use = g / kStages;
          const int key0 = t * kKeysPerTile;
          const int page = g == 0 ? S.page0 : page_of(a, table, key0);
          const int j0 = key0 % a.block_size, ph = page * a.Hkv + wk.h;
          if (g >= kStages && !mbar_wait(&empty[stage], (use - 1) & 1, abort, a.err, kErrTimeoutEmpty)) {
            ok = false;
            break;
          }
          const int subs = t == wk.r.nt - 1 ? (wk.r.L - key0 + kSubKeys - 1) / kSubKeys : kKeysPerTile / kSubKeys;
          unsigned char* dst = ring + stage * kTileBytes;
          mbar_arrive_expect_tx(&full[stage], subs * kSubKeys * kHeadDim + (is_k ? 2 * scale_bytes : 0));
          if (subs == kKeysPerTile / kSubKeys) {
            tma_load_3d(dst, map, 0, j0, ph, &full[stage]);
          } else {
            for (int j = 0; j < subs; ++j)
              tma_load_3d(dst + j * kSubKeys * kHeadDim, map32, 0, j0 + j * kSubKeys, ph, &full[stage]);
          }
          if (is_k) {
            const long long at = (long long)ph * per_block + j0 / kKeysPerTile * per_tile;
            bulk_load(S.scales[g % kScaleStages][0], a.k_scale + at, scale_bytes, &full[stage]);
            bulk_load(S.scales[g % kScaleStages][1], a.v_scale + at, scale_bytes, &full[stage]);
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer: the whole warp, one lane issuing
    if (ntiles > 0) {
      constexpr uint32_t idesc_s = idesc_f8_f32(128, kQParts * kCols, 0, 0, 0, 0);    // e4m3 . e4m3
      constexpr uint32_t idesc_o = idesc_f8_f32(128, kPParts * kCols, 0, 1, 1, 1);    // e4m3 . e5m2
      constexpr unsigned kAll = 0xffffffffu;
      const uint32_t leader = elect_one();
      // descriptors of the first buffers; the others differ in the low word's address (16-byte units)
      const uint64_t kd = smem_desc(sK, 16, 1024, kSwizzle128B), qd = smem_desc(sQ, 16, 1024, kSwizzle128B);
      const uint64_t vd = smem_desc(sV, kTileBytes, 1024, kSwizzle128B), pd = smem_desc(sP, kPPartBytes, 256, kSwizzle32B);
      const uint32_t kd_hi = (uint32_t)(kd >> 32), qd_hi = (uint32_t)(qd >> 32), vd_hi = (uint32_t)(vd >> 32),
                     pd_hi = (uint32_t)(pd >> 32);
      const uint32_t tm = __shfl_sync(kAll, tmem, 0);
      const int count = __shfl_sync(kAll, ntiles, 0);
      PairCursor<QMAX> cs, cp;       // the score MMAs run two pairs ahead of the PV MMAs
      cs.start(a, S);
      cp.start(a, S);
      int sk = 0, sv = 0;            // ring stages of the next K and V tile, and their phases
      uint32_t sk_phase = 0, sv_phase = 0;
      int qn = 0, on = 0;            // the cursors' segment numbers, warp-uniform
      int done_s = 0, done_pv = 0;   // tiles issued
      auto wait = [&](uint64_t* bar, uint32_t phase, int code) -> bool {
        return __all_sync(kAll, mbar_wait(bar, phase, abort, a.err, code));
      };
      auto issue_s = [&](int u) -> bool {        // scores of pair u
        const int qb = qn & 1;
        const bool two = __any_sync(kAll, cs.two());
        if (__any_sync(kAll, cs.first) && !wait(&S.q_full[qb], (qn >> 1) & 1, kErrTimeoutQ)) return false;
        const uint32_t qa = (uint32_t)qd + qb * (kQBytes >> 4);
        for (int i = 0; i < (two ? 2 : 1); ++i) {
          if (!wait(&S.k_full[sk], sk_phase, kErrTimeoutK)) return false;
          tc_fence_after();
          const uint32_t ka = (uint32_t)kd + sk * (kTileBytes >> 4);
          const uint32_t tmem_s = tm + (u & 1) * kTmemSPair + i * kTmemSTile;
#pragma unroll
          for (int kk = 0; kk < kHeadDim / 32; ++kk)
            mma_f8_ss(leader, tmem_s, ka + kk * 2, kd_hi, qa + kk * 2, qd_hi, idesc_s, kk > 0 ? 1u : 0u);
          mma_commit_leader(leader, &S.k_empty[sk]);
          if (++sk == kStages) {
            sk = 0;
            sk_phase ^= 1;
          }
        }
        mma_commit_leader(leader, &S.s_full[u & 1]);
        if (__any_sync(kAll, cs.last())) {
          mma_commit_leader(leader, &S.q_empty[qb]);
          ++qn;
        }
        done_s += two ? 2 : 1;
        cs.advance(a, x_begin, x_end);
        return true;
      };
      auto issue_pv = [&](int u) -> bool {
        const int ob = on & 1;
        const bool two = __any_sync(kAll, cp.two()), fresh = __any_sync(kAll, cp.first);
        if (fresh && on >= 2 && !wait(&S.o_free[ob], ((on - 2) >> 1) & 1, kErrTimeoutO)) return false;
        if (!wait(&S.p_full[u & 1], (u >> 1) & 1, kErrTimeoutP)) return false;
        const uint32_t tmem_o = tm + kTmemO + ob * kTmemOStride;
        for (int i = 0; i < (two ? 2 : 1); ++i) {
          if (!wait(&S.v_full[sv], sv_phase, kErrTimeoutV)) return false;
          tc_fence_after();
          const uint32_t va = (uint32_t)vd + sv * (kTileBytes >> 4), pa = (uint32_t)pd + ((u & 1) * 2 + i) * (kPBytes >> 4);
#pragma unroll
          for (int kk = 0; kk < kKeysPerTile / 32; ++kk)
            mma_f8_ss(leader, tmem_o, va + kk * (32 * kHeadDim >> 4), vd_hi, pa + kk * (32 * kCols >> 4), pd_hi, idesc_o,
                      kk > 0 || i > 0 || !fresh ? 1u : 0u);
          mma_commit_leader(leader, &S.v_empty[sv]);
          if (++sv == kStages) {
            sv = 0;
            sv_phase ^= 1;
          }
        }
        mma_commit_leader(leader, &S.o_done[u & 1]);
        if (__any_sync(kAll, cp.last())) ++on;
        done_pv += two ? 2 : 1;
        cp.advance(a, x_begin, x_end);
        return true;
      };
      // PV of pair u goes out before S of pair u + 2.  The wait for P(u) says that the softmax has read S(u) and the tiles'
      // scales, so S's buffer is free; and as MMAs complete in order, a softmax that sees S(u + 2) knows that PV(u) has
      // read P's.
      bool ok = issue_s(0);
      if (ok && done_s < count) ok = issue_s(1);
      for (int u = 0; ok && done_pv < count; ++u) {
        ok = issue_pv(u);
        if (ok && done_s < count) ok = issue_s(u + 2);
      }
    }
  } else if (warp >= kQueryWarp) {
    // ------------------------------------------------------------------ query parts: 32 columns x 128 dims an item
    // a column's 128 dims belong to four threads, 32 each
    const int tid = threadIdx.x - kQueryWarp * 32, col = tid >> 2, quarter = tid & 3;
    const int p = col / G, gq = col % G;
    if (ntiles > 0) {
      Walk<QMAX, true> wk;
      wk.start(a, S);
      for (int n = 0; wk.A < x_end; wk.next(a), ++n) {
        uint4 raw[4];
        unsigned most = 0;
        const uint4* src = reinterpret_cast<const uint4*>(
            a.q + (long long)(wk.r.q_start + p) * a.q_row_stride + (wk.h * G + gq) * kHeadDim + quarter * 32);
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[i] = p < wk.r.ql ? src[i] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const unsigned lo = w[k] & 0x7fffu, hi = (w[k] >> 16) & 0x7fffu;
            most = max(most, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
          }
        }
        most = __reduce_max_sync(0xffffffffu, most);
        named_barrier(kBarQuery, 128);         // the last item's maxima have been read
        if (lane == 0) S.red_q[warp - kQueryWarp] = most;
        named_barrier(kBarQuery, 128);
        most = max(max(S.red_q[0], S.red_q[1]), max(S.red_q[2], S.red_q[3]));
        // 2^e with every |q| <= 448 * 2^e = 1.75 * 2^(e + 8)
        int e = (int)(most >> 7) - 135 + ((most & 0x7fu) > 0x60u ? 1 : 0);
        e = max(e, -100);
        const float inv = __uint_as_float((unsigned)(127 - e) << 23);
        if (n >= 2 && !mbar_wait(&S.q_empty[n & 1], ((n - 2) >> 1) & 1, abort, a.err, kErrTimeoutEmpty)) break;
        unsigned char* q1 = sQ + (n & 1) * kQBytes + col * 128;
        unsigned char* q2 = q1 + kCols * 128;
#pragma unroll
        for (int i = 0; i < 4; i += 2) {       // 16 dims: one 16-byte chunk of each part
          unsigned b1[8], b2[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint4& r4 = raw[i + k / 4];
            const unsigned w = k % 4 == 0 ? r4.x : k % 4 == 1 ? r4.y : k % 4 == 2 ? r4.z : r4.w;
            float x = __uint_as_float(w << 16) * inv, y = __uint_as_float(w & 0xffff0000u) * inv;
            x += x - x;                        // infinities become NaN (a saturating conversion would hide them)
            y += y - y;
            b1[k] = encode_e4m3x2(x, y);
            const float2 d = decode_e4m3x2(b1[k]);
            b2[k] = encode_e4m3x2((x - d.x) * 16.0f, (y - d.y) * 16.0f);
          }
          const int phys = ((quarter * 2 + i / 2) ^ (col & 7)) * 16;
          *reinterpret_cast<uint4*>(q1 + phys) = make_uint4(b1[0] | b1[1] << 16, b1[2] | b1[3] << 16,
                                                            b1[4] | b1[5] << 16, b1[6] | b1[7] << 16);
          *reinterpret_cast<uint4*>(q2 + phys) = make_uint4(b2[0] | b2[1] << 16, b2[2] | b2[3] << 16,
                                                            b2[4] | b2[5] << 16, b2[6] | b2[7] << 16);
        }
        // read by the softmax before it hands over P of the item's first tile; written again four items on, after that
        if (tid == 0) S.q_scale[n & 3] = __uint_as_float((unsigned)(e + 127) << 23);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.q_full[n & 1]);
      }
    }
    // rows of queries without a key: zeros
    for (int b = blockIdx.x; b < a.R; b += gridDim.x) {
      const RowInfo r = row_info<QMAX, true>(a, b, false);
      if (r.ql <= 0 || r.ql > QMAX || r.L != 0) continue;
      const int chunks = a.H * (kHeadDim / 8);
      for (int i = tid; i < r.ql * chunks; i += 128)
        reinterpret_cast<uint4*>(a.out + (long long)(r.q_start + i / chunks) * a.out_row_stride)[i % chunks] =
            make_uint4(0u, 0u, 0u, 0u);
    }
  } else if (softmax) {
    registers_up<kSoftmaxRegs>();
    // ------------------------------------------------------------------ softmax / correction / epilogue
    const int wg = (warp - kSoftmaxWarp) >> 2;   // column group: columns cb .. cb + 15
    const int cb = wg * kGroupCols, p0 = cb / G; // and its first query position (G divides 16)
    const int w = warp & 3;                      // TMEM lane quadrant
    const int row = (threadIdx.x - kSoftmaxWarp * 32) & 127;   // key within the tile (S^T) / head dim (O^T)
    const int col = cb + (lane & 15);            // the column that lane j (and j + 16) speaks for
    const uint32_t lane_off = static_cast<uint32_t>(w * 32) << 16;
    const int bar_wg = 1 + wg;
    const bool first_thread = threadIdx.x == kSoftmaxWarp * 32;
    const long long T = S.total_tiles, Ge = S.active;
    const int c = blockIdx.x;
    const int my_group = row / a.group;
    Walk<QMAX, true> wk;
    bool ok = ntiles > 0;
    if (ok) wk.start(a, S);
    int g = 0, u = 0;              // tiles and pairs handed over
    for (int n = 0; ok && wk.A < x_end; wk.next(a), ++n) {
      const int L = wk.r.L, ql = wk.r.ql;
      const int t0 = wk.t0(x_begin), t1 = wk.t1(x_end);
      const uint32_t tmem_o = tmem + lane_off + kTmemO + (n & 1) * kTmemOStride + cb;
      const int min_limit = a.causal ? L - ql : L - 1;       // smallest limit among the valid columns
      // A group none of whose columns holds a query only keeps the barriers going: its columns of P and O are never read.
      const bool live = cb < ql * G;
      const long long c_lo = mul_ceil_div(wk.A + 1, Ge, T) - 1, c_hi = mul_ceil_div(wk.A + wk.r.nt, Ge, T) - 1;
      int seen_early = -1;
      if (first_thread && c_lo != c_hi && c == c_lo)
        seen_early = ld_acquire_gpu(a.counters + (long long)wk.b * a.Hkv + wk.h);
      float q_factor = 0.0f;
      // running maxima of t (log2 domain; lane j owns column cb + (j & 15)'s), every thread's copy negated with the bias, and
      // this thread's share of the column sums
      float m_lane = kNegBig, m_neg[kGroupCols], l_part[kGroupCols];
#pragma unroll
      for (int j = 0; j < kGroupCols; ++j) {
        m_neg[j] = -kNegBig;
        l_part[j] = 0.0f;
      }
      for (int t = t0; t < t1; t += 2, ++u) {
        const bool two = t + 1 < t1;
        const int buf = u & 1;
        if (!mbar_wait(&S.s_full[buf], (u >> 1) & 1, abort, a.err, kErrTimeoutS)) { ok = false; break; }
        tc_fence_after();
        if (live) {
          if (t == t0) q_factor = S.q_scale[n & 3] * a.scale_log2;
          // distances of both tiles' t = score + log2 vs from the running maxima (a missing second tile: nothing)
          float d[2][kGroupCols], inv_vs[2];
          {
            uint32_t r[2][16], r2[2][16];
            const uint32_t tmem_s = tmem + lane_off + buf * kTmemSPair + cb;
            tmem_ld_start_2x16(tmem_s, tmem_s + kCols, r[0], r2[0]);
            if (two) tmem_ld_start_2x16(tmem_s + kTmemSTile, tmem_s + kTmemSTile + kCols, r[1], r2[1]);
            float factor[2], log_vs[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int e = (g + i) % kScaleStages;
              const float ks = S.scales[e][0][my_group], vs = fmaxf(S.scales[e][1][my_group], kMinScale);
              factor[i] = ks * q_factor;
              log_vs[i] = __log2f(vs);
              inv_vs[i] = __fdividef(1.0f, vs);
            }
            tmem_ld_wait_2x16(r[0], r2[0]);
            tmem_ld_wait_2x16(r[1], r2[1]);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int j = 0; j < kGroupCols; j += 2) {
                const float2 s2 = fma_x2(make_float2(__uint_as_float(r2[i][j]), __uint_as_float(r2[i][j + 1])),
                                         make_float2(0.0625f, 0.0625f),
                                         make_float2(__uint_as_float(r[i][j]), __uint_as_float(r[i][j + 1])));
                const float2 t2 = fma_x2(s2, make_float2(factor[i], factor[i]), make_float2(log_vs[i], log_vs[i]));
                d[i][j] = t2.x;
                d[i][j + 1] = t2.y;
              }
          }
          if ((t + 2) * kKeysPerTile - 1 > min_limit) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int key = (t + i) * kKeysPerTile + row;
#pragma unroll
              for (int j = 0; j < kGroupCols; ++j) {
                const int p = p0 + j / G;
                const int limit = (a.causal && p < ql) ? L - ql + p : L - 1;
                d[i][j] = key <= limit && (i == 0 || two) ? d[i][j] : -INFINITY;
              }
            }
          } else if (!two) {         // the piece's last tile, its item going on in another CTA
#pragma unroll
            for (int j = 0; j < kGroupCols; ++j) d[1][j] = -INFINITY;
          }
          // ---- does any score of the group pass its column's running maximum by more than 2^8?  Only then (always at an
          // item's first pair) are the pair's column maxima taken: this warp's, then the four warps'
          float over = -INFINITY;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < kGroupCols; ++j) over = fmaxf(over, d[i][j] + m_neg[j]);
          if (named_barrier_or(bar_wg, 128, over > 8.0f + kPBias)) {
            float wmax = -INFINITY;
#pragma unroll
            for (int j = 0; j < kGroupCols; ++j) {
              const float v = warp_max_redux(fmaxf(d[0][j], d[1][j]));
              wmax = lane == j ? v : wmax;
            }
            if (lane < kGroupCols) S.red_max[buf][col][w] = wmax;
            named_barrier(bar_wg, 128);
            const float4 r4 = *reinterpret_cast<const float4*>(S.red_max[buf][col]);
            const float tmax = fmaxf(fmaxf(r4.x, r4.y), fmaxf(r4.z, r4.w));
            const float m_new = tmax > m_lane + 8.0f ? tmax : m_lane;
            const float alpha_lane = ex2_approx(m_lane - m_new);
            m_lane = m_new;
#pragma unroll
            for (int j = 0; j < kGroupCols; ++j) m_neg[j] = kPBias - __shfl_sync(0xffffffffu, m_new, j);
            if (t > t0) {     // O holds this item's earlier tiles: rescale its parts once the last PV has landed
#pragma unroll
              for (int j = 0; j < kGroupCols; ++j) l_part[j] *= __shfl_sync(0xffffffffu, alpha_lane, j);
              if (!mbar_wait(&S.o_done[(u - 1) & 1], ((u - 1) >> 1) & 1, abort, a.err, kErrTimeoutO)) { ok = false; break; }
              tc_fence_after();
#pragma unroll 1
              for (int part = 0; part < kPParts; ++part) {
                float o[kGroupCols];
                tmem_ld_32x32b_x16(tmem_o + part * kCols, o);
#pragma unroll
                for (int j = 0; j < kGroupCols; ++j) o[j] *= __shfl_sync(0xffffffffu, alpha_lane, j);
                tmem_st_32x32b_x16(tmem_o + part * kCols, o);
              }
            }
          }
          // ---- probabilities, column sums, and this group's 16 columns of row `row` of the parts (S(u) seen: PV(u-2) has
          // released the buffer).  An fp16 pattern's high byte is its value cut to e5m2; what is left over, less than a
          // quarter of it, is exact in fp16, and 8 times that stays below 2^15 as p' does.  Two cuts, then the third part to
          // nearest: fp16's 2^-12 and e5m2's last half step off it, 2^-9 of p' or 2^-17 / 64.
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (i == 1 && !two) break;
            __half2 ph[kGroupCols / 2];
#pragma unroll
            for (int j = 0; j < kGroupCols; j += 2) {
              const float2 d2 = add_x2(make_float2(d[i][j], d[i][j + 1]), make_float2(m_neg[j], m_neg[j + 1]));
              const float2 p2 = make_float2(ex2_approx(d2.x), ex2_approx(d2.y));      // masked: 0
              const float2 l2 = fma_x2(p2, make_float2(inv_vs[i], inv_vs[i]), make_float2(l_part[j], l_part[j + 1]));
              l_part[j] = l2.x;
              l_part[j + 1] = l2.y;
              ph[j / 2] = __floats2half2_rn(p2.x, p2.y);
            }
            const __half2 eight = bits_half2(0x48004800u);
            unsigned char* prow = sP + (buf * 2 + i) * kPBytes + row * kCols + (wg ^ ((row >> 2) & 1)) * 16;
#pragma unroll
            for (int part = 0; part < kPParts; ++part) {
              unsigned wd[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                unsigned lo = half2_bits(ph[2 * k]), hi = half2_bits(ph[2 * k + 1]);
                if (part == kPParts - 1) {
                  lo += 0x00800080u;
                  hi += 0x00800080u;
                } else {
                  ph[2 * k] = __hmul2(__hsub2(ph[2 * k], bits_half2(lo & 0xff00ff00u)), eight);
                  ph[2 * k + 1] = __hmul2(__hsub2(ph[2 * k + 1], bits_half2(hi & 0xff00ff00u)), eight);
                }
                wd[k] = __byte_perm(lo, hi, 0x7531);
              }
              *reinterpret_cast<uint4*>(prow + part * kPPartBytes) = make_uint4(wd[0], wd[1], wd[2], wd[3]);
            }
          }
        }
        const int last = two ? 1 : 0;
        // ---- the row's last tile: V rows past the context are zeroed; each group zeroes half of the row
        if ((t + last + 1) * kKeysPerTile > L) {
          const int gl = g + last, stage = gl % kStages;
          if (!mbar_wait(&S.v_full[stage], (gl / kStages) & 1, abort, a.err, kErrTimeoutV)) { ok = false; break; }
          if ((t + last) * kKeysPerTile + row >= L) {
            unsigned char* v0 = sV + stage * kTileBytes + row * kHeadDim + wg * 64;
#pragma unroll
            for (int cc = 0; cc < 4; ++cc) *reinterpret_cast<uint4*>(v0 + cc * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        g += last + 1;
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.p_full[buf]);
      }
      if (!ok) break;
      // ---- item epilogue: column sums over the 128 key threads, O^T out of TMEM
      if (live) {
        const float s = column_reduce16(l_part, lane);
        if (lane < kGroupCols) S.red_sum[col][w] = s;
      }
      named_barrier(bar_wg, 128);
      if (!mbar_wait(&S.o_done[(u - 1) & 1], ((u - 1) >> 1) & 1, abort, a.err, kErrTimeoutO)) break;
      tc_fence_after();
      float o[kGroupCols];
      {
        float o2[kGroupCols], o3[kGroupCols];
        tmem_ld_32x32b_2x16(tmem_o, tmem_o + kCols, o, o2);
        tmem_ld_32x32b_x16(tmem_o + 2 * kCols, o3);
#pragma unroll
        for (int j = 0; j < kGroupCols; ++j) o[j] = fmaf(o3[j], 1.0f / 64.0f, fmaf(o2[j], 0.125f, o[j]));
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.o_free[n & 1]);
      const float4 s4 = *reinterpret_cast<const float4*>(S.red_sum[col]);
      float l_lane = (s4.x + s4.y) + (s4.z + s4.w);
      // ---- a split item: pieces published, the last to arrive merges them in CTA order (as the bf16 kernel)
      const long long A = wk.A;
      if (c_lo != c_hi) {
        int* counter = a.counters + (long long)wk.b * a.Hkv + wk.h;
        if (first_thread) {
          const int need = (int)(c_hi - c_lo);
          S.last_piece = (c == c_lo && (seen_early == need || ld_acquire_gpu(counter) == need)) ? 2 : 0;
        }
        named_barrier(kBarMerge, kSoftmaxThreads);
        const bool own_in_registers = S.last_piece == 2;
        if (!own_in_registers) {
          float* mine = a.partial + (2LL * c + (x_begin < A ? 1 : 0)) * kPartialFloats;
          if (live) {
#pragma unroll
            for (int j = 0; j < kGroupCols; ++j) __stcg(mine + (cb + j) * kHeadDim + row, o[j]);
            if (w == 0 && lane < kGroupCols) {
              __stcg(mine + kCols * kHeadDim + col, m_lane);
              __stcg(mine + kCols * kHeadDim + kCols + col, l_lane);
            }
          }
          __threadfence();
          named_barrier(kBarMerge, kSoftmaxThreads);             // all groups published
          if (first_thread) {
            const int last = atomicAdd(counter, 1) == (int)(c_hi - c_lo);
            if (last) atomicExch(counter, 0);
            S.last_piece = last;
          }
          named_barrier(kBarMerge, kSoftmaxThreads);
          // S.last_piece is next written at the next split item's epilogue, which its writer reaches only after every
          // softmax warp has handed over P for that item's tiles (so after every thread's read here)
          if (!S.last_piece) continue;
        } else if (first_thread) {
          atomicExch(counter, 0);            // every other piece has arrived: nobody else touches it
        }
        __threadfence();
        if (!live) continue;
        // pieces in CTA order, the common maximum first so that the pieces' loads do not wait for one another
        // (only the first piece's CTA can hold an earlier item before it)
        const int c_lo_slot = mul_div(T, c_lo, Ge) < A ? 1 : 0;
        auto piece_of = [&](long long cc) {
          return a.partial + (2 * cc + (cc == c_lo ? c_lo_slot : 0)) * kPartialFloats;
        };
        const float m_own = m_lane, l_own = l_lane;
        float m_acc = own_in_registers ? m_own : kNegBig;
        const long long c_from = c_lo + (own_in_registers ? 1 : 0);
#pragma unroll 4
        for (long long cc = c_from; cc <= c_hi; ++cc) m_acc = fmaxf(m_acc, __ldcg(piece_of(cc) + kCols * kHeadDim + col));
        float l_acc = 0.0f;
        if (own_in_registers) {              // piece c_lo = this CTA's
          const float sb = ex2_approx(m_own - m_acc);
          l_acc = __fmul_rn(l_own, sb);
#pragma unroll
          for (int j = 0; j < kGroupCols; ++j) o[j] = __fmul_rn(o[j], __shfl_sync(0xffffffffu, sb, j));
        } else {
#pragma unroll
          for (int j = 0; j < kGroupCols; ++j) o[j] = 0.0f;
        }
#pragma unroll 2
        for (long long cc = c_from; cc <= c_hi; ++cc) {
          const float* piece = piece_of(cc);
          const float mp = __ldcg(piece + kCols * kHeadDim + col), lp = __ldcg(piece + kCols * kHeadDim + kCols + col);
          float op[kGroupCols];
#pragma unroll
          for (int j = 0; j < kGroupCols; ++j) op[j] = __ldcg(piece + (cb + j) * kHeadDim + row);
          const float sb = ex2_approx(mp - m_acc);
          l_acc = __fmaf_rn(lp, sb, l_acc);
#pragma unroll
          for (int j = 0; j < kGroupCols; ++j) o[j] = __fmaf_rn(op[j], __shfl_sync(0xffffffffu, sb, j), o[j]);
        }
        l_lane = l_acc;
      }
      if (!live) continue;
      const float inv_lane = l_lane > 0.0f ? 1.0f / l_lane : l_lane;      // nothing seen: 0 (and NaN stays)
      __nv_bfloat16* dst = a.out + (long long)(wk.r.q_start + p0) * a.out_row_stride + wk.h * (G * kHeadDim) + row;
#pragma unroll
      for (int j = 0; j < kGroupCols; ++j) {
        const float inv = __shfl_sync(0xffffffffu, inv_lane, j);
        if (p0 + j / G < ql) dst[(j / G) * a.out_row_stride + (j % G) * kHeadDim] = __float2bfloat16_rn(o[j] * inv);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// 3-D map of a code cache: {128 dims, block_size slots, blocks * heads}, 128-byte swizzle, box {128, keys, 1}.
static int make_map(CUtensorMap* map, const void* base, uint64_t block_size, uint64_t block_heads, uint32_t keys) {
  auto fn = encoder();
  if (!fn) return set_error(kCudaError, "cuTensorMapEncodeTiled is unavailable from the driver");
  cuuint64_t dims[3] = {kHeadDim, block_size, block_heads};
  cuuint64_t strides[2] = {kHeadDim, kHeadDim * block_size};
  cuuint32_t box[3] = {kHeadDim, keys, 1};
  cuuint32_t elem[3] = {1, 1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, elem,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(kCudaError, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return kOk;
}

template <int G>
static int launch(const CUtensorMap (&m)[4], const Args& a, int grid, bool early, cudaStream_t stream) {
  if (int st = ensure_dynamic_smem<verify_attention_fp8_kernel<G>>(kSmemBytes)) return st;
  static const int regs = [] {
    cudaFuncAttributes attr;
    return cudaFuncGetAttributes(&attr, verify_attention_fp8_kernel<G>) == cudaSuccess ? attr.numRegs : -1;
  }();
  if (regs < kLaunchRegs)      // the register shares would wait for registers that the block does not have
    return set_error(kCudaError, "attention built with %d registers a thread, %d needed", regs, kLaunchRegs);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 1 : 0;
  SPECDEC_CUDA_TRY(cudaLaunchKernelEx(&cfg, verify_attention_fp8_kernel<G>, m[0], m[1], m[2], m[3], a));
  SPECDEC_LAUNCH_CHECK();
  return kOk;
}

}  // namespace attention_fp8
}  // namespace specdec

using namespace specdec;

extern "C" {

int specdec_paged_attention_fp8(const void* q, long long T, long long q_row_stride, int num_heads, int num_kv_heads,
                                int head_dim, const void* k_cache, const void* v_cache, const float* k_scale,
                                const float* v_scale, long long num_blocks, int block_size, int scale_group,
                                const int* cu_seqlens_q, const int* cu_seqlens_k, const int* context_lens,
                                int q_per_seq, int R, const int* block_tables, int W, int max_seqlen_q,
                                float softmax_scale, int causal, void* out, long long out_row_stride, void* workspace,
                                long long workspace_bytes, int* err, unsigned flags, void* stream) {
  using namespace attention_fp8;
  SPECDEC_CHECK_ARG((flags & ~((unsigned)SPECDEC_ATTN_EARLY_LAUNCH | SPECDEC_ATTN_MAX_CTAS(0xff))) == 0,
                    "unknown flags 0x%x", flags);
  SPECDEC_CHECK_ARG(q && k_cache && v_cache && k_scale && v_scale && block_tables && out && workspace && err,
                    "null pointer argument");
  SPECDEC_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, "workspace must be 256-byte aligned");
  SPECDEC_CHECK_ARG(head_dim == kHeadDim, "head_dim %d: this build implements 128", head_dim);
  SPECDEC_CHECK_ARG(num_kv_heads >= 1 && num_heads >= 1 && num_heads % num_kv_heads == 0,
                    "heads %d not a multiple of kv heads %d", num_heads, num_kv_heads);
  const int G = num_heads / num_kv_heads;
  if (G != 1 && G != 2 && G != 4 && G != 8)
    return set_error(kUnsupported, "GQA group %d: this build packs groups of 1, 2, 4 or 8", G);
  SPECDEC_CHECK_ARG(max_seqlen_q >= 1, "max_seqlen_q must be >= 1");
  if ((long long)max_seqlen_q * G > kCols)
    return set_error(kUnsupported, "%d queries x group %d exceed the %d packed columns", max_seqlen_q, G, kCols);
  SPECDEC_CHECK_ARG(block_size >= 1 && block_size % kKeysPerTile == 0, "block_size %d must be a multiple of %d",
                    block_size, kKeysPerTile);
  SPECDEC_CHECK_ARG(scale_group == 16 || scale_group == 32, "scale_group %d: 16 or 32 slots share a scale", scale_group);
  SPECDEC_CHECK_ARG(R >= 1 && R <= 65535 && W >= 1 && T >= 1 && T <= 0x7fffffffLL, "bad row/table sizes");
  SPECDEC_CHECK_ARG((cu_seqlens_q && cu_seqlens_k) || (context_lens && q_per_seq >= 1),
                    "give cu_seqlens_q/k (varlen) or context_lens and q_per_seq (decode)");
  SPECDEC_CHECK_ARG(cu_seqlens_q || (q_per_seq <= max_seqlen_q && (long long)R * q_per_seq <= T),
                    "decode mode: q_per_seq must fit the batch");
  SPECDEC_CHECK_ARG(num_blocks >= 1 && num_blocks <= 0x7fffffffLL / num_kv_heads, "num_blocks * kv heads must fit 32 bits");
  SPECDEC_CHECK_ARG((long long)W * block_size <= 0x7fffffffLL - kKeysPerTile, "a row's table spans more than 2^31 keys");
  SPECDEC_CHECK_ARG((reinterpret_cast<uintptr_t>(q) & 15) == 0 && q_row_stride % 8 == 0 && out_row_stride % 8 == 0 &&
                        (reinterpret_cast<uintptr_t>(out) & 15) == 0,
                    "q and out rows must be 16-byte aligned");
  SPECDEC_CHECK_ARG(((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
                      reinterpret_cast<uintptr_t>(k_scale) | reinterpret_cast<uintptr_t>(v_scale)) & 15) == 0,
                    "caches and scales must be 16-byte aligned");
  DeviceInfo info;
  if (int st = device_info(&info)) return st;
  const long long need = attention::workspace_bytes(R, num_kv_heads, info.sm_count);
  if (workspace_bytes < need)
    return set_error(kWorkspaceTooSmall, "attention workspace of %lld bytes, %lld needed", workspace_bytes, need);
  CUtensorMap m[4];
  const uint64_t bh = (uint64_t)num_blocks * num_kv_heads;
  for (int i = 0; i < 4; ++i)
    if (int st = make_map(&m[i], i & 1 ? v_cache : k_cache, block_size, bh, i < 2 ? kKeysPerTile : kSubKeys)) return st;
  Args a{};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.q_row_stride = q_row_stride;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.cu_seqlens_q = cu_seqlens_q;
  a.cu_seqlens_k = cu_seqlens_k;
  a.context_lens = context_lens;
  a.q_per_seq = q_per_seq;
  a.R = R;
  a.T = (int)T;
  a.block_tables = block_tables;
  a.W = W;
  a.block_size = block_size;
  a.group = scale_group;
  a.num_blocks = (int)num_blocks;
  a.H = num_heads;
  a.Hkv = num_kv_heads;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  a.causal = causal;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.out_row_stride = out_row_stride;
  a.err = err;
  a.partial = static_cast<float*>(workspace);
  a.counters = reinterpret_cast<int*>(static_cast<unsigned char*>(workspace) + partial_bytes(info.sm_count));
  const long long max_tiles = (long long)R * num_kv_heads * ((long long)W * block_size / kKeysPerTile);
  const int cap = (int)((flags >> SPECDEC_ATTN_CTAS_SHIFT) & 0xffu);
  const int ctas = cap > 0 && cap < info.sm_count ? cap : info.sm_count;
  const int grid = (int)(max_tiles < ctas ? max_tiles : ctas);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool early = (flags & SPECDEC_ATTN_EARLY_LAUNCH) != 0;
  switch (G) {
    case 1: return launch<1>(m, a, grid, early, s);
    case 2: return launch<2>(m, a, grid, early, s);
    case 4: return launch<4>(m, a, grid, early, s);
    default: return launch<8>(m, a, grid, early, s);
  }
}

}  // extern "C"
