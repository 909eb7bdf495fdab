// The K/V store into an 8-bit paged cache: e4m3 codes with one power-of-two scale per (group of slots, KV head).
//
// Beside store_kvcache (nanovllm/layers/attention.py:10-40), whose slot mapping it takes; the reference's cache is
// bf16 only.  Cache [blocks, Hkv, block_size, 128] e4m3, scales [blocks, Hkv, block_size / group] fp32: the elements
// stand for code * scale.
//
// Mathematics.  For a group and head let a be the largest finite |x| of the tokens this call stores there, and
// e = max(-100, smallest e with a <= 448 * 2^e) (448: e4m3's largest).  A power of two costs a floating-point code
// nothing: the mantissa's 3 bits are the same at any scale, only the bottom of the range moves by less than one
// bit, and x / 2^e, the products of the attention and every requantisation but into subnormals are exact.
//   - the call writes the group's first slot: the group starts, scale = 2^e;
//   - otherwise scale' = max(scale, 2^e), and where that rises the group's other slots become
//     e4m3(code * scale / scale').
// x is stored as e4m3(x / scale), round to nearest even (half a step: 2^-4 of the value), infinities as +-448 * scale,
// NaN as NaN.  A slot given twice holds its last token.
//
// One launch, no atomics on global memory, any order of slots: a token leads its group when no earlier token of the call
// has a slot there; the leader's CTA looks over the call's slots (4 bytes a token, from L1 / L2) for the group's members and
// does the whole group, so each group and its scales are written by one CTA.  A CTA takes some consecutive tokens, and one
// of K and V (blockIdx.y); a warp takes a head's rows of a group into registers, 16 loads in flight.
// Measured (8 KV heads, groups of 16): 16,000 tokens of four prompts 26 us, 98.5 MB at 3.8 TB/s (70 MB of them cross to DRAM
// inside the launch: the codes stay in L2): 6 us of it the look over the slots, then bound by instructions fetched and issued
// for the rows (prefetching the rows into L2 during the look 27.6 us).  Groups of 32 take 26 us too.  A warp keeps to one head
// of eight, so fewer heads leave warps idle: 4, 2 and 1 heads 20, 19 and 17 us (groups of 32: 19, 16 and 14), where the bytes
// are worth 7.6, 3.8 and 1.9.  512 verified tokens of 64 rows take 6.6 us and one token 3.4 us, bound by the launch and the dependent reads
// (slot, members, rows, and the old codes where a scale rises).
#include "common.cuh"
#include "sm100.cuh"

#include <cuda_fp8.h>

namespace specdec {
namespace kv_fp8 {

constexpr int kHeadDim = 128;
constexpr int kSideThreads = 256;       // of one side (K or V): a warp for each of 8 KV heads
constexpr int kMaxChunk = 128;          // tokens of a CTA
constexpr int kMinExponent = -100;
constexpr int kMaxTokens = 16384;      // each leader scans the call's slots: bounds that scan

struct StoreArgs {
  struct Side {
    const __nv_bfloat16* x;       // rows [N][Hkv][128]
    long long row_stride;
    unsigned char* cache;         // [blocks][Hkv][block_size][128] e4m3
    float* scale;                 // [blocks][Hkv][block_size / group]
  } k, v;
  const int* slots;               // [N]
  int N, N4, chunk, Hkv, block_size;   // N4: whole 16-byte quads of slots (0: the mapping is not 16-byte aligned)
  long long num_slots;
  int* err;
};

// Largest finite magnitude of two packed bf16, as bf16 bits (non-finite: 0).
__device__ __forceinline__ unsigned finite_magnitude(unsigned pair) {
  unsigned lo = pair & 0x7fffu, hi = (pair >> 16) & 0x7fffu;
  lo = lo < 0x7f80u ? lo : 0u;
  hi = hi < 0x7f80u ? hi : 0u;
  return lo > hi ? lo : hi;
}

// 2^e for the largest magnitude's bf16 bits: 448 = 1.75 * 2^8.
__device__ __forceinline__ float scale_for(unsigned bits) {
  int e = (int)(bits >> 7) - 127 - 8 + ((bits & 0x7fu) > 0x60u ? 1 : 0);
  if (bits == 0 || e < kMinExponent) e = kMinExponent;
  return __uint_as_float((unsigned)(e + 127) << 23);
}

__device__ __forceinline__ unsigned encode4(float a, float b, float c, float d) {
  const unsigned lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const unsigned hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ __forceinline__ float2 decode2(unsigned pair) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(pair & 0xffffu), __NV_E4M3);
  return __half22float2(__half2(h));
}

// kWide: K and V in one CTA of two sides' threads, many tokens a CTA; else blockIdx.y is the side.
template <int GROUP, bool kWide>
__global__ void __launch_bounds__(kWide ? 2 * kSideThreads : kSideThreads, kWide ? 1 : GROUP == 16 ? 4 : 2)
    store_fp8_kernel(const StoreArgs a) {
  constexpr int kThreads = kWide ? 2 * kSideThreads : kSideThreads;
  // The chunk's groups: the first slot of each, the token that leads it, its members (the last token of each slot, or -1)
  // and whether an earlier token of the call has a slot of it (another CTA's then, or an earlier entry's).
  __shared__ int first_slot[kMaxChunk], leader[kMaxChunk], winner[kMaxChunk][GROUP];
  __shared__ unsigned char earlier[kMaxChunk];
  __shared__ unsigned filter[32];
  __shared__ int count;
  griddep_wait();                  // may be launched as a dependent of the kernel that wrote its input
  griddep_launch_dependents();     // after it: what comes next may read what the kernels before this one wrote
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const StoreArgs::Side side = (kWide ? warp >= kSideThreads / 32 : blockIdx.y) ? a.v : a.k;
  const int t_begin = blockIdx.x * a.chunk, t_end = min(a.N, t_begin + a.chunk);
  if (threadIdx.x == 0) count = 0;
  if (threadIdx.x < 32) filter[threadIdx.x] = 0;
  __syncthreads();
  for (int t = t_begin + threadIdx.x; t < t_end; t += kThreads) {
    const int slot = a.slots[t], before = t > 0 ? a.slots[t - 1] : -1;
    if (slot < 0) continue;
    if (slot >= a.num_slots) {
      atomicCAS(a.err, 0, 3);
      continue;
    }
    const int g0 = slot / GROUP * GROUP;
    if ((unsigned)(before - g0) < (unsigned)GROUP) continue;       // not a run's first token
    const int l = atomicAdd(&count, 1);
    first_slot[l] = g0;
    leader[l] = t;
    earlier[l] = 0;
  }
  __syncthreads();
  const int groups = count;
  if (groups == 0) return;
  for (int i = threadIdx.x; i < groups * GROUP; i += kThreads) winner[i / GROUP][i % GROUP] = -1;
  // every slot of the call against the chunk's groups; a bit for each group number modulo 1024 turns nearly all others away
  for (int l = threadIdx.x; l < groups; l += kThreads) {
    const unsigned g = (unsigned)first_slot[l] / GROUP;
    atomicOr(&filter[g / 32 % 32], 1u << (g % 32));
  }
  __syncthreads();
  auto member = [&](int slot, int i) {
    const unsigned g = (unsigned)slot / GROUP;
    if (!(filter[g / 32 % 32] >> (g % 32) & 1)) return;
    for (int l = 0; l < groups; ++l) {
      const unsigned o = (unsigned)(slot - first_slot[l]);
      if (o < (unsigned)GROUP) {
        atomicMax(&winner[l][o], i);
        if (i < leader[l]) earlier[l] = 1;
      }
    }
  };
  constexpr int kAhead = 4;
  for (int i0 = threadIdx.x; i0 < a.N4; i0 += kAhead * kThreads) {
    int4 four[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) four[u] = __ldg(reinterpret_cast<const int4*>(a.slots) + min(i0 + u * kThreads, a.N4 - 1));
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u * kThreads;
      if (i >= a.N4) break;
      member(four[u].x, 4 * i);
      member(four[u].y, 4 * i + 1);
      member(four[u].z, 4 * i + 2);
      member(four[u].w, 4 * i + 3);
    }
  }
  for (int i = 4 * a.N4 + threadIdx.x; i < a.N; i += kThreads) member(a.slots[i], i);
  __syncthreads();
  // A warp's units: its heads of each group.  fetch issues a unit's loads, finish turns them into codes.
  constexpr int kHeadWarps = kSideThreads / 32;
  const int h0 = warp % kHeadWarps;
  auto first_group = [&](int l) {
    while (l < groups && earlier[l]) ++l;
    return l;
  };
  auto fetch = [&](int l, int h, uint2 (&v)[GROUP], float& old) {
    const int mine = lane < GROUP ? winner[l][lane] : -1;
    const int source = mine >= 0 ? mine : leader[l];      // the row read for a slot that the call does not write: any of its own
    const int g0 = first_slot[l];
    old = side.scale[((long long)(g0 / a.block_size) * a.Hkv + h) * (a.block_size / GROUP) + g0 % a.block_size / GROUP];
    const __nv_bfloat16* x = side.x + h * kHeadDim + lane * 4;
#pragma unroll
    for (int o = 0; o < GROUP; ++o)          // unconditional, so that all are in flight at once: a branch would serialise them
      v[o] = *reinterpret_cast<const uint2*>(x + __shfl_sync(0xffffffffu, source, o) * side.row_stride);
  };
  auto finish = [&](int l, int h, uint2 (&v)[GROUP], float old) {
    const unsigned members = __ballot_sync(0xffffffffu, lane < GROUP && winner[l][lane % GROUP] >= 0);
    const bool started = members & 1;
    const int g0 = first_slot[l], j0 = g0 % a.block_size;
    const long long head = (long long)(g0 / a.block_size) * a.Hkv + h;
    constexpr unsigned kAllSlots = GROUP == 32 ? 0xffffffffu : (1u << (GROUP % 32)) - 1u;
    if (members != kAllSlots) {
#pragma unroll
      for (int o = 0; o < GROUP; ++o)
        if (!(members >> o & 1)) v[o] = make_uint2(0u, 0u);
    }
    // the largest magnitude, in packed pairs (the maximum drops NaN); an infinity has it taken again without them
    __nv_bfloat162 most2 = as_h2<__nv_bfloat162>(0u);
#pragma unroll
    for (int o = 0; o < GROUP; ++o)
      most2 = __hmax2(most2, __hmax2(as_h2<__nv_bfloat162>(v[o].x & 0x7fff7fffu), as_h2<__nv_bfloat162>(v[o].y & 0x7fff7fffu)));
    unsigned most = max(__bfloat16_as_ushort(__low2bfloat16(most2)), __bfloat16_as_ushort(__high2bfloat16(most2)));
    most = __reduce_max_sync(0xffffffffu, most);
    if (most >= 0x7f80u) {
      most = 0;
#pragma unroll
      for (int o = 0; o < GROUP; ++o) most = max(most, max(finite_magnitude(v[o].x), finite_magnitude(v[o].y)));
      most = __reduce_max_sync(0xffffffffu, most);
    }
    const float wanted = scale_for(most);
    const float now = started ? wanted : fmaxf(old, wanted);
    const float inv = 1.0f / now;
    const bool rescale = !started && now > old;
    const float ratio = old * inv;
    unsigned* row = reinterpret_cast<unsigned*>(side.cache + (head * a.block_size + j0) * kHeadDim) + lane;
    const float2 k2 = make_float2(inv, inv);
    auto code = [&](uint2 r) {
      const float2 lo = sm100::mul_x2(make_float2(__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u)), k2);
      const float2 hi = sm100::mul_x2(make_float2(__uint_as_float(r.y << 16), __uint_as_float(r.y & 0xffff0000u)), k2);
      return encode4(lo.x, lo.y, hi.x, hi.y);
    };
#pragma unroll
    for (int o = 0; o < GROUP; ++o) {           // predicated stores: no branches between the rows
      const unsigned c = code(v[o]);
      if (members >> o & 1) row[o * (kHeadDim / 4)] = c;
    }
    if (rescale)
      for (unsigned rest = kAllSlots & ~members; rest; rest &= rest - 1) {
        unsigned* p = row + (__ffs(rest) - 1) * (kHeadDim / 4);
        const unsigned c = *p;
        const float2 lo = decode2(c), hi = decode2(c >> 16);
        *p = encode4(lo.x * ratio, lo.y * ratio, hi.x * ratio, hi.y * ratio);
      }
    __syncwarp();
    if (lane == 0 && now != old) side.scale[head * (a.block_size / GROUP) + j0 / GROUP] = now;
  };
  uint2 v[GROUP];
  float old;
  if constexpr (kWide && GROUP == 16) {       // the next unit's loads pass under this one's arithmetic
    uint2 v2[GROUP];
    float old2;
    auto next = [&](int& l, int& h) {
      h += kHeadWarps;
      if (h >= a.Hkv) {
        h = h0;
        l = first_group(l + 1);
      }
    };
    int l = first_group(0), h = h0;
    if (h0 >= a.Hkv || l >= groups) return;
    fetch(l, h, v, old);
    for (;;) {
      int l2 = l, h2 = h;
      next(l2, h2);
      if (l2 < groups) fetch(l2, h2, v2, old2);
      finish(l, h, v, old);
      if (l2 >= groups) break;
      l = l2;
      h = h2;
      next(l, h);
      if (l < groups) fetch(l, h, v, old);
      finish(l2, h2, v2, old2);
      if (l >= groups) break;
    }
  } else {
    for (int l = first_group(0); l < groups; l = first_group(l + 1))
      for (int h = h0; h < a.Hkv; h += kHeadWarps) {
        fetch(l, h, v, old);
        finish(l, h, v, old);
      }
  }
}

}  // namespace kv_fp8
}  // namespace specdec

using namespace specdec;

extern "C" {

int specdec_store_kvcache_fp8(const void* key, long long key_row_stride, const void* value,
                              long long value_row_stride, void* k_cache, void* v_cache, float* k_scale,
                              float* v_scale, const int* slot_mapping, long long N, int num_kv_heads, int head_dim,
                              long long num_blocks, int block_size, int scale_group, int* err, void* stream) {
  using namespace kv_fp8;
  SPECDEC_CHECK_ARG(N >= 0 && num_kv_heads >= 1 && num_blocks >= 1 && block_size >= 1, "bad sizes");
  SPECDEC_CHECK_ARG(N == 0 || (key && value && slot_mapping), "null pointer argument");
  SPECDEC_CHECK_ARG(k_cache && v_cache && k_scale && v_scale && err, "null pointer argument");
  SPECDEC_CHECK_ARG(head_dim == kHeadDim, "head_dim %d: this build implements 128", head_dim);
  SPECDEC_CHECK_ARG(scale_group == 16 || scale_group == 32, "scale_group %d: 16 or 32 slots share a scale", scale_group);
  SPECDEC_CHECK_ARG(block_size % scale_group == 0, "block_size %d is not a multiple of scale_group %d", block_size,
                    scale_group);
  SPECDEC_CHECK_ARG(num_blocks <= 0x7fffffffLL / block_size, "the cache's slots must fit 32 bits");
  SPECDEC_CHECK_ARG(N <= kMaxTokens, "%lld tokens: a call stores at most %d", N, kMaxTokens);
  SPECDEC_CHECK_ARG(key_row_stride % 4 == 0 && value_row_stride % 4 == 0, "rows must be 8-byte multiples");
  SPECDEC_CHECK_ARG(((reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value)) & 7) == 0 &&
                        ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15) == 0 &&
                        ((reinterpret_cast<uintptr_t>(k_scale) | reinterpret_cast<uintptr_t>(v_scale)) & 3) == 0,
                    "keys and values must be 8-byte aligned, caches 16-byte, scales 4-byte");
  if (N == 0) return kOk;
  DeviceInfo info;
  if (int st = device_info(&info)) return st;
  StoreArgs a{};
  a.k = {static_cast<const __nv_bfloat16*>(key), key_row_stride, static_cast<unsigned char*>(k_cache), k_scale};
  a.v = {static_cast<const __nv_bfloat16*>(value), value_row_stride, static_cast<unsigned char*>(v_cache), v_scale};
  a.slots = slot_mapping;
  a.N = (int)N;
  a.N4 = (reinterpret_cast<uintptr_t>(slot_mapping) & 15) == 0 ? (int)(N / 4) : 0;
  a.Hkv = num_kv_heads;
  a.block_size = block_size;
  a.num_slots = num_blocks * block_size;
  a.err = err;
  // Tokens a CTA: one while the GPU holds that many CTAs at once (each token of a decode is a group of its own).  More of
  // them come from a prompt: a CTA an SM, which looks over the call's slots once for all its groups (the looks' total grows
  // with the CTAs) and loads one group's rows while it converts another's.  Narrow against wide: 512 tokens in rows of 8
  // 6.6 and 7.7 us, 1024 in rows of 8 9.1 and 9.9 us; a prompt's 1184 tokens 8.0 and 5.2 us, 2368 12.3 and 5.7 us, 9472
  // 43 and 18 us.  (A run gains from 400 tokens on, rows of a few tokens up to 1184 do not.)
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = N > 8 * info.sm_count;
  a.chunk = wide ? (int)((N + info.sm_count - 1) / info.sm_count) : 1;
  if (a.chunk > kMaxChunk) a.chunk = kMaxChunk;
  const unsigned ctas = (unsigned)((N + a.chunk - 1) / a.chunk);
  const dim3 grid(ctas, wide ? 1 : 2), block(wide ? 2 * kSideThreads : kSideThreads);
  if (wide)
    SPECDEC_CUDA_TRY(scale_group == 16 ? launch_dependent(store_fp8_kernel<16, true>, grid, block, s, a)
                                       : launch_dependent(store_fp8_kernel<32, true>, grid, block, s, a));
  else
    SPECDEC_CUDA_TRY(scale_group == 16 ? launch_dependent(store_fp8_kernel<16, false>, grid, block, s, a)
                                       : launch_dependent(store_fp8_kernel<32, false>, grid, block, s, a));
  SPECDEC_LAUNCH_CHECK();
  return kOk;
}

}  // extern "C"
