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
// One launch, no atomics on global memory, any order of slots: a token is its group's leader when no earlier token
// of the call has a slot there; the leader's CTA scans the call's slots for the group's members (4 bytes a token,
// from L1 / L2) and does the whole group, so each group and its scales are written by one CTA.  A CTA takes a run of
// consecutive tokens, about one group's worth in a prompt.
#include "common.cuh"

#include <cuda_fp8.h>

namespace specdec {
namespace kv_fp8 {

constexpr int kHeadDim = 128;
constexpr int kThreads = 256;
constexpr int kMinExponent = -100;
constexpr int kMaxTokens = 16384;      // each leader scans the call's slots: bounds that scan

struct StoreArgs {
  const __nv_bfloat16* x[2];      // K rows, V rows [N][Hkv][128]
  long long row_stride[2];
  unsigned char* cache[2];        // [blocks][Hkv][block_size][128] e4m3
  float* scale[2];                // [blocks][Hkv][block_size / group]
  const int* slots;               // [N]
  int N, chunk, Hkv, block_size;
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

template <int GROUP>
__global__ void __launch_bounds__(kThreads) store_fp8_kernel(const StoreArgs a) {
  __shared__ int winner[GROUP];    // the group's members: the last token of each slot, or -1
  __shared__ int earlier;          // a token before this one has a slot of the group
  griddep_launch_dependents();
  griddep_wait();                  // may be launched as a dependent of the kernel that wrote its input
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t_begin = blockIdx.x * a.chunk, t_end = min(a.N, t_begin + a.chunk);
  for (int t = t_begin; t < t_end; ++t) {             // uniform over the CTA
    const int slot = a.slots[t];
    if (slot < 0) continue;
    if (slot >= a.num_slots) {
      if (threadIdx.x == 0) atomicCAS(a.err, 0, 3);
      continue;
    }
    const int g0 = slot / GROUP * GROUP;              // the group's first slot
    if (t > 0 && (unsigned)(a.slots[t - 1] - g0) < (unsigned)GROUP) continue;
    __syncthreads();
    if (threadIdx.x < GROUP) winner[threadIdx.x] = -1;
    if (threadIdx.x == 0) earlier = 0;
    __syncthreads();
#pragma unroll 4
    for (int i = threadIdx.x; i < a.N; i += kThreads) {
      const unsigned o = (unsigned)(a.slots[i] - g0);
      if (o < (unsigned)GROUP) {
        atomicMax(&winner[o], i);
        if (i < t) earlier = 1;
      }
    }
    __syncthreads();
    if (earlier) continue;
    const bool started = winner[0] >= 0;
    const int block = g0 / a.block_size, j0 = g0 % a.block_size;
    for (int u = warp; u < 2 * a.Hkv; u += kThreads / 32) {
      const int side = u >= a.Hkv, h = u - side * a.Hkv;
      const __nv_bfloat16* x = a.x[side] + h * kHeadDim + lane * 4;
      uint2 v[GROUP];
      unsigned most = 0;
#pragma unroll
      for (int o = 0; o < GROUP; ++o) {
        const int w = winner[o];
        v[o] = w >= 0 ? *reinterpret_cast<const uint2*>(x + w * a.row_stride[side]) : make_uint2(0u, 0u);
      }
#pragma unroll
      for (int o = 0; o < GROUP; ++o) most = max(most, max(finite_magnitude(v[o].x), finite_magnitude(v[o].y)));
      most = __reduce_max_sync(0xffffffffu, most);
      const long long head = (long long)block * a.Hkv + h;
      float* scale = a.scale[side] + head * (a.block_size / GROUP) + j0 / GROUP;
      const float old = *scale, wanted = scale_for(most);
      const float now = started ? wanted : fmaxf(old, wanted);
      const float inv = 1.0f / now;
      const bool rescale = !started && now > old;
      const float ratio = old * inv;
      unsigned* row = reinterpret_cast<unsigned*>(a.cache[side] + (head * a.block_size + j0) * kHeadDim) + lane;
#pragma unroll
      for (int o = 0; o < GROUP; ++o) {
        unsigned* p = row + o * (kHeadDim / 4);
        if (winner[o] >= 0) {
          *p = encode4(__uint_as_float(v[o].x << 16) * inv, __uint_as_float(v[o].x & 0xffff0000u) * inv,
                       __uint_as_float(v[o].y << 16) * inv, __uint_as_float(v[o].y & 0xffff0000u) * inv);
        } else if (rescale) {
          const unsigned c = *p;
          const float2 lo = decode2(c), hi = decode2(c >> 16);
          *p = encode4(lo.x * ratio, lo.y * ratio, hi.x * ratio, hi.y * ratio);
        }
      }
      __syncwarp();
      if (lane == 0 && now != old) *scale = now;
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
  a.x[0] = static_cast<const __nv_bfloat16*>(key);
  a.x[1] = static_cast<const __nv_bfloat16*>(value);
  a.row_stride[0] = key_row_stride;
  a.row_stride[1] = value_row_stride;
  a.cache[0] = static_cast<unsigned char*>(k_cache);
  a.cache[1] = static_cast<unsigned char*>(v_cache);
  a.scale[0] = k_scale;
  a.scale[1] = v_scale;
  a.slots = slot_mapping;
  a.N = (int)N;
  a.Hkv = num_kv_heads;
  a.block_size = block_size;
  a.num_slots = num_blocks * block_size;
  a.err = err;
  const int most = 8 * info.sm_count;
  a.chunk = (int)((N + most - 1) / most);
  const dim3 grid((unsigned)((N + a.chunk - 1) / a.chunk));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (scale_group == 16)
    SPECDEC_CUDA_TRY(launch_dependent(store_fp8_kernel<16>, grid, dim3(kThreads), s, a));
  else
    SPECDEC_CUDA_TRY(launch_dependent(store_fp8_kernel<32>, grid, dim3(kThreads), s, a));
  SPECDEC_LAUNCH_CHECK();
  return kOk;
}

}  // extern "C"
