// Verify / decode attention over the 8-bit paged cache (e4m3 codes, a scale per group of slots and KV head).
//
// Reference behaviour: Attention.forward, verify and decode branches (nanovllm/layers/attention.py:59-77), over a
// cache whose keys and values are code * scale:
//   o = sum_j softmax_j(softmax_scale * ks_j * (q . k_j)) * vs_j * v_j.
//
// First form: a warp per (token, query head) walks the row's keys with a running maximum and sum, 4 dims a lane.
#include "common.cuh"
#include "specdec_b200.h"

#include <cuda_fp8.h>
#include <math.h>

namespace specdec {
namespace attention_fp8 {

constexpr int kHeadDim = 128;
constexpr int kCols = 32;
constexpr int kKeysPerTile = 128;

struct Args {
  const __nv_bfloat16* q;
  long long q_row_stride;
  const unsigned char *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  const int *cu_seqlens_q, *cu_seqlens_k, *context_lens;
  int q_per_seq, R, max_q;
  const int* block_tables;
  int W, block_size, group;
  long long num_blocks;
  int H, Hkv;
  float scale;
  int causal;
  __nv_bfloat16* out;
  long long out_row_stride;
  int* err;
};

__device__ __forceinline__ float4 decode4(unsigned c) {
  const float2 lo = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c & 0xffffu), __NV_E4M3)));
  const float2 hi = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c >> 16), __NV_E4M3)));
  return make_float4(lo.x, lo.y, hi.x, hi.y);
}

__global__ void __launch_bounds__(256) simple_kernel(const Args a) {
  const int b = blockIdx.x, lane = threadIdx.x & 31;
  int q0, ql, L;
  if (a.cu_seqlens_q) {
    q0 = a.cu_seqlens_q[b];
    ql = a.cu_seqlens_q[b + 1] - q0;
    L = a.cu_seqlens_k[b + 1] - a.cu_seqlens_k[b];
  } else {
    q0 = b * a.q_per_seq;
    ql = a.q_per_seq;
    L = a.context_lens[b];
  }
  if (ql <= 0) return;
  if (ql > a.max_q || L < 0 || L > a.W * a.block_size) {
    if (threadIdx.x == 0) atomicCAS(a.err, 0, 2);
    return;
  }
  for (int u = blockIdx.y * 8 + (threadIdx.x >> 5); u < ql * a.H; u += gridDim.y * 8) {
    const int p = u / a.H, head = u % a.H, h = head / (a.H / a.Hkv);
    const uint2 qq = *reinterpret_cast<const uint2*>(a.q + (long long)(q0 + p) * a.q_row_stride + head * kHeadDim + lane * 4);
    const float qf[4] = {__uint_as_float(qq.x << 16), __uint_as_float(qq.x & 0xffff0000u), __uint_as_float(qq.y << 16),
                         __uint_as_float(qq.y & 0xffff0000u)};
    const int limit = a.causal ? min(L, L - ql + p + 1) : L;
    float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int key = 0; key < limit; ++key) {
      const long long block = a.block_tables[(long long)b * a.W + key / a.block_size];
      if (block < 0 || block >= a.num_blocks) {
        if (lane == 0) atomicCAS(a.err, 0, 5);
        continue;
      }
      const long long bh = block * a.Hkv + h;
      const int j = key % a.block_size;
      const long long at = (bh * a.block_size + j) * kHeadDim + lane * 4;
      const long long sat = bh * (a.block_size / a.group) + j / a.group;
      const float4 k = decode4(*reinterpret_cast<const unsigned*>(a.k_cache + at));
      const float4 v = decode4(*reinterpret_cast<const unsigned*>(a.v_cache + at));
      const float s = warp_sum_f32(qf[0] * k.x + qf[1] * k.y + qf[2] * k.z + qf[3] * k.w) * a.k_scale[sat] * a.scale;
      const float vs = a.v_scale[sat], mn = fmaxf(m, s), c = expf(m - mn), pr = expf(s - mn);
      m = mn;
      l = l * c + pr;
      o[0] = o[0] * c + pr * vs * v.x;
      o[1] = o[1] * c + pr * vs * v.y;
      o[2] = o[2] * c + pr * vs * v.z;
      o[3] = o[3] * c + pr * vs * v.w;
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    __nv_bfloat162* dst =
        reinterpret_cast<__nv_bfloat162*>(a.out + (long long)(q0 + p) * a.out_row_stride + head * kHeadDim + lane * 4);
    dst[0] = __floats2bfloat162_rn(o[0] * inv, o[1] * inv);
    dst[1] = __floats2bfloat162_rn(o[2] * inv, o[3] * inv);
  }
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
  SPECDEC_CHECK_ARG(R >= 1 && R <= 65535 && W >= 1 && T >= 1, "bad row/table sizes");
  SPECDEC_CHECK_ARG((cu_seqlens_q && cu_seqlens_k) || (context_lens && q_per_seq >= 1),
                    "give cu_seqlens_q/k (varlen) or context_lens and q_per_seq (decode)");
  SPECDEC_CHECK_ARG(cu_seqlens_q || (q_per_seq <= max_seqlen_q && (long long)R * q_per_seq <= T),
                    "decode mode: q_per_seq must fit the batch");
  SPECDEC_CHECK_ARG(num_blocks >= 1 && num_blocks <= 0x7fffffffLL / num_kv_heads, "num_blocks * kv heads must fit 32 bits");
  SPECDEC_CHECK_ARG((long long)W * block_size <= 0x7fffffffLL, "a row's table spans more than 2^31 keys");
  SPECDEC_CHECK_ARG((reinterpret_cast<uintptr_t>(q) & 15) == 0 && q_row_stride % 8 == 0 && out_row_stride % 8 == 0 &&
                        (reinterpret_cast<uintptr_t>(out) & 15) == 0,
                    "q and out rows must be 16-byte aligned");
  SPECDEC_CHECK_ARG(((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
                      reinterpret_cast<uintptr_t>(k_scale) | reinterpret_cast<uintptr_t>(v_scale)) & 15) == 0,
                    "caches and scales must be 16-byte aligned");
  Args a{static_cast<const __nv_bfloat16*>(q), q_row_stride, static_cast<const unsigned char*>(k_cache),
         static_cast<const unsigned char*>(v_cache), k_scale, v_scale, cu_seqlens_q, cu_seqlens_k, context_lens,
         q_per_seq, R, max_seqlen_q, block_tables, W, block_size, scale_group, num_blocks, num_heads, num_kv_heads,
         softmax_scale, causal, static_cast<__nv_bfloat16*>(out), out_row_stride, err};
  const int warps = max_seqlen_q * num_heads;
  dim3 grid((unsigned)R, (unsigned)((warps + 7) / 8));
  simple_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(a);
  SPECDEC_LAUNCH_CHECK();
  return kOk;
}

}  // extern "C"
