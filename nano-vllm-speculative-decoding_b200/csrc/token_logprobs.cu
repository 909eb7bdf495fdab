// Log probabilities of given tokens, with each row's entropy and its most likely tokens, from [T, V] logits.
//
// Beside probs_from_logits (nanovllm/layers/spec_sampler.py:65-69), which writes all T * V probabilities; a server that
// answers with log probabilities needs a few numbers a row.  With x = logit / temperature, m = max x:
//   S = sum e^(x - m),  log p_t = x_t - m - log S,  H = log S - (sum (x - m) e^(x - m)) / S   (both terms >= 0).
// The alternatives are the num_top largest logits (ties to the lowest index, NaN above all) with their log p.
//
// What bounds it: HBM for the logits, read once, with the exponentials close behind (T * V of them at 16 a clock and SM:
// 0.74 of the read's time for bf16).
// C CTAs take a row, each a contiguous part of it.  A thread keeps a running maximum and, relative to it, S and
// sum (x - m) e^(x - m) in fp32: nothing of the row is kept.  For the alternatives, the CTA's 64 groups of four threads
// tell their maxima: those are 64 elements of its part, so their num_top-th largest is at most the part's, and only the
// threads whose own maximum reaches it read their elements again (from L2): some 24 candidates for 20 alternatives
// where no value is shared by many.  Where ties bring more than the list holds, the part's alternatives are found one by one,
// a pass each.  So does a row that a mask leaves fewer tokens than alternatives in some part, or has in fewer than num_top
// groups: its bound is the mask's value.  With 5 tokens of 151,936 left and 20 alternatives, 8 rows take 59 us, 64 rows 370 and
// 512 rows 2440 (unmasked 14, 18 and 46); with 1000 left 16, 28 and 92 behind -inf (the threads that saw nothing else look
// again) and 14, 18 and 46 behind the type's lowest value.
// The CTA that finishes a row last (a ticket that wraps itself; nobody waits) merges the parts in their order.  Clusters
// with distributed shared memory in place of the tickets took 137 us where this takes 44.5 us (512 rows): their barriers
// kept every CTA of a row until its slowest.
// Measured at 151,936 tokens: 512 bf16 rows (480 of them asked for) with 20 alternatives 44.5 to 47 us (146 MB at 3.2 TB/s),
// 8 rows with 5 10 to 11.5 us; 288 fp32 rows of 50,257 tokens without alternatives 14 to 15 us (3.7 TB/s).  Between the floor
// and these: a row's chain of bound, second reads, ranking and merge, some 6 us, which only other CTAs' rows cover, and 480
// live rows on 148 SMs being 3 or 4 each (1.23 times an equal share).
#include "common.cuh"
#include "sm100.cuh"

#include <float.h>
#include <math.h>

namespace specdec {
namespace logprobs {

constexpr int kThreads = 256;
constexpr int kMaxTop = 32;
constexpr int kGroups = 64;          // groups of four threads
constexpr int kMaxParts = 32;        // CTAs a row
constexpr int kCandidates = 1024;    // holds every element of a part that fills fewer than kMaxTop groups
constexpr int kErrToken = 8;
constexpr int kSteps = 16, kMaxHits = 1024;      // a thread's steps are told apart modulo 16
constexpr int kUnroll = 5;           // 16-byte vectors a thread has in flight

// Ranks logits: larger first, the two zeros equal, NaN above all (but below the all-ones sentinel), ties to the lower index.
__device__ __forceinline__ unsigned rank_high(float f) {
  return f != f ? 0xfffffffeu : ordered_key(f == 0.0f ? 0.0f : f);
}
__device__ __forceinline__ unsigned long long rank_key(float f, unsigned index) {
  return (static_cast<unsigned long long>(rank_high(f)) << 32) | (0xffffffffu - index);
}

template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int kN = 4;
  __device__ static void unpack(const uint4& v, float (&x)[4]) { unpack16(v, x); }
  __device__ static float most(const uint4& v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static constexpr unsigned kNegInf = 0xff800000u;
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int kN = 8;
  __device__ static void unpack(const uint4& v, float (&x)[8]) { unpack16_bf16(v, x); }
  __device__ static float most(const uint4& v) {
    const __nv_bfloat162 m = group_max_h2<__nv_bfloat162>(v);
    return fmaxf(__low2float(m), __high2float(m));
  }
  static constexpr unsigned kNegInf = Packed16<__nv_bfloat162>::kNegInf;
};
template <> struct Vec<__half> {
  static constexpr int kN = 8;
  __device__ static void unpack(const uint4& v, float (&x)[8]) { unpack16_f16(v, x); }
  __device__ static float most(const uint4& v) {
    const __half2 m = group_max_h2<__half2>(v);
    return fmaxf(__low2float(m), __high2float(m));
  }
  static constexpr unsigned kNegInf = Packed16<__half2>::kNegInf;
};

// A row as 16-byte vectors from the aligned address at or below its start: element e of vector v is x[v * kN - lead + e].
// Vectors [0, nvec) hold it; all but the first and last (its edges, when the row's ends fall inside them) are whole and
// read as vectors.
template <typename T>
struct Row {
  static constexpr int kN = Vec<T>::kN;
  const T* x;
  const uint4* base;
  int V, lead, nvec;
  __device__ __forceinline__ Row(const T* p, int n) : x(p), V(n) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    base = reinterpret_cast<const uint4*>(at & ~uintptr_t(15));
    lead = (int)((at & 15) / sizeof(T));
    nvec = (lead + n + kN - 1) / kN;
  }
  __device__ __forceinline__ int index(int v, int e) const { return v * kN - lead + e; }
  __device__ __forceinline__ int whole_begin() const { return lead ? 1 : 0; }
  __device__ __forceinline__ int whole_end() const { return (lead + V) / kN; }
  __device__ __forceinline__ uint4 load(int v) const { return __ldg(base + v); }     // a whole vector
  __device__ __noinline__ uint4 edge(int v) const {                                  // missing elements -inf
    unsigned w[4] = {Vec<T>::kNegInf, Vec<T>::kNegInf, Vec<T>::kNegInf, Vec<T>::kNegInf};
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      const int i = index(v, e);
      if (i < 0 || i >= V) continue;
      if constexpr (kN == 4) {
        w[e] = __float_as_uint(to_f32(x[i]));
      } else {
        const unsigned bits = reinterpret_cast<const unsigned short*>(x)[i];
        w[e / 2] = e & 1 ? (w[e / 2] & 0xffffu) | bits << 16 : (w[e / 2] & 0xffff0000u) | bits;
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void any(int v, float (&f)[kN]) const {
    const uint4 raw = v >= whole_begin() && v < whole_end() ? load(v) : edge(v);
    Vec<T>::unpack(raw, f);
  }
};

// A part's numbers: maximum, sum, sum of (x - m) e^(x - m) in log2 units.  Its keys follow the parts'.
struct Part {
  float m, s, e;
};

struct Shared {
  unsigned group[kGroups];
  unsigned bound;
  int count, last, hits;
  unsigned short step_high[kSteps][kThreads];    // upper half of the rank of a thread's largest in each of its steps
  int hit[kMaxHits];                             // steps that reach the bound: step << 8 | thread
  unsigned long long list[kCandidates + 32], top[kMaxTop];
  float red_m[kThreads / 32], red_s[kThreads / 32], red_e[kThreads / 32];
  unsigned long long red_k[kThreads / 32];
  Part parts[kMaxParts];
};

// S and E (log2 units) relative to m moved to the larger maximum mn; nothing yet: s = 0, m = -FLT_MAX.
__device__ __forceinline__ void rebase(float& m, float& s, float& e, float mn, float k2) {
  const float shift = fmaxf((m - mn) * k2, -200.0f), f = exp2f(shift);
  e = (e + shift * s) * f;
  s *= f;
  m = mn;
}

// grid (C, T).  parts [T][C], keys [T][C][num_top]: the workspace, read by the row's last CTA; tickets [T], 0 between calls.
template <typename T>
__global__ void __launch_bounds__(kThreads, 5)
    logprobs_kernel(const T* logits, long long row_stride, int V, const long long* tokens, const float* temps, int num_top,
                    float* lp, float* entropy, long long* top_ids, float* top_lp, unsigned* tickets, Part* parts,
                    unsigned long long* keys, int* err) {
  constexpr int kN = Vec<T>::kN;
  __shared__ Shared sh;
  const int C = gridDim.x, part = blockIdx.x;
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long token = tokens[row];
  if (token < 0) {                               // a padding row
    if (part == 0) {
      if (tid == 0) lp[row] = entropy[row] = 0.0f;
      if (tid < num_top) {
        top_ids[(long long)row * num_top + tid] = -1;
        top_lp[(long long)row * num_top + tid] = 0.0f;
      }
    }
    return;
  }
  const Row<T> r(logits + row * row_stride, V);
  const int per = (r.nvec + C - 1) / C;
  const int v0 = min(r.nvec, part * per), v1 = min(r.nvec, v0 + per);
  const float temp = temps ? temps[row] : 1.0f;
  const float k2 = 1.4426950408889634f / temp;
  if (tid == 0) sh.count = sh.hits = 0;

  // ---- one pass: running maximum, sum and weighted sum of this thread's elements (every kThreads-th vector of the part)
  float m = -FLT_MAX, s = 0.0f, e2 = 0.0f;
  const uint4 nothing = make_uint4(Vec<T>::kNegInf, Vec<T>::kNegInf, Vec<T>::kNegInf, Vec<T>::kNegInf);
  const int w0 = max(v0, r.whole_begin()), w1 = min(v1, r.whole_end());
  int step = 0;
  for (int v = v0 + tid; v < w1; v += kUnroll * kThreads) {
    uint4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int at = v + u * kThreads;
      raw[u] = at >= w0 && at < w1 ? r.load(at) : nothing;
    }
    float most = -INFINITY;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) most = fmaxf(most, Vec<T>::most(raw[u]));
    if (num_top > 0) {
      const unsigned short h = (unsigned short)(rank_high(most) >> 16);
      unsigned short& slot = sh.step_high[step % kSteps][tid];
      slot = step < kSteps || h > slot ? h : slot;
      ++step;
    }
    rebase(m, s, e2, fmaxf(m, most), k2);
    const float2 neg = make_float2(-m, -m), kk = make_float2(k2, k2);
    float2 ss = make_float2(0.0f, 0.0f), ee = ss;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float x[kN];
      Vec<T>::unpack(raw[u], x);
#pragma unroll
      for (int i = 0; i < kN; i += 2) {
        const float2 d = sm100::mul_x2(sm100::add_x2(make_float2(x[i], x[i + 1]), neg), kk);
        const float2 p = make_float2(sm100::ex2_approx(d.x), sm100::ex2_approx(d.y));
        ss = sm100::add_x2(ss, p);
        ee = sm100::fma_x2(make_float2(fmaxf(d.x, -200.0f), fmaxf(d.y, -200.0f)), p, ee);     // -inf: -200 * 0
      }
    }
    s += ss.x + ss.y;
    e2 += ee.x + ee.y;
  }
  // the row's edges, where they are this thread's
  for (int end = 0; end < 2; ++end) {
    const int v = end ? r.whole_end() : 0;
    if ((end ? v >= r.nvec || v < r.whole_begin() : r.whole_begin() == 0) || v < v0 || v >= v1 || (v - v0) % kThreads != tid)
      continue;
    float x[kN];
    const uint4 raw = r.edge(v);
    Vec<T>::unpack(raw, x);
    rebase(m, s, e2, fmaxf(m, Vec<T>::most(raw)), k2);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const float d = (x[i] - m) * k2, p = sm100::ex2_approx(d);
      s += p;
      e2 = fmaf(fmaxf(d, -200.0f), p, e2);
    }
  }
  unsigned high = 0;                             // this thread's largest, as ranked; 0: no elements
  if (num_top > 0 && v0 + tid < v1) {
    high = rank_high(m);
    // that says too little where a NaN or +inf is among its elements, or none above the type's lowest
    if (s != s || m == -FLT_MAX) {
      high = 0;
      for (int v = v0 + tid; v < v1; v += kThreads) {
        float x[kN];
        r.any(v, x);
#pragma unroll
        for (int i = 0; i < kN; ++i)
          if (r.index(v, i) >= 0 && r.index(v, i) < V) high = max(high, rank_high(x[i]));
      }
    }
  }

  // ---- the part's sums, and the groups' maxima
  float bm = warp_max_f32(m);
  if (lane == 0) sh.red_m[warp] = bm;
  if (num_top > 0) {
    unsigned g = max(high, __shfl_xor_sync(0xffffffffu, high, 1));
    g = max(g, __shfl_xor_sync(0xffffffffu, g, 2));
    if ((tid & 3) == 0) sh.group[tid >> 2] = g;
  }
  __syncthreads();
  bm = sh.red_m[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) bm = fmaxf(bm, sh.red_m[w]);
  const float s_own = s;
  rebase(m, s, e2, bm, k2);
  s = warp_sum_f32(s);
  e2 = warp_sum_f32(e2);
  if (lane == 0) {
    sh.red_s[warp] = s;
    sh.red_e[warp] = e2;
  }
  // ---- the bound: the num_top-th largest of the groups' maxima
  if (num_top > 0 && tid < kGroups) {
    const unsigned k = sh.group[tid];
    int larger = 0;
#pragma unroll 16
    for (int i = 0; i < kGroups; ++i) larger += sh.group[i] > k || (sh.group[i] == k && i < tid);
    if (larger == num_top - 1) sh.bound = k;
  }
  __syncthreads();
  Part mine{bm, 0.0f, 0.0f};
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    mine.s += sh.red_s[w];
    mine.e += sh.red_e[w];
  }
  if (num_top > 0) {
    const unsigned bound = sh.bound;
    // the steps that reach it (all of a thread's that saw a NaN), then their vectors spread over the CTA, and the edges
    const bool nan = s_own != s_own;
    if (high >= bound)
      for (int i = 0; i < min(step, kSteps); ++i)
        if (nan || sh.step_high[i][tid] >= bound >> 16) {
          const int at = atomicAdd(&sh.hits, 1);
          if (at < kMaxHits) sh.hit[at] = i << 8 | tid;
        }
    __syncthreads();
    auto consider = [&](int v) {
      float x[kN];
      r.any(v, x);
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        const int at = r.index(v, j);
        if (rank_high(x[j]) >= bound && at >= 0 && at < V) {
          const int slot = atomicAdd(&sh.count, 1);
          if (slot < kCandidates) sh.list[slot] = rank_key(x[j], at);
        }
      }
    };
    constexpr int kStride = kUnroll * kThreads;
    const int each = ((v1 - v0 + kStride - 1) / kStride + kSteps - 1) / kSteps * kUnroll;    // vectors a hit stands for
    const int all = min(sh.hits, kMaxHits) * each;
#pragma unroll 2
    for (int i = tid; i < all; i += kThreads) {
      const int hit = sh.hit[i / each], u = i % each;
      const int v = v0 + (hit & 255) + ((hit >> 8) + u / kUnroll * kSteps) * kStride + u % kUnroll * kThreads;
      if (v >= w0 && v < w1) consider(v);
    }
    if (tid < 2) {
      const int v = tid ? r.nvec - 1 : 0;
      if (v >= v0 && v < v1 && (v < w0 || v >= w1) && (tid == 0 || v > 0)) consider(v);
    }
    if (tid == 0 && sh.hits > kMaxHits) atomicAdd(&sh.count, kCandidates + 1);       // not all looked at
    if (tid < num_top) sh.top[tid] = 0;
    __syncthreads();
    const int found = sh.count;
    if (found <= kCandidates) {
      block_top_sorted<kThreads>(sh.list, found, num_top, sh.top);
    } else {             // ties past the list: one alternative a pass
      unsigned long long last = ~0ull;
      for (int n = 0; n < num_top; ++n) {
        unsigned long long best = 0;
        if (high >= bound)
          for (int v = v0 + tid; v < v1; v += kThreads) {
            float x[kN];
            r.any(v, x);
#pragma unroll
            for (int i = 0; i < kN; ++i) {
              const int at = r.index(v, i);
              const unsigned long long key = rank_key(x[i], at);
              if (at >= 0 && at < V && key < last && key > best) best = key;
            }
          }
        best = warp_max_u64(best);
        if (lane == 0) sh.red_k[warp] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) best = sh.red_k[w] > best ? sh.red_k[w] : best;
        last = best;
        if (tid == 0) sh.top[n] = best;
        __syncthreads();
      }
    }
  }
  // ---- the row's last CTA merges the parts
  if (C > 1) {
    if (tid == 0) parts[(long long)row * C + part] = mine;
    if (tid < num_top) keys[((long long)row * C + part) * num_top + tid] = sh.top[tid];
    __threadfence();
    __syncthreads();
    if (tid == 0) sh.last = atomicInc(&tickets[row], C - 1) == (unsigned)(C - 1);
    __syncthreads();
    if (!sh.last) return;
    __threadfence();
    if (tid < C) sh.parts[tid] = Part{__ldcg(&parts[(long long)row * C + tid].m), __ldcg(&parts[(long long)row * C + tid].s),
                                      __ldcg(&parts[(long long)row * C + tid].e)};
    for (int i = tid; i < C * num_top; i += kThreads) sh.list[i] = __ldcg(keys + (long long)row * C * num_top + i);
    __syncthreads();
    if (num_top > 0) block_top_sorted<kThreads>(sh.list, C * num_top, num_top, sh.top);
    float mn = sh.parts[0].m;
    for (int c = 1; c < C; ++c) mn = fmaxf(mn, sh.parts[c].m);
    mine = Part{mn, 0.0f, 0.0f};
    for (int c = 0; c < C; ++c) {
      Part o = sh.parts[c];
      rebase(o.m, o.s, o.e, mn, k2);
      mine.s += o.s;
      mine.e += o.e;
    }
  }
  const float log_s = logf(mine.s);
  if (tid == 0) {
    if (token >= V) {
      atomicCAS(err, 0, kErrToken);
      lp[row] = NAN;
    } else {
      lp[row] = (to_f32(r.x[token]) - mine.m) / temp - log_s;
    }
    entropy[row] = log_s - mine.e * 0.6931471805599453f / mine.s;
  }
  if (tid < num_top) {
    const unsigned long long key = sh.top[tid];
    const unsigned h = (unsigned)(key >> 32);
    const float x = h == 0xfffffffeu ? NAN : key_to_float(h);
    top_ids[(long long)row * num_top + tid] = argmax_key_index(key);
    top_lp[(long long)row * num_top + tid] = (x - mine.m) / temp - log_s;
  }
}

// CTAs a row: enough for three an SM over the rows, each thread left at least four vectors; one where the rows do that alone.
// (64 bf16 rows of 151,936 with 5 alternatives: 15.5, 15.2, 16.5, 16.9 and 20.8 us with 1, 2, 3, 4 and 6 an SM; 288 fp32 rows
// of 151,936 without 36.0, 32.8, 32.8, 40.3 and 37.0, of 50,257 15.3, 14.8, 14.8, 18.9 and 18.3; 512 bf16 rows of 151,936 with
// 20 45.8 to three, then 57.)
static int parts_of(long long rows, long long V, int dtype, int sm_count) {
  const long long vectors = V / (16 / (long long)dtype_bytes(dtype));
  const long long wanted = (3LL * sm_count + rows - 1) / rows, most = vectors / (kThreads * 4);
  const long long c = wanted < most ? wanted : most;
  return (int)(c < 1 ? 1 : c > kMaxParts ? kMaxParts : c);
}

// Workspace: [rows] tickets at a fixed place (zero between calls), then the parts and their keys.
constexpr long long kTicketBytes = 65536 * 4;
static long long workspace_bytes(long long rows, int C, int num_top) {
  return kTicketBytes + rows * C * 8 * num_top + (rows * C * (long long)sizeof(Part) + 255) / 256 * 256;
}

template <typename T>
static int launch(const void* logits, long long rows, int V, long long row_stride, const long long* tokens,
                  const float* temps, int num_top, int C, float* lp, float* entropy, long long* top_ids, float* top_lp,
                  void* workspace, int* err, cudaStream_t stream) {
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  unsigned long long* keys = reinterpret_cast<unsigned long long*>(ws + kTicketBytes);
  Part* parts = reinterpret_cast<Part*>(keys + rows * C * num_top);
  logprobs_kernel<T><<<dim3((unsigned)C, (unsigned)rows), kThreads, 0, stream>>>(
      static_cast<const T*>(logits), row_stride, V, tokens, temps, num_top, lp, entropy, top_ids, top_lp,
      reinterpret_cast<unsigned*>(ws), parts, keys, err);
  SPECDEC_LAUNCH_CHECK();
  return kOk;
}

}  // namespace logprobs
}  // namespace specdec

using namespace specdec;

extern "C" {

long long specdec_logprobs_workspace_bytes(long long T, long long V, int dtype, int num_top) {
  namespace L = specdec::logprobs;
  DeviceInfo info;
  if (T < 0 || T > 65535 || V < 1 || num_top < 0 || num_top > L::kMaxTop || !dtype_ok(dtype) || device_info(&info) != kOk)
    return -1;
  return T == 0 ? 0 : L::workspace_bytes(T, L::parts_of(T, V, dtype, info.sm_count), num_top);
}

int specdec_token_logprobs(const void* logits, int dtype, long long T, long long V, long long row_stride,
                           const long long* tokens, const float* temperatures, int num_top, float* logprobs,
                           float* entropy, long long* top_ids, float* top_logprobs, void* workspace,
                           long long workspace_bytes, int* err, void* stream) {
  namespace L = specdec::logprobs;
  SPECDEC_CHECK_ARG(dtype_ok(dtype), "dtype code %d", dtype);
  SPECDEC_CHECK_ARG(T >= 0 && T <= 65535 && V >= 1 && V <= (1 << 24) && row_stride >= V, "bad sizes: %lld rows of %lld", T, V);
  SPECDEC_CHECK_ARG(num_top >= 0 && num_top <= L::kMaxTop && num_top <= V, "num_top %d: 0 to %d and at most V", num_top,
                    L::kMaxTop);
  if (T == 0) return kOk;
  SPECDEC_CHECK_ARG(logits && tokens && logprobs && entropy && workspace && err && (num_top == 0 || (top_ids && top_logprobs)),
                    "null pointer argument");
  SPECDEC_CHECK_ARG(reinterpret_cast<uintptr_t>(logits) % dtype_bytes(dtype) == 0, "logits not aligned to their type");
  SPECDEC_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, "workspace must be 256-byte aligned");
  DeviceInfo info;
  if (int st = device_info(&info)) return st;
  const int C = L::parts_of(T, V, dtype, info.sm_count);
  if (workspace_bytes < L::workspace_bytes(T, C, num_top))
    return set_error(kWorkspaceTooSmall, "log-probability workspace of %lld bytes, %lld needed", workspace_bytes,
                     L::workspace_bytes(T, C, num_top));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto go = [&](auto fn) {
    return fn(logits, T, (int)V, row_stride, tokens, temperatures, num_top, C, logprobs, entropy, top_ids, top_logprobs,
              workspace, err, s);
  };
  if (dtype == kF32) return go(L::launch<float>);
  if (dtype == kBF16) return go(L::launch<__nv_bfloat16>);
  return go(L::launch<__half>);
}

}  // extern "C"
