// A verification round's metadata on the GPU: block tables, slot map, input ids, positions and the cumulative lengths
// from the requests' token counts, with the blocks a row still lacks taken from a free stack.
//
// Same values as verify_varlen_metadata (nanovllm/engine/batch_metadata.py:121-181; its packed host form is
// pack_verify_metadata) followed by the placement of the drafts among the input ids (speculative.py:514-517), and as
// the block manager's append of the blocks a row needs (nanovllm/engine/block_manager.py, scheduler.py:75-92), taken
// from the top of the stack in row order.
//
// For rows r < R with start_r = lengths_r - 1 and n_r = verified_lens_r (or k + 1):
//   need_r = ceil((start_r + n_r) / block_size) blocks; new_r = max(0, need_r - held_r);
//   token j of row r: flat index sum_{r' < r} n_r' + j, position start_r + j, slot by the table, id the last token (j = 0)
//   or draft j - 1; keys of the row start_r + n_r.
// Rows R .. num_rows - 1 are padding: min(left, k + 1) tokens each at positions 0 on, slot -1, id 0, the pad block.
//
// One launch, one warp a row.  Everything is a prefix over R rows of three numbers; a warp sums the rows before its own
// straight from the inputs (a few loads a lane) instead of waiting for a scan of another block.  The rows' block counts
// and the free count, which every warp reads, are written by the CTA that finishes last (a ticket).  A block id outside the
// cache is met only where a row's table is read; the ticket counts the CTAs that met one, and the last CTA empties the
// metadata then instead of writing the counts.
// Latency-bound: the loads' and the ticket's round trips.  64 rows of up to 64 blocks take 4.7 us, 512 rows 7.5 us
// (4.6 and 7.1 without the check of the ids; a chain of array operations on the GPU: 646 and 667 us).  Every warp's sums over
// all rows make it grow as their square from there: 2048 rows 20 us, 4096 rows 67 us.
#include "common.cuh"

namespace specdec {
namespace metadata {

constexpr int kThreads = 256;
constexpr int kRowsPerCta = kThreads / 32;
constexpr int kErrPool = 6, kErrRows = 7, kErrBlock = 9;
constexpr unsigned kSpoiled = 1u << 16;  // in the ticket, above the count of at most 65535 / kRowsPerCta + 1 CTAs

struct Args {
  const long long* lengths;        // [R] tokens of each row, the last token included
  const long long* last_tokens;    // [R]
  const long long* drafts;         // [R, k] or null: their ids are left 0
  const long long* verified_lens;  // [R] or null: k + 1 each
  int* tables;                     // [R, table_width], in place
  int* num_blocks;                 // [R] blocks each row holds, in place
  const int* free_blocks;          // [capacity] stack, top at *free_count - 1; null: rows hold what they need
  int* free_count;                 // [1], in place
  int R, k, table_width, capacity, block_size, num_rows, num_tokens, pad_block_id, width;
  unsigned cache_blocks;           // ids of the rows' blocks are below it
  long long *input_ids, *positions;
  int *slots, *cu_q, *cu_k, *out_tables;
  unsigned* ticket;                // 0 between launches
  int* err;
};

struct Row {
  int n, held, need;               // verified tokens, blocks held, blocks needed
  long long start;
  int bad;
};

__device__ __forceinline__ Row row_of(const Args& a, int r) {
  Row x;
  const long long length = a.lengths[r], n = a.verified_lens ? a.verified_lens[r] : a.k + 1;
  x.held = a.num_blocks[r];
  x.start = length - 1;
  // the length against what the table leaves for the other tokens: their sum could pass 64 bits
  x.bad = n < 1 || n > a.k + 1 || length < 1 || x.held < 0 || x.held > a.table_width ||
          length > (long long)a.table_width * a.block_size - (n - 1);
  x.n = x.bad ? 0 : (int)n;
  if (x.bad) x.start = 0;
  x.need = (int)(((unsigned)(x.start + x.n) + (unsigned)a.block_size - 1u) / (unsigned)a.block_size);   // below 2^31 here
  if (!x.bad && (max(x.need, x.held) > a.width || (!a.free_blocks && x.need > x.held))) x.bad = 1;
  return x;
}

__device__ __forceinline__ long long warp_sum_ll(long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Every row empty, every token padding: by the last CTA, over what the others wrote.  Not inlined: it has no part in the
// registers of the path that every call takes (inlined, 512 rows took 9.4 us for 7.5).
__device__ __noinline__ void clear(const Args& a) {
  __threadfence();
  if (threadIdx.x == 0) atomicCAS(a.err, 0, kErrBlock);
  for (int i = threadIdx.x; i <= a.num_rows; i += kThreads) a.cu_q[i] = a.cu_k[i] = 0;
  for (int t = threadIdx.x; t < a.num_tokens; t += kThreads) {
    a.positions[t] = 0;
    a.input_ids[t] = 0;
    a.slots[t] = -1;
  }
  for (long long i = threadIdx.x; i < (long long)a.num_rows * a.width; i += kThreads) a.out_tables[i] = a.pad_block_id;
}

__global__ void __launch_bounds__(kThreads) verify_metadata_kernel(const __grid_constant__ Args a) {
  __shared__ int last_cta, spoiled;
  const int lane = threadIdx.x & 31;
  const int r = blockIdx.x * kRowsPerCta + (threadIdx.x >> 5);
  // sums over the rows before r and over all rows: tokens, keys, new blocks
  int tokens = 0, all_tokens = 0, fresh = 0, all_fresh = 0, bad = 0;
  long long keys = 0, all_keys = 0;
#pragma unroll 4
  for (int i = lane; i < a.R; i += 32) {
    const Row x = row_of(a, i);
    const int f = max(0, x.need - x.held);
    bad |= x.bad;
    all_tokens += x.n;
    all_fresh += f;
    all_keys += x.start + x.n;
    if (i < r) {
      tokens += x.n;
      fresh += f;
      keys += x.start + x.n;
    }
  }
  tokens = __reduce_add_sync(0xffffffffu, tokens);
  all_tokens = __reduce_add_sync(0xffffffffu, all_tokens);
  fresh = __reduce_add_sync(0xffffffffu, fresh);
  all_fresh = __reduce_add_sync(0xffffffffu, all_fresh);
  keys = warp_sum_ll(keys);
  all_keys = warp_sum_ll(all_keys);
  bad = __any_sync(0xffffffffu, bad);
  const int query_len = a.k + 1;
  const int available = a.free_blocks ? min(*a.free_count, a.capacity) : 0;
  const int left = a.num_tokens - all_tokens;
  bad |= left < 0 || left > (long long)(a.num_rows - a.R) * query_len || all_keys + left > 0x7fffffffLL;
  const bool dry = !bad && all_fresh > available;
  const bool idle = bad || dry;      // nothing is assigned or stored: every row empty
  if (idle && r == 0 && lane == 0) atomicCAS(a.err, 0, bad ? kErrRows : kErrPool);
  bool bad_id = false;
  if (r < a.num_rows) {
    int first, n, kv;
    long long start = 0, k0;
    if (idle) {
      first = n = kv = 0;
      k0 = 0;
    } else if (r < a.R) {
      const Row x = row_of(a, r);
      first = tokens;
      n = x.n;
      start = x.start;
      kv = (int)(x.start + x.n);
      k0 = keys;
    } else {
      const int before = (int)min((long long)(r - a.R) * query_len, (long long)left);
      first = all_tokens + before;
      n = min(left - before, query_len);
      kv = n;
      k0 = all_keys + before;
    }
    if (lane == 0) {
      if (r == 0) a.cu_q[0] = a.cu_k[0] = 0;
      a.cu_q[r + 1] = first + n;
      a.cu_k[r + 1] = (int)(k0 + kv);
    }
    // the row's table: what it holds, then its new blocks from the top of the stack, then the pad block
    int* out = a.out_tables + (long long)r * a.width;
    int* table = a.tables + (long long)r * a.table_width;
    int held = 0, have = 0, need = 0;
    if (r < a.R && !idle) {
      const Row x = row_of(a, r);
      held = x.held;
      need = x.need;
      have = max(held, need);
    }
    for (int j = lane; j < a.width; j += 32) {
      int b = a.pad_block_id;
      if (j < held) {
        b = table[j];
      } else if (j < have) {
        b = a.free_blocks[available - 1 - (fresh + j - held)];
        table[j] = b;
      }
      if (j < need && (unsigned)b >= a.cache_blocks) bad_id = true;
      out[j] = b;
    }
    __syncwarp();
    for (int j = lane; j < n; j += 32) {
      const unsigned pos = (unsigned)start + j, bs = (unsigned)a.block_size;
      const int t = first + j;
      const bool real = r < a.R;
      a.positions[t] = pos;
      a.input_ids[t] = !real ? 0 : j == 0 ? a.last_tokens[r] : a.drafts ? a.drafts[(long long)r * a.k + j - 1] : 0;
      a.slots[t] = real ? (int)((unsigned)table[pos / bs] * bs + pos % bs) : -1;    // of a bad id: emptied by the last CTA
    }
  }
  if (idle)                           // no row has tokens: the whole token range is padding
    for (int t = blockIdx.x * kThreads + threadIdx.x; t < a.num_tokens; t += gridDim.x * kThreads) {
      a.positions[t] = 0;
      a.input_ids[t] = 0;
      a.slots[t] = -1;
    }
  // ---- the last CTA to get here (every other has read the counts) writes the rows' block counts and the free count
  const int any_bad = __syncthreads_or(bad_id);
  if (threadIdx.x == 0) {
    __threadfence();
    const unsigned mine = any_bad ? 1u + kSpoiled : 1u, all = atomicAdd(a.ticket, mine) + mine;
    last_cta = all % kSpoiled == gridDim.x;
    spoiled = all >= kSpoiled;
    if (last_cta) *a.ticket = 0;
  }
  __syncthreads();
  if (!last_cta || idle) return;
  if (spoiled) {
    clear(a);
    return;
  }
  if (!a.free_blocks) return;
  for (int i = threadIdx.x; i < a.R; i += kThreads) {
    const Row x = row_of(a, i);
    if (x.need > x.held) a.num_blocks[i] = x.need;
  }
  if (threadIdx.x == 0) *a.free_count = available - all_fresh;
}

}  // namespace metadata
}  // namespace specdec

using namespace specdec;

extern "C" {

int specdec_verify_metadata_ex(const long long* lengths, const long long* last_tokens, const long long* drafts,
                               const long long* verified_lens, int R, int k, int* block_tables, int table_width,
                               int* num_blocks, const int* free_blocks, int* free_count, int free_capacity,
                               int block_size, int num_rows, int num_tokens, int pad_block_id, int width,
                               long long* buf64, int* buf32, unsigned* ticket, int* err, long long cache_blocks,
                               void* stream) {
  using namespace metadata;
  SPECDEC_CHECK_ARG(R >= 0 && num_rows >= R && num_rows >= 1 && num_rows <= 65535 && k >= 0 && k <= 1023,
                    "bad row sizes: %d of %d rows, %d drafts", R, num_rows, k);
  SPECDEC_CHECK_ARG(num_tokens >= 1 && width >= 1 && table_width >= 1 && block_size >= 1,
                    "token, table and block sizes must be positive");
  SPECDEC_CHECK_ARG((long long)num_rows * (k + 1) <= 0x7fffffffLL && (long long)table_width * block_size <= 0x7fffffffLL,
                    "sizes past 32 bits");
  SPECDEC_CHECK_ARG(R == 0 || (lengths && last_tokens && block_tables && num_blocks), "null row argument");
  SPECDEC_CHECK_ARG(!free_blocks == !free_count && free_capacity >= 0, "give free_blocks and free_count together");
  SPECDEC_CHECK_ARG(buf64 && buf32 && ticket && err, "null pointer argument");
  SPECDEC_CHECK_ARG(cache_blocks >= 0 && cache_blocks <= 0x7fffffffLL / block_size, "the cache's slots must fit 32 bits");
  Args a{};
  a.lengths = lengths;
  a.last_tokens = last_tokens;
  a.drafts = drafts;
  a.verified_lens = verified_lens;
  a.tables = block_tables;
  a.num_blocks = num_blocks;
  a.free_blocks = free_blocks;
  a.free_count = free_count;
  a.R = R;
  a.k = k;
  a.table_width = table_width;
  a.capacity = free_capacity;
  a.block_size = block_size;
  a.num_rows = num_rows;
  a.num_tokens = num_tokens;
  a.pad_block_id = pad_block_id;
  a.width = width;
  a.cache_blocks = (unsigned)(cache_blocks ? cache_blocks : 0x7fffffffLL / block_size);
  a.input_ids = buf64;
  a.positions = buf64 + num_tokens;
  a.slots = buf32;
  a.cu_q = buf32 + num_tokens;
  a.cu_k = a.cu_q + num_rows + 1;
  a.out_tables = a.cu_k + num_rows + 1;
  a.ticket = ticket;
  a.err = err;
  const unsigned grid = (unsigned)((num_rows + kRowsPerCta - 1) / kRowsPerCta);
  verify_metadata_kernel<<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  SPECDEC_LAUNCH_CHECK();
  return kOk;
}

int specdec_verify_metadata(const long long* lengths, const long long* last_tokens, const long long* drafts,
                            const long long* verified_lens, int R, int k, int* block_tables, int table_width,
                            int* num_blocks, const int* free_blocks, int* free_count, int free_capacity,
                            int block_size, int num_rows, int num_tokens, int pad_block_id, int width,
                            long long* buf64, int* buf32, unsigned* ticket, int* err, void* stream) {
  return specdec_verify_metadata_ex(lengths, last_tokens, drafts, verified_lens, R, k, block_tables, table_width, num_blocks,
                                    free_blocks, free_count, free_capacity, block_size, num_rows, num_tokens, pad_block_id,
                                    width, buf64, buf32, ticket, err, 0, stream);
}

}  // extern "C"
