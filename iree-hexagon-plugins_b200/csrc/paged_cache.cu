// The paged KV cache of a batch of requests with different lengths: the block
// tables and slot maps of a step, built on the GPU from the request lengths,
// and the cache update through the slot map. attention_paged.cu reads the
// cache through the same tables.
//
// The reference's KV-cache models keep one length for the whole batch
// (integration_tests/models/kv_cache.py:91-112); these entries have no
// counterpart there.
#include <algorithm>

#include "runtime_common.h"
#include "sm100.cuh"

namespace hxb {
namespace {

// ------------------------------------------------------------ step tables
// For request b with c_b cached and n_b new tokens, T_b = c_b + n_b and blocks
// of P rows:
//   q_start[b]  = sum_{a<b} n_a
//   fresh blocks f_b = ceil(T_b / P) - ceil(c_b / P), taken from the free list
//   at cursor + F_b, F_b = sum_{a<b} f_a
//   slot of token i of b = block(pos / P) * P + pos % P,  pos = c_b + i
// i.e. two prefix sums over the requests, then independent writes. The work is a
// few bytes per request and token: latency is the cost. Every CTA scans all the
// requests by itself (c_b, q_start and F_b stay in its shared memory) and the
// CTAs share the writes; one launch, no scratch. Table entries of fresh blocks
// are written, entries of begun blocks read, never the same. In place (kv_lens
// over cached_lens, the cursor over itself) every read of an input has to come
// before the first write of an output: then the CTAs are one cluster with a
// barrier in between. Measured (one B200): 8 requests 2.5 us, 1001 requests with
// 33 thousand tokens 6.1 us (in place 10.3).
constexpr int kTabThreads = 1024;
constexpr int kTabCluster = 8;
constexpr int kTabMaxBatch = 16384;  // three ints per request in shared memory

struct TabArgs {
  const int* cached;
  const int* fresh_tokens;
  const int* free_blocks;
  const int* cursor;
  int* block_table;
  int* q_start;
  int* kv_lens;
  long long* slots;
  int* cursor_out;
  long long table_ld, max_tokens, num_free;
  int batch, block_rows, table_cols;
  int in_place;  // outputs over inputs: the CTAs are one cluster
  int* status;
};

// Index of the last element of the non-decreasing v[0, n) that is <= x
// (v[0] <= x).
__device__ __forceinline__ int last_not_above(const int* v, int n, int x) {
  int lo = 0, hi = n;  // v[lo] <= x, v[hi] > x
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (v[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Inclusive scans over the warp of two sums.
__device__ __forceinline__ void scan_pair(long long& a, long long& b, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, a, o);
    const long long y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) a += x, b += y;
  }
}

__global__ void __launch_bounds__(kTabThreads) paged_tables_kernel(const TabArgs a) {
  extern __shared__ int tab_smem[];
  int* s_start = tab_smem;             // q_start, clamped to max_tokens
  int* s_first = s_start + a.batch;    // F_b
  int* s_cached = s_first + a.batch;   // c_b
  __shared__ long long s_warp[2][kTabThreads / 32];
  const int tid = threadIdx.x, nt = blockDim.x;
  const int lane = tid & 31, warp = tid >> 5;
  const int ctas = gridDim.x, rank = blockIdx.x;
  const int P = a.block_rows;
  pdl_wait();
  pdl_trigger();

  // (rows and blocks fit 31 bits: the host checks table_cols * block_rows)
  const int capacity = a.table_cols * P;
  const int num_free = (int)a.num_free, max_tokens = (int)a.max_tokens;
  const int cur = a.cursor[0];
  const int cursor = min(max(cur, 0), num_free);
  bool bad = cur < 0 || cur > num_free;
  // the blocks of request b that are new to it: columns [before, after)
  auto blocks_of = [&](int rows) { return (int)(((unsigned)rows + P - 1) / (unsigned)P); };
  auto length_of = [&](int c, int n) { return n > capacity - c ? capacity : c + n; };
  // thread-contiguous chunks of requests, then one block scan of both sums
  const int per = (a.batch + nt - 1) / nt;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  long long tok = 0;
  long long blk = 0;
#pragma unroll 4
  for (int b = b0; b < b1; ++b) {
    int c = a.cached[b], n = a.fresh_tokens[b];
    bad |= c < 0 || n < 0 || c > capacity || n > capacity - c;
    c = min(max(c, 0), capacity);
    n = max(n, 0);
    s_cached[b] = c;
    s_start[b] = n;  // replaced by the prefix sum below
    tok += n;
    blk += blocks_of(length_of(c, n)) - blocks_of(c);
  }
  const long long my_tok = tok, my_blk = blk;
  scan_pair(tok, blk, lane);
  if (lane == 31) s_warp[0][warp] = tok, s_warp[1][warp] = blk;
  __syncthreads();
  // every warp scans the warps' sums
  long long wt = lane < nt / 32 ? s_warp[0][lane] : 0, wb = lane < nt / 32 ? s_warp[1][lane] : 0;
  scan_pair(wt, wb, lane);
  const long long tok_total = __shfl_sync(0xffffffffu, wt, 31);
  const long long blk_total = __shfl_sync(0xffffffffu, wb, 31);
  const long long tok_base = __shfl_sync(0xffffffffu, wt, max(warp - 1, 0)) * (warp > 0);
  const long long blk_base = __shfl_sync(0xffffffffu, wb, max(warp - 1, 0)) * (warp > 0);
  tok += tok_base - my_tok;  // exclusive
  blk += blk_base - my_blk;
#pragma unroll 1
  for (int b = b0; b < b1; ++b) {
    const int c = s_cached[b], n = s_start[b];
    s_start[b] = (int)min(tok, (long long)max_tokens);
    s_first[b] = (int)min(blk, (long long)INT32_MAX);
    tok += n;
    blk += blocks_of(length_of(c, n)) - blocks_of(c);
  }
  bad |= tok_total > max_tokens;
  const int total = (int)min(tok_total, (long long)max_tokens);
  const int available = num_free - cursor;
  const int taken = (int)min(blk_total, (long long)available);
  __syncthreads();
  if (a.in_place && ctas > 1) cluster_sync_all();  // every input has been read

  const int step = ctas * nt, first = rank * nt + tid;
#pragma unroll 1
  for (int b = first; b < a.batch; b += step) {
    a.q_start[b] = s_start[b];
    a.kv_lens[b] = length_of(s_cached[b], max(a.fresh_tokens[b], 0));
  }
  if (first == 0) {
    a.q_start[a.batch] = total;
    a.cursor_out[0] = cursor + taken;
    a.cursor_out[1] = (int)min(blk_total - taken, (long long)INT32_MAX);
  }
  // table entries of the fresh blocks (-1 where the free list has run out)
  const int entries = (int)min(blk_total, (long long)INT32_MAX - step);
#pragma unroll 1
  for (int f = first; f < entries; f += step) {
    const int b = last_not_above(s_first, a.batch, f);
    const int col = blocks_of(s_cached[b]) + f - s_first[b];
    if (col < a.table_cols)
      a.block_table[b * a.table_ld + col] = f < available ? a.free_blocks[cursor + f] : -1;
  }
  // slots of the new tokens, -1 behind the last one and where there is none
#pragma unroll 1
  for (long long t = first; t < max_tokens; t += step) {
    long long slot = -1;
    if (t < total) {
      const int b = last_not_above(s_start, a.batch, (int)t);
      const int c = s_cached[b], i = (int)t - s_start[b];
      if (i < capacity - c) {
        const unsigned col = (unsigned)(c + i) / (unsigned)P;
        const int row = c + i - (int)col * P, begun = blocks_of(c);
        int block;
        if ((int)col < begun) {
          block = a.block_table[b * a.table_ld + col];
          bad |= block < 0;  // a begun block that is not there
        } else {
          const int f = s_first[b] + (int)col - begun;
          block = f < available ? a.free_blocks[cursor + f] : -1;
        }
        if (block >= 0) slot = (long long)block * P + row;
      }
    }
    a.slots[t] = slot;
  }
  if (bad) atomicOr(a.status, kStatusBadIndex);
}

// ------------------------------------------------------- cache update
// k_cache[slot / P, h, slot % P, :] = k_src[t, h*D:(h+1)*D], V alike. Pure
// data movement: one thread moves one 16-byte vector of K and of V, so a
// warp's loads are contiguous and its stores cover whole 256-byte (D = 128)
// rows. block_rows is a power of two, so a slot splits by shift and mask.
// Measured (one B200): 8246 tokens of 8 heads of 128, 64.6 MB in 12.1 us, 81 % of
// the measured copy rate; 8 tokens 1.6 us.
constexpr int kPutThreads = 256;

struct PutArgs {
  const __half* k_src;
  const __half* v_src;
  const long long* slots;
  __half* k_cache;
  __half* v_cache;
  long long ld_src, block_stride, num_blocks, vectors;
  int row_vectors, head_dim, rows_log2;
  int* status;
};

__global__ void __launch_bounds__(kPutThreads) paged_write_kernel(const PutArgs a) {
  pdl_wait();
  pdl_trigger();
  const long long idx = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (idx >= a.vectors) return;
  const long long t = idx / a.row_vectors;
  const int col = (int)(idx - t * a.row_vectors) * 8;
  const long long slot = a.slots[t];
  if (slot < 0) return;  // a padded row, or a token without a block
  const long long block = slot >> a.rows_log2;
  if (block >= a.num_blocks) {
    if (col == 0) atomicOr(a.status, kStatusBadIndex);
    return;
  }
  const int h = col / a.head_dim, d = col - h * a.head_dim;
  const long long row = slot & ((1ll << a.rows_log2) - 1);
  const long long to = block * a.block_stride + (((long long)h << a.rows_log2) + row) * a.head_dim + d;
  const uint4 k = *reinterpret_cast<const uint4*>(a.k_src + t * a.ld_src + col);
  const uint4 v = *reinterpret_cast<const uint4*>(a.v_src + t * a.ld_src + col);
  *reinterpret_cast<uint4*>(a.k_cache + to) = k;
  *reinterpret_cast<uint4*>(a.v_cache + to) = v;
}

}  // namespace

hxb_status_t check_paged_cache(const char* what, const void* k_cache, const void* v_cache,
                               int64_t block_stride, int64_t num_blocks, int64_t kv_heads,
                               int64_t block_rows, int64_t head_dim) {
  if (!k_cache || !v_cache)
    return fail(HXB_STATUS_INVALID_ARGUMENT, "%s: null cache", what);
  if (!aligned16(k_cache) || !aligned16(v_cache))
    return fail(HXB_STATUS_INVALID_ARGUMENT, "%s: caches must be 16-byte aligned", what);
  if (block_rows < 16 || block_rows > 1024 || (block_rows & (block_rows - 1)))
    return fail(HXB_STATUS_UNSUPPORTED,
                "%s: block_rows %lld is not a power of two from 16 to 1024", what,
                (long long)block_rows);
  if (kv_heads < 1 || kv_heads > (1 << 16) || num_blocks < 1 || num_blocks > INT32_MAX)
    return fail(HXB_STATUS_INVALID_ARGUMENT, "%s: bad cache extents", what);
  if (head_dim < 8 || head_dim % 8 || head_dim > 1024)
    return fail(HXB_STATUS_UNSUPPORTED, "%s: head_dim %lld is not a multiple of 8 up to 1024",
                what, (long long)head_dim);
  if (block_stride % 8 || block_stride < kv_heads * block_rows * head_dim ||
      block_stride > ((int64_t)1 << 38))
    return fail(HXB_STATUS_INVALID_ARGUMENT,
                "%s: block_stride %lld must be a multiple of 8 that holds kv_heads * block_rows * "
                "head_dim elements", what, (long long)block_stride);
  return HXB_OK;
}

}  // namespace hxb

using hxb::fail;

extern "C" hxb_status_t hxb_paged_tables(const hxb_paged_tables_t* args, void* stream) {
  using namespace hxb;
  if (!args) return fail(HXB_STATUS_INVALID_ARGUMENT, "paged_tables: null arguments");
  const auto& [cached_lens, new_lens, batch, block_rows, free_blocks, num_free, cursor, block_table,
               table_ld, table_cols, q_start, kv_lens, slots, max_tokens, cursor_out] = *args;
  if (batch < 1 || batch > kTabMaxBatch)
    return fail(HXB_STATUS_INVALID_ARGUMENT, "paged_tables: 1 to %d requests, not %lld",
                kTabMaxBatch, (long long)batch);
  if (block_rows < 1 || block_rows > (1 << 20) || table_cols < 1 || table_ld < table_cols ||
      table_cols > INT32_MAX / block_rows || max_tokens < 0 || max_tokens > INT32_MAX ||
      num_free < 0 || num_free > INT32_MAX)
    return fail(HXB_STATUS_INVALID_ARGUMENT, "paged_tables: bad extents");
  if (!cached_lens || !new_lens || !cursor || !block_table || !q_start || !kv_lens ||
      !cursor_out || (num_free && !free_blocks) || (max_tokens && !slots))
    return fail(HXB_STATUS_INVALID_ARGUMENT, "paged_tables: null pointer");
  DeviceInfo* dev = nullptr;
  hxb_status_t s = current_device(&dev);
  if (s != HXB_OK) return s;
  TabArgs a{};
  a.cached = cached_lens;
  a.fresh_tokens = new_lens;
  a.free_blocks = free_blocks;
  a.cursor = cursor;
  a.block_table = block_table;
  a.q_start = q_start;
  a.kv_lens = kv_lens;
  a.slots = reinterpret_cast<long long*>(slots);
  a.cursor_out = cursor_out;
  a.table_ld = table_ld;
  a.max_tokens = max_tokens;
  a.num_free = num_free;
  a.batch = (int)batch;
  a.block_rows = (int)block_rows;
  a.table_cols = (int)table_cols;
  a.status = dev->status_word;
  const size_t smem = (size_t)batch * 3 * sizeof(int);
  static bool configured[64] = {};
  if (!configured[dev->ordinal]) {
    const cudaError_t e =
        cudaFuncSetAttribute(paged_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kTabMaxBatch * 3 * (int)sizeof(int));
    if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(paged tables)");
    configured[dev->ordinal] = true;
  }
  a.in_place = kv_lens == cached_lens || cursor_out == cursor;
  // one CTA for small steps; otherwise a token per thread on up to one CTA per
  // SM (in place: one cluster), each wide enough to scan the requests quickly
  const int64_t items = std::max(batch, max_tokens);
  const int threads = items <= 256 || (items > 2 * kTabThreads && batch <= 512) ? 256 : kTabThreads;
  int64_t ctas = 1;
  if (items > 2 * kTabThreads)
    ctas = a.in_place ? kTabCluster
                      : std::min<int64_t>((items + threads - 1) / threads, dev->num_sms);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(a.in_place && ctas > 1 ? kTabThreads : threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ctas;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.in_place && ctas > 1 ? 2 : 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, paged_tables_kernel, a), "paged tables launch");
}

extern "C" hxb_status_t hxb_kv_cache_write_paged_f16(const hxb_kv_cache_write_paged_t* args,
                                                     void* stream) {
  using namespace hxb;
  if (!args) return fail(HXB_STATUS_INVALID_ARGUMENT, "paged cache write: null arguments");
  const auto& [k_src, v_src, ld_src, slots, tokens, k_cache, v_cache, block_stride, num_blocks,
               kv_heads, block_rows, head_dim] = *args;
  hxb_status_t s = check_paged_cache("paged cache write", k_cache, v_cache, block_stride,
                                     num_blocks, kv_heads, block_rows, head_dim);
  if (s != HXB_OK) return s;
  if (tokens < 0 || tokens > INT32_MAX)
    return fail(HXB_STATUS_INVALID_ARGUMENT, "paged cache write: bad token count");
  if (tokens == 0) return HXB_OK;
  if (!k_src || !v_src || !slots)
    return fail(HXB_STATUS_INVALID_ARGUMENT, "paged cache write: null pointer");
  if (!aligned16(k_src) || !aligned16(v_src) || ld_src % 8 || ld_src < kv_heads * head_dim)
    return fail(HXB_STATUS_INVALID_ARGUMENT,
                "paged cache write: 16-byte aligned source rows that hold kv_heads * head_dim "
                "elements required");
  DeviceInfo* dev = nullptr;
  if ((s = current_device(&dev)) != HXB_OK) return s;
  PutArgs a{};
  a.k_src = static_cast<const __half*>(k_src);
  a.v_src = static_cast<const __half*>(v_src);
  a.slots = reinterpret_cast<const long long*>(slots);
  a.k_cache = static_cast<__half*>(k_cache);
  a.v_cache = static_cast<__half*>(v_cache);
  a.ld_src = ld_src;
  a.block_stride = block_stride;
  a.num_blocks = num_blocks;
  a.row_vectors = (int)(kv_heads * head_dim / 8);
  a.vectors = (long long)tokens * a.row_vectors;
  a.head_dim = (int)head_dim;
  while ((1 << a.rows_log2) < block_rows) ++a.rows_log2;
  a.status = dev->status_word;
  const long long blocks = (a.vectors + kPutThreads - 1) / kPutThreads;
  if (blocks > INT32_MAX)
    return fail(HXB_STATUS_INVALID_ARGUMENT, "paged cache write: extent too large");
  return launch_pdl(paged_write_kernel, dim3((unsigned)blocks), dim3(kPutThreads), 0,
                    static_cast<cudaStream_t>(stream), "paged cache write launch", a);
}
