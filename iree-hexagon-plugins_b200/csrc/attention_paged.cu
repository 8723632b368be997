// Grouped-query attention of a batch of requests over a paged KV cache with a
// prefix that all of them share:
//   O[t, h, :] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q[t, h] . k_j - m)
// j over the keys of the shared prefix (visible to every token) and over the
// request's own keys (causal within the request). The two key sets are
// independent softmaxes that merge exactly: with the partial results O_i and
// L_i = log2(sum 2^...) of any partition of the keys,
//   O = sum_i 2^(L_i - M) O_i / sum_i 2^(L_i - M),  M = max_i L_i.
// So the prefix is read ONCE for the batch: the rows (token, query head of the
// group) of ALL requests are packed into tiles per KV head and walk the prefix
// keys together, while each request's rows walk its own keys.
//
// Two kernels share the work (paged_work.cuh says how it is cut): the narrow one
// (attention_paged_narrow.cuh, keys on the TMEM lanes, bound by HBM) takes the
// own keys of decode batches, at most 16 rows per KV head and request, the wide
// one (attention_paged_wide.cuh, rows on the lanes, bound by the tensor core)
// those of other batches and a prefix that many rows share. A decode batch behind
// a long prefix has both at once, each on its share of the SMs (256 requests of
// 550 keys behind 4096: 115 us, one kernel after the other in the same code 143). A
// combine kernel merges what each row has. K and V blocks come through 3-D tensor
// maps, one TMA box per cache block and 64 columns, straight into the 128B-swizzled
// tile.
//
// The reference's KV-cache models attend one contiguous cache with one length
// for the batch (integration_tests/models/kv_cache.py:46-112); the shared
// prefix and the block tables have no counterpart there.
#include <math.h>

#include <algorithm>

#include "attention_paged_narrow.cuh"
#include "attention_paged_wide.cuh"
#include "runtime_common.h"

namespace hxb {
namespace {

// Whether a prefix of `blocks` key blocks that `rows` rows per KV head share goes
// to the narrow kernel, beside the requests' own keys. It reads the prefix once
// per 16 rows (from L2 after the first), 0.85 us a block and SM, the wide kernel
// takes 2.05 us per 256 rows or 1.4 for the last 128; a second kernel costs the call
// 3 us (one B200, D = 128, 8 KV heads: 64 rows on 16 blocks 23.0 us narrow, 25.9
// wide; 128 rows on 32 blocks 47.1 us narrow, 35.8 wide, with the step's tables).
// Both sides were measured at D = 128 only; D = 64 goes by the same numbers.
bool prefix_to_narrow(int64_t rows, int64_t blocks, int64_t kv_heads, int num_sms) {
  const double narrow = (double)((rows + 15) / 16) * 0.85;
  const double wide = rows <= 128 ? 1.4 : (double)((rows + 255) / 256) * 2.05;
  return (narrow - wide) * (double)(blocks * kv_heads) <= 3.0 * num_sms;
}

// What a row unit costs on top of its key blocks (Q, the first softmax without an
// overlapping product, the epilogue), in blocks.
constexpr int kWideUnitCost = 2;
constexpr int kNarrowUnitCost = 1;

// Merges the partials of every row: a block has 32 packed rows of one KV head
// (lane = row) and a group of V float4 columns per warp or, where there are rows
// enough to fill the SMs, all columns in turn; so partials, which lie row by row
// in groups of four columns, are read in whole lines, many pieces in flight at a
// time. A row has one partial per CTA that walked a part of its prefix keys or of
// its own keys; a row without any key is 0.
constexpr int kCombineThreads = 128;

template <int D, int V>
__global__ void __launch_bounds__(kCombineThreads) attention_paged_combine_kernel(const PagedArgs a) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kStep = kCombineThreads / 32 * V;  // float4 columns of a block
  const int col_blocks = gridDim.y / a.kv_heads;   // 1 or D / 4 / kStep
  const int h = blockIdx.y / col_blocks;
  const int R = a.total_q * a.group;
  const int pr = blockIdx.x * 32 + lane;
  // the lengths and tables of the call, checked once
  if (blockIdx.x == 0 && blockIdx.y == 0) {
    bool bad = false;
    for (int b = threadIdx.x; b < a.batch; b += kCombineThreads)
      bad |= a.q_start[b] < 0 || a.q_start[b + 1] < a.q_start[b] || a.q_start[b + 1] > a.total_q ||
             a.kv_lens[b] < 0 || a.kv_lens[b] > (long long)a.table_cols << a.rows_log2;
    if (bad) atomicOr(a.status, kStatusBadIndex);
  }
  if (pr >= R) return;
  const long long at = (long long)h * R + pr;
  const int2 own = a.info[0][at];
  const int2 pre = a.prefix_len > 0 ? a.info[1][at] : make_int2(0, 0);
  const int tok = pr / a.group;
  if (tok < clamp_token(a, 0) || tok >= clamp_token(a, a.batch)) return;
  const bool prefix = a.prefix_len > 0 && !(own.x & kWithPrefix);
  const int n_own = own.y & 0xffff, n_pre = prefix ? pre.y & 0xffff : 0;
  if (!prefix && n_own == 1) return;  // written by the attention kernel
  // (records left unwritten by a launch that gave up on a wait)
  auto wrong = [&](int2 info, int n) {
    const bool narrow = (info.x & kNarrowSlot) != 0;
    return n < 1 || info.x < 0 || (unsigned)info.y >> 16 >= (narrow ? 16u : 256u) ||
           (info.x & (kWithPrefix - 1)) + n > a.ctas[narrow];
  };
  if (wrong(own, n_own) || (prefix && wrong(pre, n_pre))) return;
  const int pieces = n_own + n_pre;
  // v0: this warp's first float4 column
#pragma unroll 1
  for (int v0 = blockIdx.y % col_blocks * kStep + warp * V; v0 < D / 4;
       v0 += col_blocks == 1 ? kStep : D) {
    float m = -INFINITY, sum = 0.0f;
    float acc[4 * V];
#pragma unroll
    for (int e = 0; e < 4 * V; ++e) acc[e] = 0.0f;
    constexpr int kBatch = V == 1 ? 12 : 8;
#pragma unroll 1
    for (int p0 = 0; p0 < pieces; p0 += kBatch) {
      float lse[kBatch];
      float4 x[kBatch][V];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        lse[i] = -INFINITY;
        if (p0 + i < pieces) {
          const bool set = p0 + i >= n_own;
          const int2 info = set ? pre : own;
          const int n = set ? n_pre : n_own, p = set ? p0 + i - n_own : p0 + i;
          const float *src, *stat;
          int pitch;
          if (n == 1) {
            src = a.whole_o[set] + ((long long)h * (D / 4) * R + pr) * 4;
            stat = a.whole_lse[set] + at;
            pitch = R;
          } else {
            const bool narrow = (info.x & kNarrowSlot) != 0;
            pitch = narrow ? kNarrowRows : 256;
            const int cta = (info.x & (kWithPrefix - 1)) + p;
            const int row = (2 * cta + (p == 0)) * pitch + (info.y >> 16);
            stat = a.cut_lse[narrow] + row;
            src = a.cut_o[narrow] + ((long long)(2 * cta + (p == 0)) * (D / 4) * pitch + (info.y >> 16)) * 4;
          }
          lse[i] = *stat;
#pragma unroll
          for (int v = 0; v < V; ++v)
            x[i][v] = *reinterpret_cast<const float4*>(src + (long long)(v0 + v) * pitch * 4);
        }
      }
      float m_new = m;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) m_new = fmaxf(m_new, lse[i]);
      if (m != -INFINITY) {  // (nothing visible so far: sum and acc are 0, or NaN)
        const float scale = ex2_approx(m - m_new);
        sum *= scale;
#pragma unroll
        for (int e = 0; e < 4 * V; ++e) acc[e] *= scale;
      }
      m = m_new;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (lse[i] == -INFINITY) continue;
        const float w = ex2_approx(lse[i] - m);
        sum += w;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          acc[4 * v + 0] = fmaf(w, x[i][v].x, acc[4 * v + 0]);
          acc[4 * v + 1] = fmaf(w, x[i][v].y, acc[4 * v + 1]);
          acc[4 * v + 2] = fmaf(w, x[i][v].z, acc[4 * v + 2]);
          acc[4 * v + 3] = fmaf(w, x[i][v].w, acc[4 * v + 3]);
        }
      }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint32_t o[2 * V];
#pragma unroll
    for (int e = 0; e < 2 * V; ++e) o[e] = pack_half2(acc[2 * e] * inv, acc[2 * e + 1] * inv);
    __half* to = a.O + tok * a.ldo +
                 ((long long)h * a.group + pr - (long long)tok * a.group) * D + v0 * 4;
    if constexpr (V == 1) *reinterpret_cast<uint2*>(to) = make_uint2(o[0], o[1]);
    else *reinterpret_cast<uint4*>(to) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// Workspace: what the partials of a call take, in this order.
struct PagedLayout {
  size_t cut_o[2], cut_lse[2], whole_o[2], whole_lse[2], info[2], total;
};

PagedLayout paged_layout(int64_t rows, int64_t D, bool prefix, int num_sms) {
  PagedLayout l{};
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off += (bytes + 255) & ~size_t(255);
    return at;
  };
  for (int k = 0; k < 2; ++k) {
    const size_t cut = (size_t)num_sms * (k ? 2 * 2 * kNarrowRows : 2 * 256);
    l.cut_o[k] = take(cut * D * sizeof(float));
    l.cut_lse[k] = take(cut * sizeof(float));
    l.whole_o[k] = take(prefix ? (size_t)rows * D * sizeof(float) : 0);
    l.whole_lse[k] = take(prefix ? (size_t)rows * sizeof(float) : 0);
    l.info[k] = take(k == 0 || prefix ? (size_t)rows * sizeof(int2) : 0);
  }
  l.total = off;
  return l;
}

template <int D>
hxb_status_t configure_paged(const DeviceInfo& dev) {
  static bool configured[64] = {};
  if (configured[dev.ordinal]) return HXB_OK;
  // the wide kernel's register split assumes this launch count (see attention.cu)
  cudaFuncAttributes fa{};
  cudaError_t e = cudaFuncGetAttributes(&fa, attention_paged_wide_kernel<D>);
  if (e != cudaSuccess) return cuda_status(e, "cudaFuncGetAttributes(paged attention)");
  if (fa.numRegs != kPagedRegsLaunch)
    return fail(HXB_STATUS_UNSUPPORTED, "paged attention kernel built with %d registers per "
                "thread, its register split needs %d", fa.numRegs, kPagedRegsLaunch);
  e = cudaFuncSetAttribute(attention_paged_wide_kernel<D>,
                           cudaFuncAttributeMaxDynamicSharedMemorySize, WideSmem<D>::kAlloc);
  for (auto kernel : {attention_paged_narrow_kernel<D, 4>, attention_paged_narrow_kernel<D, 8>,
                      attention_paged_narrow_kernel<D, 16>}) {
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               NarrowSmem<D>::kAlloc);
    // all of the unified L1 as shared memory: two CTAs per SM
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                               cudaSharedmemCarveoutMaxShared);
  }
  if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(paged attention)");
  configured[dev.ordinal] = true;
  return HXB_OK;
}

template <int D>
hxb_status_t launch_paged(const CUtensorMap& tmQ, const CUtensorMap& tmK, const CUtensorMap& tmV,
                          PagedArgs a, int64_t max_q_len, const DeviceInfo& dev,
                          cudaStream_t stream) {
  hxb_status_t s = configure_paged<D>(dev);
  if (s != HXB_OK) return s;
  // Batches whose requests are expected to have at most 16 rows per KV head go to
  // the narrow kernel, others to the wide one (its solo mode is as near to HBM
  // on a long request). So one longer request takes the whole batch there: a second
  // launch for the short requests of a mixed batch cost more than it saved when the
  // two kernels ran one after the other, and has not been measured beside the other.
  const int narrow_tok = kNarrowRows / a.group;
  const bool narrow = narrow_tok > 0 && max_q_len <= narrow_tok;
  const bool prefix = a.prefix_len > 0;
  const bool narrow_prefix =
      narrow && prefix && prefix_to_narrow((int64_t)a.total_q * a.group,
                                           (a.prefix_len + kBN - 1) / kBN, a.kv_heads, dev.num_sms);
  // rows of a unit of the narrow kernel: what the largest request, and a prefix,
  // can fill
  int64_t rows = std::max<int64_t>(1, max_q_len) * a.group;
  if (narrow_prefix) rows = std::max(rows, std::min<int64_t>((int64_t)a.total_q * a.group, kNarrowRows));
  const int nr = rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
  const bool wide = !narrow || (prefix && !narrow_prefix);
  if (wide) {
    PagedArgs w = a;
    w.unit_tok = 2 * a.tile_tok;
    w.unit_cost = kWideUnitCost;
    w.requests_here = !narrow;
    w.prefix_here = prefix;
    w.fat_tok = !narrow && prefix ? a.tile_tok : 0;
    w.beside = narrow;
    w.other_tok = nr / a.group;
    w.other_cost = kNarrowUnitCost;
    // Beside the narrow kernel in clusters of two CTAs, which share a TPC: the CTAs
    // without work leave both SMs of one, and a wide CTA that has a narrow one's
    // loads on the other SM of its TPC takes a third longer.
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)dev.num_sms);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = WideSmem<D>::kAlloc;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = narrow && dev.num_sms % 2 == 0 ? 2 : 1;
    s = cuda_status(cudaLaunchKernelEx(&cfg, attention_paged_wide_kernel<D>, tmQ, tmK, tmV, w),
                    "paged attention launch");
    if (s != HXB_OK) return s;
  }
  if (narrow) {
    PagedArgs n = a;
    n.unit_tok = nr / a.group;
    n.unit_cost = kNarrowUnitCost;
    n.requests_here = 1;
    n.prefix_here = narrow_prefix;
    n.beside = wide;
    n.other_tok = 2 * a.tile_tok;
    n.other_cost = kWideUnitCost;
    const auto kernel = nr == 4   ? attention_paged_narrow_kernel<D, 4>
                        : nr == 8 ? attention_paged_narrow_kernel<D, 8>
                                  : attention_paged_narrow_kernel<D, 16>;
    int ctas = 2 * dev.num_sms;
    if (wide) {
      // Not many more than will have work (the lengths are at most what the table
      // holds): those that find no SM beside the wide kernel start behind it.
      const int64_t units = ((int64_t)a.total_q + n.other_tok - 1) / n.other_tok * a.kv_heads;
      const int64_t work = (a.prefix_len + kBN - 1) / kBN + n.other_cost;
      const float own = (float)a.kv_heads *
                        (float)std::min<int64_t>(a.total_q, a.batch + a.total_q / n.unit_tok) *
                        (float)(((int64_t)a.table_cols << a.rows_log2) / kBN + 1 + n.unit_cost);
      ctas = ctas_beside(a, (int)units, wide_share(a, (int)units, (int)work, own));
    }
    s = launch_pdl(kernel, dim3((unsigned)ctas), dim3(kNarThreads),
                   NarrowSmem<D>::kAlloc, stream, "paged attention launch", tmK, tmV, n);
    if (s != HXB_OK) return s;
  }
  // few rows: many blocks of few columns, to have the partials of a row in flight
  // at once; many: all columns in a block, so that rows without work are few blocks
  const int64_t chunks = ((int64_t)a.total_q * a.group + 31) / 32, units = chunks * a.kv_heads;
  const bool few = 2 * units < dev.num_sms;
  const int col_blocks = units >= 4 * dev.num_sms ? 1 : D / (few ? 16 : 32);
  const auto combine = few ? attention_paged_combine_kernel<D, 1> : attention_paged_combine_kernel<D, 2>;
  return launch_pdl(combine, dim3((unsigned)chunks, (unsigned)(a.kv_heads * col_blocks)),
                    dim3(kCombineThreads), 0, stream, "paged attention combine launch", a);
}

}  // namespace
}  // namespace hxb

using hxb::fail;

extern "C" size_t hxb_attention_paged_workspace_bytes(int64_t total_q, int64_t q_heads,
                                                      int64_t head_dim, int64_t prefix_len) {
  using namespace hxb;
  DeviceInfo* dev = nullptr;
  if (total_q < 1 || q_heads < 1 || total_q > INT32_MAX / q_heads ||
      (head_dim != 64 && head_dim != 128) || prefix_len < 0 || current_device(&dev) != HXB_OK)
    return 0;
  return paged_layout(total_q * q_heads, head_dim, prefix_len > 0, dev->num_sms).total;
}

extern "C" hxb_status_t hxb_attention_paged_f16(const hxb_attention_paged_t* args, void* stream) {
  using namespace hxb;
  if (!args) return fail(HXB_STATUS_INVALID_ARGUMENT, "paged attention: null arguments");
  const auto& [Q, ldq, O, ldo, q_start, kv_lens, batch, total_q, max_q_len, k_cache, v_cache,
               block_stride, num_blocks, block_rows, block_table, table_ld, table_cols,
               prefix_table, prefix_len, q_heads, kv_heads, head_dim, scale, causal, workspace,
               workspace_bytes] = *args;
  if (head_dim != 64 && head_dim != 128)
    return fail(HXB_STATUS_UNSUPPORTED, "paged attention: head dim %lld not supported (64 or 128)",
                (long long)head_dim);
  hxb_status_t s = check_paged_cache("paged attention", k_cache, v_cache, block_stride, num_blocks,
                                     kv_heads, block_rows, head_dim);
  if (s != HXB_OK) return s;
  if (batch < 1 || batch > (1 << 20) || total_q < 0 || max_q_len < 0 || q_heads < 1 ||
      q_heads % kv_heads)
    return fail(HXB_STATUS_INVALID_ARGUMENT,
                "paged attention: batch >= 1 and q_heads a multiple of kv_heads required");
  const int64_t group = q_heads / kv_heads;
  if (group > kBM)
    return fail(HXB_STATUS_UNSUPPORTED, "paged attention: %lld query heads per KV head (at most %d)",
                (long long)group, kBM);
  if (kv_heads * (head_dim / 16) > 65535 || total_q > INT32_MAX / q_heads || table_cols < 1 ||
      table_ld < table_cols || table_cols > INT32_MAX / 2 / block_rows || prefix_len < 0 || prefix_len > INT32_MAX / 2)
    return fail(HXB_STATUS_INVALID_ARGUMENT, "paged attention: bad extents");
  if (!(scale > 0.0f) || !isfinite(scale))
    return fail(HXB_STATUS_INVALID_ARGUMENT, "paged attention: scale must be finite and > 0");
  if (total_q == 0) return HXB_OK;
  if (!Q || !O || !q_start || !kv_lens || !block_table || (prefix_len && !prefix_table))
    return fail(HXB_STATUS_INVALID_ARGUMENT, "paged attention: null pointer");
  if (!aligned16(Q) || !aligned16(O) || ldq % 8 || ldo % 8 || ldq < q_heads * head_dim ||
      ldo < q_heads * head_dim || ldq > ((int64_t)1 << 38))
    return fail(HXB_STATUS_INVALID_ARGUMENT,
                "paged attention: Q and O need 16-byte aligned rows that hold q_heads * head_dim "
                "elements");
  DeviceInfo* dev = nullptr;
  if ((s = current_device(&dev)) != HXB_OK) return s;
  const PagedLayout l = paged_layout(total_q * q_heads, head_dim, prefix_len > 0, dev->num_sms);
  if (!workspace || !aligned16(workspace) || workspace_bytes < l.total)
    return fail(HXB_STATUS_INVALID_ARGUMENT,
                "paged attention: a 16-byte aligned workspace of %zu bytes required", l.total);

  // Tokens per Q box of the wide kernel: the fewest whose rows are whole 8-row
  // swizzle groups and at least 32, so that a short tile loads few rows in few
  // boxes; one box of the whole tile where that is more than half a tile.
  int64_t box_tok = 1;
  while (box_tok * group % 8) ++box_tok;
  while (box_tok * group < 32) box_tok *= 2;
  int64_t tile_tok = kBM / (box_tok * group) * box_tok;
  if (box_tok * group > kBM / 2) box_tok = tile_tok = kBM / group;

  CUtensorMap tmQ, tmK, tmV;
  {
    const uint64_t dims[3] = {(uint64_t)head_dim, (uint64_t)q_heads, (uint64_t)total_q};
    const uint64_t strides[2] = {(uint64_t)head_dim * 2, (uint64_t)ldq * 2};
    const uint32_t box[3] = {64, (uint32_t)group, (uint32_t)box_tok};
    s = encode_tensor_map(&tmQ, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, Q, dims, strides, box,
                          CU_TENSOR_MAP_SWIZZLE_128B);
    if (s != HXB_OK) return s;
  }
  const uint64_t dims[3] = {(uint64_t)head_dim, (uint64_t)(kv_heads * block_rows),
                            (uint64_t)num_blocks};
  const uint64_t strides[2] = {(uint64_t)head_dim * 2, (uint64_t)block_stride * 2};
  const uint32_t box[3] = {64, (uint32_t)std::min<int64_t>(block_rows, kBN), 1};
  if ((s = encode_tensor_map(&tmK, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, k_cache, dims, strides, box,
                             CU_TENSOR_MAP_SWIZZLE_128B)) != HXB_OK)
    return s;
  if ((s = encode_tensor_map(&tmV, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, v_cache, dims, strides, box,
                             CU_TENSOR_MAP_SWIZZLE_128B)) != HXB_OK)
    return s;

  PagedArgs a{};
  a.q_start = q_start;
  a.kv_lens = kv_lens;
  a.block_table = block_table;
  a.prefix_table = prefix_table;
  a.Q = static_cast<const __half*>(Q);
  a.O = static_cast<__half*>(O);
  a.ldq = ldq;
  a.ldo = ldo;
  a.table_ld = table_ld;
  a.total_q = (int)total_q;
  a.batch = (int)batch;
  a.q_heads = (int)q_heads;
  a.kv_heads = (int)kv_heads;
  a.group = (int)group;
  a.tile_tok = (int)tile_tok;
  a.box_tok = (int)box_tok;
  a.table_cols = (int)table_cols;
  a.num_blocks = (int)num_blocks;
  while ((1 << a.rows_log2) < block_rows) ++a.rows_log2;
  a.prefix_len = (int)prefix_len;
  a.causal = causal ? 1 : 0;
  a.ctas[0] = dev->num_sms;
  a.ctas[1] = 2 * dev->num_sms;
  a.c = (float)((double)scale * 1.4426950408889634);  // scale * log2(e)
  char* ws = static_cast<char*>(workspace);
  for (int k = 0; k < 2; ++k) {
    a.cut_o[k] = reinterpret_cast<float*>(ws + l.cut_o[k]);
    a.cut_lse[k] = reinterpret_cast<float*>(ws + l.cut_lse[k]);
    a.whole_o[k] = reinterpret_cast<float*>(ws + l.whole_o[k]);
    a.whole_lse[k] = reinterpret_cast<float*>(ws + l.whole_lse[k]);
    a.info[k] = reinterpret_cast<int2*>(ws + l.info[k]);
  }
  a.status = dev->status_word;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t most = std::min(max_q_len, total_q);  // (no request has more tokens)
  return head_dim == 64 ? launch_paged<64>(tmQ, tmK, tmV, a, most, *dev, st)
                        : launch_paged<128>(tmQ, tmK, tmV, a, most, *dev, st);
}
