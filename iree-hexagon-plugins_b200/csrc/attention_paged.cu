// Grouped-query attention of a batch of requests over a paged KV cache with a
// prefix that all of them share:
//   O[t, h, :] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q[t, h] . k_j - m)
// j over the keys of the shared prefix (visible to every token) and over the
// request's own keys (causal within the request). The two key sets are
// independent softmaxes that merge exactly: with the partial results O_i and
// L_i = log2(sum 2^...) of any partition of the keys,
//   O = sum_i 2^(L_i - M) O_i / sum_i 2^(L_i - M),  M = max_i L_i.
// So the prefix is read ONCE for the batch: the rows (token, query head of the
// group) of ALL requests are packed into 128-row tiles per KV head and walk
// the prefix keys together, while each request's rows walk its own keys.
//
// What bounds it: a decode batch reads K and V (HBM); many rows per KV head
// (a large batch or prompt chunks) are bound by the tensor core and the
// exponentials, as in attention.cu, whose tile scheme this kernel uses:
//   * S = Q K^T (tcgen05, operands in shared memory) lands in TMEM, a softmax
//     warpgroup (thread = row) writes P = 2^(S c - m) as f16 over S, and
//     O += P V accumulates in TMEM; the maximum moves only when it grows by
//     more than 2^8.
//   * a row unit of more than 128 rows keeps two tiles in flight ("pair": both
//     tiles share every K/V block); a unit of at most 128 rows gives the two
//     softmax warpgroups alternate key blocks of the SAME tile ("solo") and
//     merges the two accumulators in the epilogue, so that short row units do
//     not wait for one softmax chain per block.
//
// Work split: one persistent CTA per SM. All (key set, KV head, row unit)
// segments are laid end to end in units of one 128-key block, and CTA i takes
// units [T i / G, T (i+1) / G): equal shares whatever the lengths, with the
// lengths read on the GPU (a captured graph follows them). A segment cut
// between CTAs leaves one partial per CTA; a combine kernel merges what each
// row has. K and V pages come through 3-D tensor maps, one TMA box per page
// and 64 columns, straight into the 128B-swizzled tile.
//
// The reference's KV-cache models attend one contiguous cache with one length
// for the batch (integration_tests/models/kv_cache.py:46-112); the shared
// prefix and the block tables have no counterpart there.
#include <math.h>

#include <algorithm>

#include "runtime_common.h"
#include "sm100.cuh"

namespace hxb {
namespace {

constexpr int kBM = 128;  // rows per tile
constexpr int kBN = 128;  // keys per block
constexpr int kBoxBytes = 128 * 64 * 2;  // 128 rows x 64 f16
constexpr int kThreads = 384;
constexpr int kItems = 4;  // work items announced ahead of the roles
constexpr float kMoveLog2 = 8.0f;
// Register split of the 384 launch threads, as in attention.cu.
constexpr int kPagedRegsLaunch = 168;
constexpr int kPagedRegsControl = 104;
constexpr int kPagedRegsSoftmax = 200;
static_assert(kPagedRegsControl * 128 + kPagedRegsSoftmax * (kThreads - 128) <=
                  kPagedRegsLaunch * kThreads,
              "register split exceeds the launch allocation");

// One piece of work: `blocks` key blocks from block j0 of a segment.
struct Item {
  int request;  // -1: the shared prefix; kEnd: no more work
  int head;     // KV head
  int tok0;     // first token of the row unit
  int ntok;     // its tokens
  int j0, blocks;
  int keys;     // keys of the segment's key set
  int pos0;     // last key that token tok0 sees (causal), else INT_MAX / 2
  int slot;     // partial slot of a cut segment, -1: the segment is whole here
  int first, pieces;  // a cut segment: slot of its first piece, and how many
};
constexpr int kEnd = -2;

template <int D>
struct PagedSmem {
  static_assert(D == 64 || D == 128, "head dimension 64 or 128");
  static constexpr int kBoxes = D / 64;
  static constexpr int kTileBytes = 128 * D * 2;
  static constexpr int kSlots = D == 64 ? 8 : 4;
  static constexpr int kOffQ = 0;
  static constexpr int kOffKV = kOffQ + 2 * kTileBytes;
  static constexpr int kOffML = kOffKV + kSlots * kTileBytes;  // [2][2][128] float2
  static constexpr int kOffItems = kOffML + 4 * 128 * 8;
  static constexpr int kOffBar = kOffItems + kItems * 64;
  // q_full, q_empty, kv_full[], kv_empty[], s_full[2], p_full[2], o_full,
  // o_free, v_need, v_ready, xsync, item_full[], item_empty[], drain
  static constexpr int kNumBars = 2 + 2 * kSlots + 4 + 5 + 2 * kItems + 1;
  static constexpr int kOffMisc = kOffBar + kNumBars * 8;
  static constexpr int kBytes = kOffMisc + 64 + 2 * (kThreads / 32) * 8;
  static constexpr int kAlloc = kBytes + 1024;
};
static_assert(sizeof(Item) <= 64, "item record");

struct PagedArgs {
  const int* q_start;
  const int* kv_lens;
  const int* block_table;
  const int* prefix_table;
  __half* O;
  long long ldo, table_ld;
  int total_q, batch, q_heads, kv_heads, group;
  int tile_tok;  // tokens per 128-row tile
  int box_tok;   // tokens per Q box
  int table_cols, num_blocks, rows_log2;
  int prefix_len;
  int causal;
  int ctas;
  float c;  // scale * log2(e)
  // partials: cut segments [2 * CTAs][256 rows], whole segments per row
  float* cut_o;
  float* cut_lse;
  float* whole_o[2];  // own keys, prefix
  float* whole_lse[2];
  int2* info[2];
  int* status;
};

__device__ __forceinline__ int clamp_token(const PagedArgs& a, int b) {
  return min(max(a.q_start[b], 0), a.total_q);
}

// One key set of one request (or of the prefix): its tokens, keys and the
// blocks that its row units visit.
struct Segment {
  int tok, n, keys;
  int units;       // row units
  long long work;  // blocks of one KV head over all row units
};

__device__ __forceinline__ int unit_blocks(const PagedArgs& a, const Segment& s, int u,
                                           bool causal) {
  int visible = s.keys;
  if (causal) {
    const int last = min((u + 1) * 2 * a.tile_tok, s.n) - 1;
    visible = max(0, min(visible, s.keys - s.n + last + 1));
  }
  return max(1, (visible + kBN - 1) / kBN);  // an empty unit still writes its rows
}

__device__ __forceinline__ Segment own_segment(const PagedArgs& a, int b) {
  Segment s;
  s.tok = clamp_token(a, b);
  s.n = max(clamp_token(a, b + 1) - s.tok, 0);
  s.keys = (int)min((long long)max(a.kv_lens[b], 0), (long long)a.table_cols << a.rows_log2);
  s.units = (s.n + 2 * a.tile_tok - 1) / (2 * a.tile_tok);
  s.work = 0;
  for (int u = 0; u < s.units; ++u) s.work += unit_blocks(a, s, u, a.causal);
  return s;
}

__device__ __forceinline__ Segment prefix_segment(const PagedArgs& a) {
  Segment s;
  s.tok = clamp_token(a, 0);
  s.n = a.prefix_len > 0 ? max(clamp_token(a, a.batch) - s.tok, 0) : 0;
  s.keys = a.prefix_len;
  s.units = (s.n + 2 * a.tile_tok - 1) / (2 * a.tile_tok);
  s.work = (long long)s.units * ((s.keys + kBN - 1) / kBN);
  return s;
}

__device__ __forceinline__ uint64_t kmajor_desc(uint32_t base) {
  return make_smem_desc(base, 16, 1024, kLayoutSwizzle128);
}
__device__ __forceinline__ uint64_t vmajor_desc(uint32_t base) {
  return make_smem_desc(base, kBoxBytes, 1024, kLayoutSwizzle128);
}
// K-major 16-element K step kk of a tile of [128 x 64] boxes, in descriptor
// address units.
__device__ __forceinline__ constexpr uint64_t kstep(int kk) {
  return (uint64_t)(((kk >> 2) * kBoxBytes + (kk & 3) * 32) >> 4);
}

// Position in a ring of N slots, counted in uses.
template <int N>
struct Ring {
  uint32_t n = 0;
  __device__ __forceinline__ int slot() const { return n % N; }
  __device__ __forceinline__ uint32_t parity() const { return (n / N) & 1; }
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    attention_paged_kernel(const __grid_constant__ CUtensorMap tmQ,
                           const __grid_constant__ CUtensorMap tmK,
                           const __grid_constant__ CUtensorMap tmV, const PagedArgs args) {
  using L = PagedSmem<D>;
  constexpr int kSlots = L::kSlots;
  constexpr int kTileBytes = L::kTileBytes;
  constexpr uint32_t kIdescQK = make_idesc_f16(kBM, kBN, 0, 0);
  constexpr uint32_t kIdescPV = make_idesc_f16(kBM, D, 0, 1);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
  uint64_t* q_empty = q_full + 1;
  uint64_t* kv_full = q_empty + 1;
  uint64_t* kv_empty = kv_full + kSlots;
  uint64_t* s_full = kv_empty + kSlots;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* o_free = o_full + 1;
  uint64_t* v_need = o_free + 1;
  uint64_t* v_ready = v_need + 1;
  uint64_t* xsync = v_ready + 1;
  uint64_t* item_full = xsync + 1;
  uint64_t* item_empty = item_full + kItems;
  uint64_t* drain = item_empty + kItems;
  Item* items = reinterpret_cast<Item*>(smem + L::kOffItems);
  float2* ml = reinterpret_cast<float2*>(smem + L::kOffML);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 4);
  int* start_b = reinterpret_cast<int*>(smem + L::kOffMisc + 8);
  long long* start_off = reinterpret_cast<long long*>(smem + L::kOffMisc + 16);
  long long* warp_sum = reinterpret_cast<long long*>(smem + L::kOffMisc + 64);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const FailState fs{abort_flag, args.status};

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], kBM);
    }
    mbar_init(o_full, 1);
    mbar_init(o_free, 2 * kBM);
    mbar_init(v_need, 1);
    mbar_init(v_ready, 1);
    mbar_init(xsync, 2 * kBM);
    for (int s = 0; s < kItems; ++s) {
      mbar_init(&item_full[s], 1);
      mbar_init(&item_empty[s], 3 + 8);  // producer, issuer, tail warp, 8 softmax warps
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    *start_b = -1;
    *start_off = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  pdl_trigger();
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;

  // ------------------------------------------------- this CTA's share of work
  // Every thread sums the work of a run of requests; a block scan gives the
  // total and the thread that holds the CTA's first unit finds its request.
  const Segment pre = prefix_segment(args);
  const int per = (args.batch + kThreads - 1) / kThreads;
  const int b0 = min((int)threadIdx.x * per, args.batch), b1 = min(b0 + per, args.batch);
  long long mine = 0;
  bool bad = false;
  for (int b = b0; b < b1; ++b) {
    mine += own_segment(args, b).work * args.kv_heads;
    bad |= args.q_start[b] < 0 || args.q_start[b + 1] < args.q_start[b] ||
           args.q_start[b + 1] > args.total_q || args.kv_lens[b] < 0 ||
           args.kv_lens[b] > ((long long)args.table_cols << args.rows_log2);
  }
  if (bad && blockIdx.x == 0) atomicOr(args.status, kStatusBadIndex);
  long long scan = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += v;
  }
  if (lane == 31) warp_sum[warp] = scan;
  __syncthreads();
  const long long pre_work = pre.work * args.kv_heads;
  long long total = pre_work, base = pre_work;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w == warp) base = total;
    total += warp_sum[w];
  }
  base += scan - mine;
  // (at most one CTA per unit, so that every CTA of a cut segment has a piece)
  const long long G = max(1ll, min((long long)gridDim.x, total));
  const long long lo = blockIdx.x < G ? total * blockIdx.x / G : 0;
  const long long hi = blockIdx.x < G ? total * (blockIdx.x + 1) / G : 0;
  if (lo < hi) {
    if (lo >= base && lo < base + mine) {
      long long at = base;
      for (int b = b0; b < b1; ++b) {
        const long long w = own_segment(args, b).work * args.kv_heads;
        if (lo < at + w) {
          *start_b = b;
          *start_off = lo - at;
          break;
        }
        at += w;
      }
    } else if (threadIdx.x == 0 && lo < pre_work) {
      *start_off = lo;
    }
  }
  __syncthreads();

  // Reads the next item; false on failure.
  Ring<kItems> it;
  auto next_item = [&](Item& item) -> bool {
    const bool ok = mbar_wait(&item_full[it.slot()], it.parity(), fs);
    if (!__all_sync(0xffffffffu, ok)) return false;
    item = items[it.slot()];
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[it.slot()]);
    ++it.n;
    return item.request != kEnd;
  };
  // Rows of the item's last key block that exist; a block with fewer than 128
  // gets the others of its V tile zeroed (their P is 0, but 0 * NaN is not).
  auto tail_rows = [&](const Item& item) { return item.keys - (item.j0 + item.blocks - 1) * kBN; };

  if (warp < 4) {
    reg_dealloc<kPagedRegsControl>();
    if (warp == 0) {
      // -------------------------------------------------------- TMA producer
      Ring<kSlots> ring;
      uint32_t q_items = 0;
      bool ok = true;
      const int page_rows = min(1 << args.rows_log2, kBN);  // rows per box
      const int boxes = kBN / page_rows * L::kBoxes;        // boxes per tile (<= 16)
      const int my_row = lane / L::kBoxes * page_rows, my_half = lane % L::kBoxes;
      Item item;
      while (ok && next_item(item)) {
        if (item.blocks == 0) continue;
        const int* table = item.request < 0 ? args.prefix_table
                                            : args.block_table + (long long)item.request * args.table_ld;
        const int nt = item.ntok > args.tile_tok ? 2 : 1;
        const int la = nt == 2 ? 1 : 2;  // K blocks ahead of the V block
        // one K or V tile: this lane's page and rows of key block j
        auto load_tile = [&](int which, int j) -> bool {
          const int row = (item.j0 + j) * kBN + my_row;
          int page = args.num_blocks;  // out of range: the box is filled with zeros
          if (lane < boxes && row < item.keys) {
            page = table[row >> args.rows_log2];
            if (page < 0 || page >= args.num_blocks) {
              if (which == 0) atomicOr(args.status, kStatusBadIndex);
              page = args.num_blocks;
            }
          }
          const int slot = ring.slot();
          if (!__all_sync(0xffffffffu, mbar_wait(&kv_empty[slot], ring.parity() ^ 1, fs)))
            return false;
          if (lane == 0) mbar_arrive_expect_tx(&kv_full[slot], kTileBytes);
          __syncwarp();
          if (lane < boxes)
            tma_load_3d(smem + L::kOffKV + slot * kTileBytes + my_half * kBoxBytes + my_row * 128,
                        which ? &tmV : &tmK, &kv_full[slot], 64 * my_half,
                        (item.head << args.rows_log2) + (row & ((1 << args.rows_log2) - 1)), page);
          ++ring.n;
          return true;
        };
        // Q of the row unit
        if (!__all_sync(0xffffffffu, mbar_wait(q_empty, (q_items & 1) ^ 1, fs))) { ok = false; break; }
        ++q_items;
        // (a second tile begins where the first one's boxes end: tile_tok is a
        // multiple of box_tok)
        const int tile_boxes = args.tile_tok / args.box_tok;
        const int q_boxes = (item.ntok + args.box_tok - 1) / args.box_tok;
        const int box_bytes = args.box_tok * args.group * 128;
        if (lane == 0)
          mbar_arrive_expect_tx(q_full, q_boxes * L::kBoxes * box_bytes);
        __syncwarp();
        for (int i = lane; i < q_boxes * L::kBoxes; i += 32) {
          const int half = i % L::kBoxes, q = i / L::kBoxes;
          const int t = q >= tile_boxes, bx = q - t * tile_boxes;
          tma_load_3d(smem + L::kOffQ + t * kTileBytes + half * kBoxBytes + bx * box_bytes, &tmQ,
                      q_full, 64 * half, item.head * args.group,
                      item.tok0 + q * args.box_tok);
        }
        for (int j = 0; j < min(la, item.blocks) && ok; ++j) ok = load_tile(0, j);
        for (int j = 0; j < item.blocks && ok; ++j) {
          ok = load_tile(1, j);
          if (ok && j + la < item.blocks) ok = load_tile(0, j + la);
        }
      }
      // bounded wait for the copies still landing (complete on the normal path)
      if (lane == 0) {
        if (q_items) {
          const unsigned long long t0 = globaltimer_ns();
          while (!mbar_try_wait(q_full, (q_items - 1) & 1) && globaltimer_ns() - t0 < kWaitLimitNs) {
          }
        }
        const uint32_t issued = ring.n;
        for (uint32_t i = 1; i <= min(issued, (uint32_t)kSlots); ++i) {
          ring.n = issued - i;
          const unsigned long long t1 = globaltimer_ns();
          while (!mbar_try_wait(&kv_full[ring.slot()], ring.parity()) &&
                 globaltimer_ns() - t1 < kWaitLimitNs) {
          }
        }
      }
    } else if (warp == 1) {
      // -------------------------------------------------------- MMA issuer
      Ring<kSlots> ring;
      uint32_t q_items = 0, fixes = 0;
      uint32_t p_par = 0;  // bit t: parity of p_full[t]'s next phase
      bool ok = true, issued_any = false;
      const uint64_t q_desc = kmajor_desc(smem_u32(smem + L::kOffQ));
      const uint64_t k_desc = kmajor_desc(smem_u32(smem + L::kOffKV));
      const uint64_t v_desc = vmajor_desc(smem_u32(smem + L::kOffKV));
      constexpr uint64_t kTileStep = kTileBytes >> 4;
      Item item;
      while (ok && next_item(item)) {
        if (item.blocks == 0) continue;
        if (lane == 0) {
          ok = mbar_wait(q_full, q_items & 1, fs);
          const bool pair = item.ntok > args.tile_tok;
          const int nb = item.blocks;
          const bool tail = tail_rows(item) < kBN;
          auto wait_tile = [&]() -> bool {
            const bool r = mbar_wait(&kv_full[ring.slot()], ring.parity(), fs);
            tc_fence_after();
            return r;
          };
          auto issue_s = [&](int t, int q, int slot) {
            const uint64_t kd = k_desc + slot * kTileStep;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              umma_f16_ss(tmem_base + t * 128, q_desc + q * kTileStep + kstep(kk), kd + kstep(kk),
                          kIdescQK, kk != 0);
            umma_commit(&s_full[t]);
            issued_any = true;
          };
          auto issue_pv = [&](int t, int slot, bool fresh) {
            const uint64_t vd = v_desc + slot * kTileStep;
#pragma unroll
            for (int kk = 0; kk < kBN / 16; ++kk)
              umma_f16_ts(tmem_base + 256 + t * D, tmem_base + t * 128 + 64 + kk * 8,
                          vd + (uint64_t)(kk * 16 * 128 >> 4), kIdescPV, !fresh || kk != 0);
          };
          auto wait_p = [&](int t) -> bool {
            const bool r = mbar_wait(&p_full[t], (p_par >> t) & 1, fs);
            p_par ^= 1u << t;
            tc_fence_after();
            return r;
          };
          auto wait_fix = [&]() -> bool { return mbar_wait(v_ready, fixes++ & 1, fs); };
          const int la = pair ? 1 : 2;
          // S of the first block(s)
          for (int j = 0; j < min(la, nb) && ok; ++j) {
            if (!(ok = wait_tile())) break;
            const int slot = ring.slot();
            if (pair) {
              issue_s(0, 0, slot);
              issue_s(1, 1, slot);
            } else {
              issue_s(j, 0, slot);
            }
            umma_commit(&kv_empty[slot]);
            ++ring.n;
          }
          if (ok && nb <= la) umma_commit(q_empty);
          for (int j = 0; j < nb && ok; ++j) {
            const int vslot = ring.slot();
            if (!(ok = wait_tile())) break;
            ++ring.n;
            const bool fix = tail && j == nb - 1;
            if (fix) mbar_arrive(v_need);  // (zeroed while the softmax runs)
            // both warpgroups have read the previous item's accumulators
            if (j == 0 && q_items && !(ok = mbar_wait(o_free, (q_items & 1) ^ 1, fs))) break;
            const bool more = j + la < nb;
            const int kslot = ring.slot();
            if (pair) {
              if (more && !(ok = wait_tile())) break;
              if (!(ok = wait_p(0))) break;
              if (fix && !(ok = wait_fix())) break;
              issue_pv(0, vslot, j == 0);
              if (more) issue_s(0, 0, kslot);
              if (!(ok = wait_p(1))) break;
              issue_pv(1, vslot, j == 0);
              umma_commit(&kv_empty[vslot]);
              if (more) issue_s(1, 1, kslot);
            } else {
              const int t = j & 1;
              if (!(ok = wait_p(t))) break;
              if (fix && !(ok = wait_fix())) break;
              issue_pv(t, vslot, j < 2);
              umma_commit(&kv_empty[vslot]);
              if (more) {
                if (!(ok = wait_tile())) break;
                issue_s(t, 0, kslot);
              }
            }
            if (more) {
              umma_commit(&kv_empty[kslot]);
              ++ring.n;
              if (j + la == nb - 1) umma_commit(q_empty);
            }
          }
          if (ok) umma_commit(o_full);
        }
        ++q_items;
        ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
      }
      if (lane == 0 && issued_any) {
        // (complete already on the normal path)
        umma_commit(drain);
        const unsigned long long t0 = globaltimer_ns();
        while (!mbar_try_wait(drain, 0) && globaltimer_ns() - t0 < kWaitLimitNs) {
        }
      }
    } else if (warp == 2) {
      // ---------------------------------------- zeros behind the last V row
      // The issuer asks for each such tile when it has landed and waits for
      // the answer before its PV, so both barriers keep in step.
      Ring<kSlots> ring;
      uint32_t fixes = 0;
      bool ok = true;
      Item item;
      while (ok && next_item(item)) {
        ring.n += 2 * item.blocks;
        const int rows = tail_rows(item);
        if (item.blocks == 0 || rows >= kBN) continue;
        ok = __all_sync(0xffffffffu, mbar_wait(v_need, fixes++ & 1, fs));
        if (!ok) break;
        // the last tile of an item is the V tile of its last block
        uint8_t* tile = smem + L::kOffKV + (ring.n - 1) % kSlots * kTileBytes;
        for (int i = max(rows, 0) * 8 + lane; i < kBN * 8; i += 32)
#pragma unroll
          for (int b = 0; b < L::kBoxes; ++b)
            *reinterpret_cast<uint4*>(tile + b * kBoxBytes + i * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_ready);
      }
    } else if (lane == 0) {
      // ---------------------------------------------------- work announcer
      Ring<kItems> out;
      int b = *start_b;
      Segment s = b < 0 ? pre : own_segment(args, b);
      int h = 0, u = 0, j = 0;
      if (lo < hi) {
        long long off = *start_off;
        h = (int)(off / s.work);
        off -= h * s.work;
        while (true) {
          const int kb = unit_blocks(args, s, u, b >= 0 && args.causal);
          if (off < kb) break;
          off -= kb;
          ++u;
        }
        j = (int)off;
      }
      // CTA that holds a unit: the last i with total * i / G <= unit
      auto cta_of = [&](long long unit) { return (int)(((unit + 1) * G - 1) / total); };
      long long pos = lo;
      bool ok = true;
      while (ok) {
        Item item;
        item.request = kEnd;
        if (pos < hi) {
          const bool causal = b >= 0 && args.causal;
          const int kb = unit_blocks(args, s, u, causal);
          const int take = (int)min((long long)(kb - j), hi - pos);
          const int unit_tok = 2 * args.tile_tok;
          item.request = b;
          item.head = h;
          item.tok0 = s.tok + u * unit_tok;
          item.ntok = min(s.n - u * unit_tok, unit_tok);
          item.j0 = j;
          item.keys = s.keys;
          item.pos0 = causal ? s.keys - s.n + u * unit_tok : INT32_MAX / 2;
          const bool empty = s.keys == 0 || item.pos0 + item.ntok <= 0;
          item.blocks = empty ? 0 : take;
          const long long begin = pos - j;
          item.slot = -1;
          item.pieces = 1;
          item.first = 0;
          if (j != 0 || take != kb) {
            const int c0 = cta_of(begin);
            item.first = 2 * c0 + (total * c0 / G != begin);
            item.pieces = cta_of(begin + kb - 1) - c0 + 1;
            item.slot = j == 0 ? item.first : 2 * (int)blockIdx.x;
          }
          pos += take;
          j = 0;
          if (pos < hi && ++u == s.units) {
            u = 0;
            if (++h == args.kv_heads) {
              h = 0;
              do s = own_segment(args, ++b);
              while (s.work == 0 && b + 1 < args.batch);
            }
          }
        }
        ok = mbar_wait(&item_empty[out.slot()], out.parity() ^ 1, fs);
        if (!ok) break;
        items[out.slot()] = item;
        mbar_arrive(&item_full[out.slot()]);
        ++out.n;
        if (item.request == kEnd) break;
      }
    }
  } else {
    // -------------------------------------------------------- softmax
    reg_alloc<kPagedRegsSoftmax>();
    const int t = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;  // row of the tile
    const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_col = t * 128, p_col = t * 128 + 64, o_col = 256 + t * D;
    const float c = args.c;
    const int rtok = r / args.group, rhead = r - rtok * args.group;
    uint32_t s_n = 0, o_n = 0, x_n = 0;
    auto cross_sync = [&]() -> bool {
      mbar_arrive(xsync);
      const bool ok = mbar_wait(xsync, x_n & 1, fs);
      ++x_n;
      return __all_sync(0xffffffffu, ok);
    };
    bool ok = true;
    // The item stays in shared memory while it is worked on (its registers
    // hold a row of scores) and is released at its end.
    while (ok) {
      if (!__all_sync(0xffffffffu, mbar_wait(&item_full[it.slot()], it.parity(), fs))) break;
      const volatile Item& item = items[it.slot()];
      if (item.request == kEnd) break;
      const bool pair = item.ntok > args.tile_tok;
      const int blocks = item.blocks;
      const int j0 = item.j0;
      const int full = min(item.keys - 1, item.pos0);  // last key every row sees
      const int tok = (pair ? t * args.tile_tok : 0) + rtok;  // token within the unit
      const bool live = rtok < args.tile_tok && tok < item.ntok;
      const bool warp_live = __any_sync(0xffffffffu, live);
      const int jstep = pair ? 1 : 2;
      const int lim = min(item.keys - 1, item.pos0 + tok);  // last key this row sees
      float m_run = -INFINITY;  // running max of S*c (log2 domain)
      float l_run = 0.0f;       // running sum of P against m_run
      for (int j = pair ? 0 : t; j < blocks; j += jstep) {
        const bool ready = mbar_wait(&s_full[t], s_n & 1, fs);
        ++s_n;
        if (!__all_sync(0xffffffffu, ready)) { ok = false; break; }
        tc_fence_after();
        if (warp_live) {
          float s[kBN];
#pragma unroll
          for (int ch = 0; ch < 4; ++ch) {
            uint32_t u[32];
            tmem_ld_32x32b_x32(lane_base + s_col + ch * 32, u);
#pragma unroll
            for (int e = 0; e < 32; ++e) s[ch * 32 + e] = __uint_as_float(u[e]);
          }
          tmem_wait_ld();
          const int key0 = (j0 + j) * kBN;
          if (key0 + kBN - 1 > full) {
#pragma unroll
            for (int e = 0; e < kBN; ++e)
              if (key0 + e > lim) s[e] = -INFINITY;
          }
          float m8[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float* v = s + 16 * i;
            float m = fmax3(v[0], v[1], v[2]);
#pragma unroll
            for (int k = 3; k < 15; k += 2) m = fmax3(m, v[k], v[k + 1]);
            m8[i] = fmaxf(m, v[15]);
          }
          const float mx =
              fmax3(fmax3(m8[0], m8[1], m8[2]), fmax3(m8[3], m8[4], m8[5]), fmaxf(m8[6], m8[7]));
          const float m_new = fmaxf(m_run, mx * c);
          bool need = false;
          if (l_run == 0.0f) {
            // nothing accumulated yet (O is rewritten by the first PV or holds 0)
            m_run = m_new;
          } else {
            need = m_new - m_run > kMoveLog2;
          }
          if (__any_sync(0xffffffffu, need)) {
            // this stream's last PV is complete: its S was issued after it
            const float alpha = need ? ex2_approx(m_run - m_new) : 1.0f;
            if (need) {
              l_run *= alpha;
              m_run = m_new;
            }
#pragma unroll 1
            for (int ch = 0; ch < D / 32; ++ch) {
              uint32_t u[32];
              tmem_ld_32x32b_x32(lane_base + o_col + ch * 32, u);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) u[e] = __float_as_uint(__uint_as_float(u[e]) * alpha);
              tmem_st_32x32b_x32(lane_base + o_col + ch * 32, u);
            }
          }
          const float m_use = m_run == -INFINITY ? 0.0f : m_run;
          const uint64_t c2 = f2_pack(c, c), nm2 = f2_pack(-m_use, -m_use);
          uint64_t acc2[2] = {0ull, 0ull};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t pk[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const uint64_t x2 = f2_fma(f2_pack(s[h * 64 + 2 * e], s[h * 64 + 2 * e + 1]), c2, nm2);
              float a, b;
              f2_unpack(x2, a, b);
              const float p0 = ex2_approx(a), p1 = ex2_approx(b);
              acc2[e & 1] = f2_add(acc2[e & 1], f2_pack(p0, p1));
              pk[e] = pack_half2(p0, p1);
            }
            tmem_st_32x32b_x32(lane_base + p_col + h * 32, pk);
          }
          float sa, sb, sc2, sd;
          f2_unpack(acc2[0], sa, sb);
          f2_unpack(acc2[1], sc2, sd);
          l_run += (sa + sb) + (sc2 + sd);
          tmem_wait_st();
        }
        tc_fence_before();
        mbar_arrive(&p_full[t]);
      }
      if (!ok) break;
      // -------------------------------------------------------- epilogue
      if (blocks > 0) {
        const bool done = mbar_wait(o_full, o_n & 1, fs);
        ++o_n;
        if (!__all_sync(0xffffffffu, done)) { ok = false; break; }
        tc_fence_after();
      }
      // weights of the two accumulators a row may have (solo: both streams)
      // (a sum of 0 is a row without visible keys; a NaN sum stays NaN)
      float w0 = l_run == 0.0f ? 0.0f : 1.0f / l_run, w1 = 0.0f;
      float lse = l_run == 0.0f ? -INFINITY : m_run + log2f(l_run);
      uint32_t a0_col = o_col;
      int col0 = 0, cols = D;
      if (!pair) {
        float2* buf = ml + (x_n & 1) * 256;
        buf[t * 128 + r] = make_float2(m_run, l_run);
        if (!cross_sync()) { ok = false; break; }
        const float2 x = buf[r], y = buf[128 + r];
        const float m = fmaxf(x.y == 0.0f ? -INFINITY : x.x, y.y == 0.0f ? -INFINITY : y.x);
        const float ex = x.y == 0.0f ? 0.0f : ex2_approx(x.x - m);
        const float ey = y.y == 0.0f ? 0.0f : ex2_approx(y.x - m);
        const float l = ex * x.y + ey * y.y;
        w0 = l == 0.0f ? 0.0f : ex / l;
        w1 = l == 0.0f ? 0.0f : ey / l;
        lse = l == 0.0f ? -INFINITY : m + log2f(l);
        a0_col = 256;
        cols = D / 2;  // warpgroup t finishes its half of the columns
        col0 = t * cols;
      }
      const long long row = ((long long)item.tok0 + tok) * args.q_heads + item.head * args.group + rhead;
      const int kind = item.request < 0;
      const int slot = item.slot;
      const bool direct = slot < 0 && args.prefix_len == 0;
      const int prow = (pair ? t * kBM : 0) + r;
      float* dst = nullptr;
      if (live) {
        if (slot >= 0) dst = args.cut_o + ((long long)slot * 256 + prow) * D;
        else if (!direct) dst = args.whole_o[kind] + row * D;
        if (pair || t == 0) {
          if (slot >= 0) args.cut_lse[(long long)slot * 256 + prow] = lse;
          else if (!direct) args.whole_lse[kind][row] = lse;
          if (j0 == 0) args.info[kind][row] = make_int2(item.first, item.pieces | (prow << 16));
        }
      }
      __half* orow = args.O + ((long long)item.tok0 + tok) * args.ldo +
                     (long long)(item.head * args.group + rhead) * D;
      if (warp_live) {
#pragma unroll 1
        for (int ch = 0; ch < cols / 32; ++ch) {
          uint32_t u[32];
          if (blocks > 0) {
            tmem_ld_32x32b_x32(lane_base + a0_col + col0 + ch * 32, u);
            tmem_wait_ld();
          }
          float o[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = w0 == 0.0f ? 0.0f : __uint_as_float(u[e]) * w0;
          if (!pair && blocks > 1) {
            tmem_ld_32x32b_x32(lane_base + 256 + D + col0 + ch * 32, u);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e)
              o[e] = w1 == 0.0f ? o[e] : fmaf(__uint_as_float(u[e]), w1, o[e]);
          }
          if (!live) continue;
          if (direct) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              uint4 x;
              x.x = pack_half2(o[v * 8 + 0], o[v * 8 + 1]);
              x.y = pack_half2(o[v * 8 + 2], o[v * 8 + 3]);
              x.z = pack_half2(o[v * 8 + 4], o[v * 8 + 5]);
              x.w = pack_half2(o[v * 8 + 6], o[v * 8 + 7]);
              *reinterpret_cast<uint4*>(orow + col0 + ch * 32 + v * 8) = x;
            }
          } else {
#pragma unroll
            for (int v = 0; v < 8; ++v)
              *reinterpret_cast<float4*>(dst + col0 + ch * 32 + v * 4) =
                  make_float4(o[v * 4], o[v * 4 + 1], o[v * 4 + 2], o[v * 4 + 3]);
          }
        }
      }
      tc_fence_before();
      if (blocks > 0) mbar_arrive(o_free);
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[it.slot()]);
      ++it.n;
    }
  }

  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Merges the partials of every row: one warp per (token, query head), lane l
// holding D / 32 output elements. A row has one partial per CTA that walked a
// part of its prefix keys or of its own keys (info: slot of the first piece,
// number of pieces, row within the slot); a row without any key is 0.
template <int D>
__global__ void __launch_bounds__(256) attention_paged_combine_kernel(const PagedArgs args) {
  pdl_wait();
  pdl_trigger();
  constexpr int kPer = D / 32;
  const long long row = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  const int tok = (int)min(row / args.q_heads, (long long)args.total_q);
  if (tok < clamp_token(args, 0) || tok >= clamp_token(args, args.batch)) return;
  const int sets = args.prefix_len > 0 ? 2 : 1;
  const int2 own = args.info[0][row];
  const int2 pre = sets == 2 ? args.info[1][row] : make_int2(0, 0);
  const int n_own = own.y & 0xffff, n_pre = pre.y & 0xffff;
  if (sets == 1 && n_own == 1) return;  // written by the attention kernel
  // (records left unwritten by a launch that gave up on a wait)
  const int slots = 2 * args.ctas;
  auto wrong = [&](int2 info, int n) {
    return n < 1 || info.x < 0 || 2 * ((info.x >> 1) + n) > slots || (unsigned)info.y >> 16 > 255u;
  };
  if (wrong(own, n_own) || (sets == 2 && wrong(pre, n_pre))) return;
  const int pieces = n_own + n_pre;
  // log2-sum of piece i of the row, and where its output is
  auto locate = [&](int i, const float** o) -> float {
    const bool prefix = i >= n_own;
    const int2 info = prefix ? pre : own;
    const int n = prefix ? n_pre : n_own, p = prefix ? i - n_own : i;
    if (n == 1) {
      *o = (prefix ? args.whole_o[1] : args.whole_o[0]) + row * D;
      return prefix ? args.whole_lse[1][row] : args.whole_lse[0][row];
    }
    const long long slot = p == 0 ? info.x : 2 * ((info.x >> 1) + p);
    const long long at = slot * 256 + (info.y >> 16);
    *o = args.cut_o + at * D;
    return args.cut_lse[at];
  };
  float m = -INFINITY;
  bool nan = false;
  for (int i = lane; i < pieces; i += 32) {
    const float* o;
    const float lse = locate(i, &o);
    m = fmaxf(m, lse);
    nan |= lse != lse;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float acc[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.0f;
  float sum = 0.0f;
  if (__any_sync(0xffffffffu, m != -INFINITY || nan)) {
    for (int base = 0; base < pieces; base += 32) {
      const int cnt = min(32, pieces - base);
      const float* src = nullptr;
      float w = 0.0f;
      if (lane < cnt) {
        const float lse = locate(base + lane, &src);
        w = lse == -INFINITY ? 0.0f : ex2_approx(lse - m);
      }
      sum += w;
      for (int i = 0; i < cnt; i += 4) {
        float v[4][kPer], wi[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int from = min(i + x, cnt - 1);
          const float* po = reinterpret_cast<const float*>(
              __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), from));
          wi[x] = __shfl_sync(0xffffffffu, w, from);
          if constexpr (kPer == 4) {
            const float4 y = *reinterpret_cast<const float4*>(po + lane * 4);
            v[x][0] = y.x, v[x][1] = y.y, v[x][2] = y.z, v[x][3] = y.w;
          } else {
            const float2 y = *reinterpret_cast<const float2*>(po + lane * 2);
            v[x][0] = y.x, v[x][1] = y.y;
          }
        }
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int e = 0; e < kPer; ++e)
            if (i + x < cnt) acc[e] = fmaf(wi[x], v[x][e], acc[e]);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  __half* orow = args.O + tok * args.ldo + (row - (long long)tok * args.q_heads) * D + lane * kPer;
  if constexpr (kPer == 4) {
    uint2 v;
    v.x = pack_half2(acc[0] * inv, acc[1] * inv);
    v.y = pack_half2(acc[2] * inv, acc[3] * inv);
    *reinterpret_cast<uint2*>(orow) = v;
  } else {
    *reinterpret_cast<uint32_t*>(orow) = pack_half2(acc[0] * inv, acc[1] * inv);
  }
}

// Workspace: what the partials of a call take, in this order.
struct PagedLayout {
  size_t cut_o, cut_lse, whole_o[2], whole_lse[2], info[2], total;
};

PagedLayout paged_layout(int64_t rows, int64_t D, bool prefix, int ctas) {
  PagedLayout l{};
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off += (bytes + 255) & ~size_t(255);
    return at;
  };
  const size_t cut = (size_t)ctas * 2 * 256;
  l.cut_o = take(cut * D * sizeof(float));
  l.cut_lse = take(cut * sizeof(float));
  for (int k = 0; k < 2; ++k) {
    l.whole_o[k] = take(prefix ? (size_t)rows * D * sizeof(float) : 0);
    l.whole_lse[k] = take(prefix ? (size_t)rows * sizeof(float) : 0);
    l.info[k] = take(k == 0 || prefix ? (size_t)rows * sizeof(int2) : 0);
  }
  l.total = off;
  return l;
}

template <int D>
hxb_status_t launch_paged(const CUtensorMap& tmQ, const CUtensorMap& tmK, const CUtensorMap& tmV,
                          const PagedArgs& args, const DeviceInfo& dev, cudaStream_t stream) {
  static bool configured[64] = {};
  if (!configured[dev.ordinal]) {
    // the register split assumes this launch count (see attention.cu)
    cudaFuncAttributes fa{};
    cudaError_t e = cudaFuncGetAttributes(&fa, attention_paged_kernel<D>);
    if (e != cudaSuccess) return cuda_status(e, "cudaFuncGetAttributes(paged attention)");
    if (fa.numRegs != kPagedRegsLaunch)
      return fail(HXB_STATUS_UNSUPPORTED, "paged attention kernel built with %d registers per "
                  "thread, its register split needs %d", fa.numRegs, kPagedRegsLaunch);
    e = cudaFuncSetAttribute(attention_paged_kernel<D>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, PagedSmem<D>::kAlloc);
    if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(paged attention)");
    configured[dev.ordinal] = true;
  }
  hxb_status_t s = launch_pdl(attention_paged_kernel<D>, dim3((unsigned)dev.num_sms),
                              dim3(kThreads), PagedSmem<D>::kAlloc, stream,
                              "paged attention launch", tmQ, tmK, tmV, args);
  if (s != HXB_OK) return s;
  const long long warps = (long long)args.total_q * args.q_heads;
  return launch_pdl(attention_paged_combine_kernel<D>, dim3((unsigned)((warps + 7) / 8)),
                    dim3(256), 0, stream, "paged attention combine launch", args);
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

extern "C" hxb_status_t hxb_attention_paged_f16(
    const void* Q, int64_t ldq, void* O, int64_t ldo, const int32_t* q_start,
    const int32_t* kv_lens, int64_t batch, int64_t total_q, int64_t max_q_len,
    const void* k_cache, const void* v_cache, int64_t block_stride, int64_t num_blocks,
    int64_t block_rows, const int32_t* block_table, int64_t table_ld, int64_t table_cols,
    const int32_t* prefix_table, int64_t prefix_len, int64_t q_heads, int64_t kv_heads,
    int64_t head_dim, float scale, int causal, void* workspace, size_t workspace_bytes,
    void* stream) {
  using namespace hxb;
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
  if (total_q > INT32_MAX / q_heads || table_cols < 1 || table_ld < table_cols ||
      table_cols > INT32_MAX / 2 / block_rows || prefix_len < 0 || prefix_len > INT32_MAX / 2)
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

  // Tokens per Q box: the fewest whose rows are whole 8-row swizzle groups, so
  // that a short tile loads few rows; one box of the whole tile where that is
  // more than half a tile.
  int64_t box_tok = 1;
  while (box_tok * group % 8) ++box_tok;
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
  a.O = static_cast<__half*>(O);
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
  a.ctas = dev->num_sms;
  a.c = (float)((double)scale * 1.4426950408889634);  // scale * log2(e)
  char* ws = static_cast<char*>(workspace);
  a.cut_o = reinterpret_cast<float*>(ws + l.cut_o);
  a.cut_lse = reinterpret_cast<float*>(ws + l.cut_lse);
  for (int k = 0; k < 2; ++k) {
    a.whole_o[k] = reinterpret_cast<float*>(ws + l.whole_o[k]);
    a.whole_lse[k] = reinterpret_cast<float*>(ws + l.whole_lse[k]);
    a.info[k] = reinterpret_cast<int2*>(ws + l.info[k]);
  }
  a.status = dev->status_word;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return head_dim == 64 ? launch_paged<64>(tmQ, tmK, tmV, a, *dev, st)
                        : launch_paged<128>(tmQ, tmK, tmV, a, *dev, st);
}
