// What the paged attention kernels (attention_paged.cu) share: the arguments of
// a call, how its work is laid end to end and shared out, and where partial
// results go.
//
// Work: a "segment" is one key set (the shared prefix, or the own keys of one
// request), its tokens cut into row units of unit_tok tokens. For every KV head
// and row unit it visits key blocks of 128. Where every request fills tiles by
// itself (prompt chunks), sharing the prefix would only add partial results: then
// each request's segment visits the prefix blocks first and its own after them.
// All of that is laid end to end in units of one block (a row unit counts
// unit_cost more for its start and end) -- prefix, request 0, request 1 ...;
// inside a segment KV head by KV head, row unit by row unit -- and CTA i takes
// units [i S, (i + 1) S), S = ceil(T / CTAs): equal shares whatever the lengths,
// which are read on the GPU (where both kernels run at once, of the CTAs that each
// has then). The part of a row unit's blocks that falls to one CTA is an item;
// a row unit cut between CTAs leaves one partial result per CTA.
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

#include "sm100.cuh"

namespace hxb {

constexpr int kBM = 128;  // rows per tile of the wide kernel
constexpr int kBN = 128;  // keys per block
constexpr int kBoxBytes = 128 * 64 * 2;  // 128 rows x 64 f16
constexpr int kNarrowRows = 16;          // rows per unit of the narrow kernel
constexpr float kMoveLog2 = 8.0f;        // the running maximum moves by more than 2^8
constexpr int kEnd = -2;

// One piece of work: `blocks` key blocks from block j0 of a row unit.
struct Item {
  int request;  // -1: the shared prefix; kEnd: no more work
  int pre;      // the first `pre` blocks of the row unit are the prefix's
  int head;     // KV head
  int tok0;     // first token of the row unit
  int ntok;     // its tokens
  int j0, blocks;
  int keys;     // keys of the segment's key set
  int pos0;     // last key that token tok0 sees (causal), else INT_MAX / 2
  int slot;     // partial slot of a cut row unit, -1: it is whole here
  int first, pieces;  // a cut row unit: CTA of its first piece, and how many
};
static_assert(sizeof(Item) <= 64, "item record");

struct PagedArgs {
  const int* q_start;
  const int* kv_lens;
  const int* block_table;
  const int* prefix_table;
  const __half* Q;  // the narrow kernel copies Q without TMA
  __half* O;
  long long ldq, ldo, table_ld;
  int total_q, batch, q_heads, kv_heads, group;
  int unit_tok;            // tokens per row unit
  int unit_cost;           // blocks that its start and end cost
  int requests_here;       // this kernel takes the requests' own keys
  int prefix_here;         // and the prefix
  int fat_tok;             // requests of so many tokens fill tiles (0: no matter)
  int beside;              // the other kernel runs at the same time, with
  int other_tok, other_cost;  // row units of so many tokens and such a cost
  int tile_tok, box_tok;   // wide kernel: tokens per 128-row tile and per Q box
  int table_cols, num_blocks, rows_log2;
  int prefix_len;
  int causal;
  float c;  // scale * log2(e)
  // Partial results, f32, normalised, with their log2-sum-exp2. Packed row
  // pr = token * group + head-in-group of KV head h. Four columns of a row lie
  // together and the rows of a tile side by side, so that threads that hold a
  // row each write and read whole lines:
  //   cut row units  cut_o[kernel][slot][D / 4][rows][4], slot = 2 CTA + 1 for
  //                  the unit's first piece, 2 CTA for the others; rows = 256
  //                  (wide, kernel 0) or 16 (narrow, kernel 1)
  //   whole ones     whole_o[set][h][D / 4][total_q * group][4], set = 0 own
  //                  keys, 1 prefix
  // info[set][h][pr]: {CTA of the first piece | flags, pieces | row in the slot
  // << 16}
  float* cut_o[2];
  float* cut_lse[2];
  float* whole_o[2];
  float* whole_lse[2];
  int2* info[2];
  int ctas[2];
  int* status;
};
constexpr int kNarrowSlot = 1 << 30;  // flag: the narrow kernel's slots
constexpr int kWithPrefix = 1 << 29;  // flag: the prefix is in these pieces

// Position in a ring of N slots, counted in uses.
template <int N>
struct Ring {
  uint32_t n = 0;
  __device__ __forceinline__ int slot() const { return n % N; }
  __device__ __forceinline__ uint32_t parity() const { return (n / N) & 1; }
};

__device__ __forceinline__ uint64_t kmajor_desc(uint32_t base) {
  return make_smem_desc(base, 16, 1024, kLayoutSwizzle128);
}
__device__ __forceinline__ uint64_t vmajor_desc(uint32_t base) {
  return make_smem_desc(base, kBoxBytes, 1024, kLayoutSwizzle128);
}
// K-major 16-element K step kk of a tile of boxes of `box` bytes x 64 columns,
// in descriptor address units.
__device__ __forceinline__ constexpr uint64_t kstep(int kk, int box = kBoxBytes) {
  return (uint64_t)(((kk >> 2) * box + (kk & 3) * 32) >> 4);
}

__device__ __forceinline__ int clamp_token(const PagedArgs& a, int b) {
  return min(max(a.q_start[b], 0), a.total_q);
}

struct Segment {
  int tok, n, keys;
  int units;       // row units
  int cost;        // units of work of a row unit's start and end
  int work;        // units of work of one KV head over all row units
  int pre;         // prefix blocks visited before the own ones
  bool causal;
};

// Keys that the last token of row unit u sees.
__device__ __forceinline__ int unit_keys(const PagedArgs& a, const Segment& s, int u) {
  if (!s.causal) return s.keys;
  const int last = min((u + 1) * a.unit_tok, s.n);
  return max(0, min(s.keys, s.keys - s.n + last));
}

__device__ __forceinline__ int unit_blocks(const PagedArgs& a, const Segment& s, int u) {
  // (a unit without keys still writes its rows)
  return max(1, s.pre + (unit_keys(a, s, u) + kBN - 1) / kBN);
}

// sum_{i < n} floor((a i + b) / m), by the Euclidean algorithm on (a, m): whole
// multiples of m leave the sum in closed form, and what is left counts the
// lattice points under a line, which swapping the axes turns into a shorter sum.
// The caller bounds the result (and so every term) below 2^31.
__device__ __forceinline__ unsigned floor_sum(unsigned n, unsigned m, unsigned a, unsigned b) {
  unsigned sum = 0;
#pragma unroll 1
  while (true) {
    const unsigned qa = a / m, qb = b / m;
    // (one of n, n - 1 is even; qa is 0 after the first round or n is short)
    sum += (n & 1 ? (n - 1) / 2 * n : n / 2 * (n - 1)) * qa + n * qb;
    a -= qa * m;
    b -= qb * m;
    const unsigned top = a * n + b;  // (a, b < m <= 256: below 2^32)
    if (top < m) return sum;
    n = top / m;
    b = top - n * m;
    const unsigned t = m;
    m = a;
    a = t;
  }
}

constexpr int kMostWork = 1 << 30;  // units of work of one call (saturated above)

// Work of the first `units` row units of one KV head.
__device__ __forceinline__ int work_before(const PagedArgs& a, const Segment& s, int units) {
  if (units == 0) return 0;
  const int last = unit_blocks(a, s, units - 1);  // the most blocks of a unit
  if ((float)units * (float)(last + s.cost) >= (float)kMostWork) return kMostWork;
  int sum = units * s.cost + last;
  if (!s.causal) return sum + (units - 1) * last;
  // unit u < units - 1 sees d + (u + 1) T own keys: none up to u = dark, then one
  // block per begun 128
  const int T = a.unit_tok, d = s.keys - s.n, full = units - 1;
  const int dark = d < 0 ? min(full, (-d) / T) : 0;
  sum += dark * max(1, s.pre) + (full - dark) * s.pre;
  if (full > dark) sum += (int)floor_sum(full - dark, kBN, T, d + (dark + 1) * T + kBN - 1);
  return sum;
}

__device__ __forceinline__ int own_tokens(const PagedArgs& a, int b) {
  return max(clamp_token(a, b + 1) - clamp_token(a, b), 0);
}

__device__ __forceinline__ Segment own_segment(const PagedArgs& a, int b, int pre) {
  Segment s;
  s.tok = clamp_token(a, b);
  s.n = own_tokens(a, b);
  s.keys = (int)min((long long)max(a.kv_lens[b], 0), (long long)a.table_cols << a.rows_log2);
  s.units = (s.n + a.unit_tok - 1) / a.unit_tok;
  s.pre = pre;
  s.causal = a.causal != 0;
  s.cost = a.unit_cost;
  s.work = work_before(a, s, s.units);
  return s;
}

__device__ __forceinline__ Segment prefix_segment(const PagedArgs& a, bool here) {
  Segment s;
  s.tok = clamp_token(a, 0);
  s.n = here ? max(clamp_token(a, a.batch) - s.tok, 0) : 0;
  s.keys = a.prefix_len;
  s.units = (s.n + a.unit_tok - 1) / a.unit_tok;
  s.pre = 0;
  s.causal = false;
  s.cost = a.unit_cost;
  s.work = work_before(a, s, s.units);
  return s;
}

// A CTA's share of the work: units [lo, hi), `per` units per CTA.
struct Share {
  int lo, hi, per;
  int pre;  // prefix blocks of the requests' own segments
};
template <int THREADS>
struct ShareSmem {
  long long sum[THREADS / 32];
  Segment seg;  // where the share begins: segment, request (-1: the prefix) and
  int b, off;   // unit within the segment
};

// Where both kernels of a call run at once, the wide one takes as many SMs as let
// both end together, the narrow one the others. Here: the wide kernel's share per SM
// of `units` row units with `work` units of work each, and what a row unit counts
// then (a little more where it is cut in equal parts). us of an SM per unit of work,
// side by side on one B200 at D = 128: the wide kernel's 2.5 for two tiles of a prefix
// or 1.7 for one, the narrow one's 0.85 for two CTAs; the narrow kernel as a whole is
// not faster than HBM, 1.25 us per unit and SM; the wide kernel spends 6 us more at
// its start and end. D = 64 goes by the same numbers although they do not scale alike:
// alone, from D = 128 to 64, the wide kernel's unit goes from 2.15 us to 2.09 (one
// tile 1.35 to 1.13), the narrow one's from 1.39 to 0.68 from HBM, 0.70 to 0.63 from L2.
struct WideShare {
  int per, work;
};
__host__ __device__ inline WideShare wide_share(const PagedArgs& a, int units, int work,
                                                float narrow) {
  const float total = (float)units * (float)work;
  const float wide = total * (a.total_q * a.group <= kBM ? 1.7f : 2.5f);
  // n (t - 6) = wide and (sms - n) t = own, the time t not below HBM's
  const float sms = (float)a.ctas[0], own = 0.85f * narrow, b = 6.0f * sms + wide + own;
  const float t = fmaxf((b + sqrtf(b * b - 24.0f * sms * own)) / (2.0f * sms), 1.25f * narrow / sms);
  const float n = fmaxf(fminf(ceilf(wide / fmaxf(t - 6.0f, 1.0f)), sms - 1.0f), 1.0f);
  // (a call of more than kMostWork is not run, but its shares are computed, on the
  // host too: an int all the same)
  const int per = (int)fminf(fmaxf(ceilf(total / n), 1.0f), (float)kMostWork);
  // whole row units, or equal parts of one, where that is near: a CTA with parts of
  // two spends the start and the end of a row unit twice
  if (per >= work) {
    const int whole = per / work * work;
    if (total <= (sms - 1.0f) * (float)whole && 4 * (per - whole) <= whole) return {whole, work};
  } else {
    const int parts = (work + per - 1) / per, part = (work + parts - 1) / parts;
    if ((float)units * (float)parts <= sms - 1.0f) return {part, part * parts};
  }
  return {per, work};
}

// CTAs of the narrow kernel beside the wide one with that share.
__host__ __device__ inline int ctas_beside(const PagedArgs& a, int units, const WideShare& w) {
  const int left = a.ctas[0] - (int)ceilf((float)units * (float)w.work / (float)w.per);
  return left < 1 ? 2 : 2 * left;
}

// This kernel's share per CTA, of `total` units. Beside the other kernel the wide
// one has a prefix only, of which the row units may get longer.
template <int THREADS>
__device__ __forceinline__ int share_per_cta(const PagedArgs& a, ShareSmem<THREADS>& sm,
                                             long long& total, Segment& prefix) {
  int ctas = gridDim.x;
  if (a.beside && a.requests_here) {
    const int tokens = max(clamp_token(a, a.batch) - clamp_token(a, 0), 1);
    const int units = (tokens + a.other_tok - 1) / a.other_tok * a.kv_heads;
    const int work = (a.prefix_len + kBN - 1) / kBN + a.other_cost;
    ctas = min(ctas, ctas_beside(a, units, wide_share(a, units, work, (float)total)));
  } else if (a.beside) {
    float narrow = 0.0f;
#pragma unroll 1
    for (int b = threadIdx.x; b < a.batch; b += THREADS)
      narrow += (float)((own_tokens(a, b) + a.other_tok - 1) / a.other_tok) *
                (float)(max(a.kv_lens[b], 0) / kBN + 1 + a.other_cost);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) narrow += __shfl_xor_sync(0xffffffffu, narrow, o);
    if ((threadIdx.x & 31) == 0) sm.sum[threadIdx.x >> 5] = (long long)narrow;
    __syncthreads();
    long long sum = 0;
#pragma unroll 1
    for (int w = 0; w < THREADS / 32; ++w) sum += sm.sum[w];
    if (prefix.units > 0) {
      const int work = prefix.work / prefix.units;
      const WideShare w = wide_share(a, prefix.units * a.kv_heads, work, (float)a.kv_heads * (float)sum);
      prefix.cost += w.work - work;
      prefix.work = prefix.units * w.work;
      total = (long long)prefix.work * a.kv_heads;
      return w.per;
    }
  }
  return max((int)((total + ctas - 1) / ctas), 1);
}

// Every thread sums the work of a run of requests; a block scan gives the total,
// and the thread that holds the CTA's first unit notes its segment. Called by
// the whole block.
template <int THREADS>
__device__ __forceinline__ Share find_share(const PagedArgs& a, ShareSmem<THREADS>& sm) {
  if (threadIdx.x == 0) sm.seg.work = 0;  // (no segment, until its thread notes one)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int each = a.requests_here ? (a.batch + THREADS - 1) / THREADS : 0;
  const int b0 = min((int)threadIdx.x * each, a.batch), b1 = min(b0 + each, a.batch);
  // every request fills tiles by itself: no shared pass over the prefix
  bool fat = false;
  if (a.fat_tok) {
    bool thin = false;
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
      const int n = own_tokens(a, b);
      thin |= n > 0 && n < a.fat_tok;
    }
    fat = !__syncthreads_or(thin);
  }
  Share r{0, 0, 1, fat ? (a.prefix_len + kBN - 1) / kBN : 0};
  Segment pre = prefix_segment(a, a.prefix_here && !fat);
  int pre_work = (int)min((long long)pre.work * a.kv_heads, (long long)kMostWork);
  long long mine = 0, base = 0, total = pre_work;
  // Two passes over the requests: their work, then (the thread that holds it) the
  // CTA's first unit.
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    long long at = base;
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
      const Segment s = own_segment(a, b, r.pre);
      const long long w = (long long)s.work * a.kv_heads;
      at += w;
      if (pass && r.lo < at) {
        sm.b = b;
        sm.off = r.lo - (int)(at - w);
        sm.seg = s;
        break;
      }
    }
    if (pass) break;
    mine = at;
    if (a.requests_here) {
      long long scan = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += v;
      }
      if (lane == 31) sm.sum[warp] = scan;
      __syncthreads();
      base = total + scan - mine;
#pragma unroll 1
      for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) base += sm.sum[w];
        total += sm.sum[w];
      }
    }
    if (total >= kMostWork) {  // (many seconds of work: not started)
      if (threadIdx.x == 0) atomicOr(a.status, kStatusBadIndex);
      break;
    }
    r.per = share_per_cta(a, sm, total, pre);
    pre_work = max(pre_work, pre.work * a.kv_heads);
    r.lo = (int)min((long long)blockIdx.x * r.per, total);
    r.hi = (int)min((long long)r.lo + r.per, total);
    if (r.lo < pre_work) {
      if (threadIdx.x == 0) {
        sm.b = -1;
        sm.off = r.lo;
        sm.seg = pre;
      }
      break;
    }
    if (r.lo >= r.hi || r.lo < base || r.lo >= base + mine) break;
  }
  __syncthreads();
  return r;
}

// Limit of a wait that a correct call may spend a large part of its time in (for a
// tile to zero, for a long item's end): a launch that is stuck ends by the limit of
// another role's wait, whose flag these waits watch. The most work of a call
// (kMostWork for each kernel) takes less than a minute.
constexpr unsigned long long kLongWaitNs = 32 * kWaitLimitNs;

// mbar_wait_for with its loop out of line: the roles of these kernels wait in many
// places, and what runs once per item should not be fetched anew for each.
static __device__ __noinline__ bool wait_slow(uint64_t* bar, uint32_t parity, volatile int* abort,
                                              int* status, unsigned long long limit_ns) {
  return mbar_wait_for(bar, parity, FailState{abort, status}, limit_ns);
}
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, const FailState& fs,
                                         unsigned long long limit_ns = kWaitLimitNs) {
  if (mbar_try_wait(bar, parity)) return true;
  return wait_slow(bar, parity, fs.abort, fs.status, limit_ns);
}

// Publishes the CTA's items, one after the other, into a ring of N records (one
// thread). item_empty[] collects one arrival of every reader of a record.
// OUT_OF_LINE: wait through wait_bar (not in a kernel that moves registers with
// setmaxnreg, where the compiler cannot place a call).
template <int N, bool OUT_OF_LINE, int THREADS>
__device__ __forceinline__ void announce(const PagedArgs& a, const Share& sh,
                                         const ShareSmem<THREADS>& sm, Item* items,
                                         uint64_t* item_full, uint64_t* item_empty,
                                         const FailState& fs) {
  Ring<N> out;
  int b = -1, h = 0, u = 0, at = 0;  // next: unit of work `at` of row unit u
  int pos = sh.lo;
  Segment s;
  s.work = 0;
  s.units = 0;
  s.cost = 0;
  // The lengths of the following segments are read again, one at a time. Lengths
  // that another stream changes meanwhile (a caller's mistake) must not lead out
  // of the tables: a position that is none ends the work.
  if (sh.lo < sh.hi) {
    s = sm.seg;
    b = sm.b;
    at = max(sm.off, 0);
    if (s.work > 0) {
      h = min(at / s.work, a.kv_heads);
      at = min(at - h * s.work, s.work - 1);
      int above = s.units, before = 0;  // before = work_before(u) <= at < work_before(above)
#pragma unroll 1
      while (above - u > 1) {
        const int mid = (u + above) >> 1, w = work_before(a, s, mid);
        if (w <= at) u = mid, before = w;
        else above = mid;
      }
      at -= before;
    }
  }
#pragma unroll 1
  while (true) {
    const int cost = s.cost;
    Item item;
    item.request = kEnd;
    item.blocks = 0;
    const int kb = unit_blocks(a, s, u);
    if (pos < sh.hi && s.work > 0 && h < a.kv_heads && u < s.units && at < kb + cost) {
      const int take = min(kb + cost - at, sh.hi - pos);
      const int begin = pos - at + cost;  // its first block, as a unit of work
      const int j = max(at - cost, 0), blocks = at + take - cost - j;
      const int keys = unit_keys(a, s, u);
      item.request = b;
      item.pre = s.pre;
      item.head = h;
      item.tok0 = s.tok + u * a.unit_tok;
      item.ntok = min(s.n - u * a.unit_tok, a.unit_tok);
      item.j0 = j;
      item.keys = s.keys;
      item.pos0 = s.causal ? s.keys - s.n + u * a.unit_tok : INT32_MAX / 2;
      item.blocks = keys + s.pre > 0 ? blocks : 0;
      item.first = begin / sh.per;
      item.pieces = (begin + kb - 1) / sh.per - item.first + 1;
      item.slot = item.pieces > 1 ? 2 * (int)blockIdx.x + (j == 0) : -1;
      pos += take;
      at = 0;
      if (pos < sh.hi && ++u == s.units) {
        u = 0;
        if (++h == a.kv_heads) {
          h = 0;
          s.work = 0;
          while (s.work == 0 && b + 1 < a.batch) s = own_segment(a, ++b, sh.pre);
        }
      }
      if (blocks <= 0) continue;  // only the start of a row unit: the next CTA's
    }
    uint64_t* free_slot = &item_empty[out.slot()];
    const uint32_t parity = out.parity() ^ 1;
    if (!(OUT_OF_LINE ? wait_bar(free_slot, parity, fs, kLongWaitNs)
                      : mbar_wait_for(free_slot, parity, fs, kLongWaitNs)))
      return;
    items[out.slot()] = item;
    mbar_arrive(&item_full[out.slot()]);
    ++out.n;
    if (item.request == kEnd) return;
  }
}

// Loads this lane's boxes of one 128-key K or V tile (a whole warp calls it): a
// box is up to 128 rows of one cache block and 64 columns. Rows from item.keys
// on are zeros where a whole box is (an out-of-range block fills with zeros).
template <int D>
struct TileLoader {
  static constexpr int kBoxes = D / 64;
  int lane, boxes, row, half;
  __device__ __forceinline__ TileLoader(const PagedArgs& a, int lane_) : lane(lane_) {
    const int page_rows = min(1 << a.rows_log2, kBN);
    boxes = kBN / page_rows * kBoxes;  // at most 16
    row = lane / kBoxes * page_rows;
    half = lane % kBoxes;
  }
  // the cache block of this lane's box of key block j
  __device__ __forceinline__ int block_of(const PagedArgs& a, int keys, const int* table,
                                          int j) const {
    const int key = j * kBN + row;
    if (lane >= boxes || key >= keys) return a.num_blocks;
    const int id = table[key >> a.rows_log2];
    if (id >= 0 && id < a.num_blocks) return id;
    atomicOr(a.status, kStatusBadIndex);
    return a.num_blocks;
  }
  __device__ __forceinline__ void load(const PagedArgs& a, int head, const CUtensorMap* map,
                                       void* tile, uint64_t* bar, int j, int block,
                                       bool once = false) const {
    if (lane == 0) mbar_arrive_expect_tx(bar, kBN * D * 2);
    __syncwarp();
    const int in = (j * kBN + row) & ((1 << a.rows_log2) - 1);
    if (lane < boxes) {
      uint8_t* dst = static_cast<uint8_t*>(tile) + half * kBoxBytes + row * 128;
      const int x = 64 * half, y = (head << a.rows_log2) + in;
      if (once) tma_load_3d_once(dst, map, bar, x, y, block);
      else tma_load_3d(dst, map, bar, x, y, block);
    }
  }
};

// Where block j of an item's row unit lies: block `j` of the key set with `keys`
// keys behind `table`.
struct BlockOf {
  const int* table;
  int keys, j;
};
template <typename I>
__device__ __forceinline__ BlockOf block_at(const PagedArgs& a, const I& item, int j) {
  if (j < item.pre || item.request < 0) return {a.prefix_table, a.prefix_len, j};
  return {a.block_table + (long long)item.request * a.table_ld, item.keys, j - item.pre};
}
// Rows of block j that exist; a block with fewer than 128 gets the others of its
// V tile zeroed (their P is 0, but 0 * NaN is not).
template <typename I>
__device__ __forceinline__ int block_rows_at(const PagedArgs& a, const I& item, int j) {
  return j < item.pre ? a.prefix_len - j * kBN : item.keys - (j - item.pre) * kBN;
}

}  // namespace hxb
