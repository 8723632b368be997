// The paged attention kernel for row units of at most 16 rows (decode: the query
// heads of one KV head times a few tokens). As in attention.cu's decode kernel
// the keys sit on the TMEM lanes:
//   S^T[key, q] = K Q^T   (tcgen05, M = 128 keys, N = 16 rows, K = D)
//   thread = key: its scores, its exponentials, P^T to shared memory
//   O^T[d, q] += V^T P^T   (M = 128 d, N = 16, K = 128 keys)
// so that a block of 128 keys costs each thread one exponential per live row
// and the tensor core next to nothing. Bound: HBM, one K and one V tile per
// block, 1.4 us a block and SM where they stream from HBM and 0.70 from L2 (one
// B200, D = 128, 4 rows, 37 long requests of 8 KV heads; 16 rows 0.75 from L2; D = 64
// 0.68 and 0.63); everything else has to hide behind the loads:
//   * two CTAs per SM, each with a three-tile ring;
//   * S of the next two blocks is computed ahead of the softmax (two TMEM
//     buffers), across items too, and Q is double-buffered: short requests
//     follow one another without a bubble;
//   * the running maxima are shared by the 128 key threads and only recomputed
//     when a score exceeds one by more than 2^8 (one hardware barrier with a
//     vote per block).
// D = 64: the V operand has 64 columns but M is 128, so its second half reads
// the bytes behind the tile (in bounds); lanes 64-127 of O^T are not used.
#pragma once

#include "paged_work.cuh"

namespace hxb {

constexpr int kNarThreads = 256;  // warps: 0 TMA, 1 MMA, 2 Q, 3 announcer, 4-7 keys
constexpr int kNarItems = 8;
constexpr int kNarTmemCols = 64;  // S^T in [0, 16) and [16, 32), O^T in [32, 48)

template <int D>
struct NarrowSmem {
  static_assert(D == 64 || D == 128, "head dimension 64 or 128");
  static constexpr int kBoxes = D / 64;
  static constexpr int kTileBytes = 128 * D * 2;
  static constexpr int kSlots = D == 64 ? 5 : 3;
  static constexpr int kRowsBox = kNarrowRows * 128;  // one [16 rows x 64] f16 box
  static constexpr int kQBytes = kBoxes * kRowsBox;
  static constexpr int kOffKV = 0;
  static constexpr int kOffQ = kOffKV + kSlots * kTileBytes;
  static constexpr int kOffP = kOffQ + 2 * kQBytes;       // P^T as [16 rows][128 keys]
  static constexpr int kOffRed = kOffP + 2 * kRowsBox;    // [3][4 warps][16] floats
  static constexpr int kOffItems = kOffRed + 768;
  static constexpr int kOffBar = kOffItems + kNarItems * 64;
  // q_full[2], q_empty[2], kv_full[], kv_empty[], s_full[2], p_full, p_done,
  // o_full, v_need, item_full[], item_empty[], drain
  static constexpr int kNumBars = 4 + 2 * kSlots + 6 + 2 * kNarItems + 1;
  static constexpr int kOffMisc = kOffBar + kNumBars * 8;
  static constexpr int kOffShare = kOffMisc + 16;
  static constexpr int kEnd_ = kOffShare + (int)sizeof(ShareSmem<kNarThreads>);
  // D = 64: the V operand reads one box behind the last ring slot
  static constexpr int kBytes =
      D == 64 && kEnd_ < kOffQ + kBoxBytes ? kOffQ + kBoxBytes : kEnd_;
  static constexpr int kAlloc = kBytes + 1024;
};

// Barrier of the 128 key threads that returns whether any of them has `flag`.
// Every key warp reaches it after bounded waits only.
__device__ __forceinline__ bool key_vote(bool flag) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "bar.red.or.pred p, 1, 128, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(any)
      : "r"((uint32_t)flag)
      : "memory");
  return any != 0;
}

// The first N of a thread's 16 columns.
template <int N>
__device__ __forceinline__ void tmem_ld_rows(uint32_t taddr, uint32_t (&r)[N]) {
  if constexpr (N == 16) {
    tmem_ld_32x32b_x16(taddr, r);
  } else if constexpr (N == 8) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                   "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
  } else {
    static_assert(N == 4, "4, 8 or 16 rows");
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(taddr));
  }
}
template <int N>
__device__ __forceinline__ void tmem_st_rows(uint32_t taddr, const uint32_t (&r)[N]) {
  if constexpr (N == 16) {
    tmem_st_32x32b_x16(taddr, r);
  } else if constexpr (N == 8) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(
                     taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
                 "r"(r[7])
                 : "memory");
  } else {
    static_assert(N == 4, "4, 8 or 16 rows");
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
                 : "memory");
  }
}

// The largest of the warp's values (a NaN is passed over).
__device__ __forceinline__ float warp_max(float x) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}

// Sums over the warp of N values per lane: lane l returns the sum of value
// l / (32 / N). Half of the values change sides at each of the first steps, so
// that N values take N - 1 + 5 - log2(N) shuffles instead of 5 N.
template <int N>
__device__ __forceinline__ float warp_sums(float (&v)[N], int lane) {
  int o = 16;
#pragma unroll
  for (int n = N / 2; n > 0; n /= 2, o /= 2) {
    const bool up = lane & o;
#pragma unroll
    for (int q = 0; q < n; ++q) {
      const float keep = up ? v[q + n] : v[q], give = up ? v[q] : v[q + n];
      v[q] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
#pragma unroll
  for (; o > 0; o /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
  return v[0];
}

// NR: rows that the instance works on (4, 8 or 16; the row unit has at most that
// many). The instruction footprint grows with it, and short requests fetch every
// instruction for few blocks.
template <int D, int NR>
__global__ void __launch_bounds__(kNarThreads, 2)
    attention_paged_narrow_kernel(const __grid_constant__ CUtensorMap tmK,
                                  const __grid_constant__ CUtensorMap tmV, const PagedArgs args) {
  using L = NarrowSmem<D>;
  constexpr int kSlots = L::kSlots;
  constexpr int kTileBytes = L::kTileBytes;
  constexpr uint32_t kIdescS = make_idesc_f16(128, kNarrowRows, 0, 0);
  constexpr uint32_t kIdescO = make_idesc_f16(128, kNarrowRows, 1, 0);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
  uint64_t* q_empty = q_full + 2;
  uint64_t* kv_full = q_empty + 2;
  uint64_t* kv_empty = kv_full + kSlots;
  uint64_t* s_full = kv_empty + kSlots;
  uint64_t* p_full = s_full + 2;
  uint64_t* p_done = p_full + 1;
  uint64_t* o_full = p_done + 1;
  uint64_t* v_need = o_full + 1;
  uint64_t* item_full = v_need + 1;
  uint64_t* item_empty = item_full + kNarItems;
  uint64_t* drain = item_empty + kNarItems;
  Item* items = reinterpret_cast<Item*>(smem + L::kOffItems);
  float* red = reinterpret_cast<float*>(smem + L::kOffRed);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 4);
  volatile int* v_slot = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 8);
  auto& share_smem = *reinterpret_cast<ShareSmem<kNarThreads>*>(smem + L::kOffShare);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const FailState fs{abort_flag, args.status};

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
      mbar_init(&s_full[s], 1);
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    mbar_init(p_full, 128);
    mbar_init(p_done, 1);
    mbar_init(o_full, 1);
    mbar_init(v_need, 1);
    for (int s = 0; s < kNarItems; ++s) {
      mbar_init(&item_full[s], 1);
      mbar_init(&item_empty[s], 3 + 4);  // producer, issuer, Q warp, 4 key warps
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, kNarTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  // (no pdl_trigger(): combine blocks started early crowd on the SMs that are free
  // first and merge from there, 1 us of a call of 24, 13 us of one of 66)
  // Beside the wide kernel: that one has waited for all before it, and started this
  // one after that, and nothing of it is read here. The fences drop what this SM may
  // hold of the inputs from before.
  if (args.beside) {
    __threadfence();
    fence_proxy_async_global();
  } else {
    pdl_wait();
  }
  const Share share = find_share(args, share_smem);

  // A reader's position in the items (each in shared memory until every reader
  // has released it). A reader that runs ahead of the key threads (the Q warp passes
  // over items without keys) waits here until their item, which may be long, has ended.
  Ring<kNarItems> it;
  auto get = [&](uint32_t n) -> const Item* {
    Ring<kNarItems> at;
    at.n = n;
    const bool ok = wait_bar(&item_full[at.slot()], at.parity(), fs, kLongWaitNs);
    return __all_sync(0xffffffffu, ok) ? &items[at.slot()] : nullptr;
  };
  auto release = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[it.slot()]);
    ++it.n;
  };

  // The producer and the issuer walk the blocks of all items in one order: V (PV)
  // block by block, with the K tiles (S) two blocks ahead, into the next item at
  // most. walk() calls step(which, item, j) in that order, which = 0 for K.
  auto walk = [&](auto step) {
    const Item* cur = get(it.n);
    const Item* nxt = nullptr;
    int j = 0, kj = 0;  // V cursor: block j of cur; K cursor: the kj-th from cur on
#pragma unroll 1
    while (cur && cur->request != kEnd) {
      const int blocks = cur->blocks;
      if (j < blocks) {
        const Item* item = cur;
        int at = j, which = 1;
        if (kj < j + 2) {
          if (kj < blocks) {
            which = 0, at = kj;
          } else {
            if (!nxt && !(nxt = get(it.n + 1))) return;
            if (nxt->request != kEnd && kj - blocks < nxt->blocks)
              which = 0, at = kj - blocks, item = nxt;
          }
        }
        if (!step(which, *item, at)) return;
        if (which == 0) ++kj;
        else ++j;
      } else {
        kj = max(0, kj - blocks);
        j = 0;
        release();
        cur = nxt ? nxt : get(it.n);
        nxt = nullptr;
      }
    }
  };

  if (warp == 0) {
    // ---------------------------------------------------------- TMA producer
    const TileLoader<D> loader(args, lane);
    Ring<kSlots> ring;
    walk([&](int which, const Item& item, int j) -> bool {
      // (the block id is on its way while the slot is waited for)
      const BlockOf at = block_at(args, item, item.j0 + j);
      const int id = loader.block_of(args, at.keys, at.table, at.j);
      const int slot = ring.slot();
      if (!__all_sync(0xffffffffu, wait_bar(&kv_empty[slot], ring.parity() ^ 1, fs))) return false;
      loader.load(args, item.head, which ? &tmV : &tmK, smem + L::kOffKV + slot * kTileBytes,
                  &kv_full[slot], at.j, id, item.request >= 0);
      ++ring.n;
      return true;
    });
    // bounded wait for the copies still landing (complete on the normal path)
    if (lane == 0) {
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
    // ------------------------------------------------------------ MMA issuer
    Ring<kSlots> ring;
    Ring<2> s_ring, q_ring;  // S buffers and Q buffers used so far
    uint32_t p_n = 0;
    bool issued_any = false;
    const uint64_t q_desc = kmajor_desc(smem_u32(smem + L::kOffQ));
    const uint64_t p_desc = kmajor_desc(smem_u32(smem + L::kOffP));
    const uint64_t k_desc = kmajor_desc(smem_u32(smem + L::kOffKV));
    const uint64_t v_desc = vmajor_desc(smem_u32(smem + L::kOffKV));
    constexpr uint64_t kTileStep = kTileBytes >> 4;
    const uint32_t o_tmem = tmem_base + 2 * kNarrowRows;
    walk([&](int which, const Item& item, int j) -> bool {
      bool ok = true;
      const bool last = j == item.blocks - 1;
      if (lane == 0) {
        const int slot = ring.slot();
        if (which == 0) {
          if (j == 0) ok = wait_bar(&q_full[q_ring.slot()], q_ring.parity(), fs);
          ok = ok && wait_bar(&kv_full[slot], ring.parity(), fs);
          if (ok) {
            tc_fence_after();
            // (the buffer's last S was read before p_full of two blocks ago)
            const uint64_t kd = k_desc + slot * kTileStep;
            const uint64_t qd = q_desc + q_ring.slot() * (uint64_t)(L::kQBytes >> 4);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              umma_f16_ss(tmem_base + s_ring.slot() * kNarrowRows, kd + kstep(kk),
                          qd + kstep(kk, L::kRowsBox), kIdescS, kk != 0);
            umma_commit(&s_full[s_ring.slot()]);
            umma_commit(&kv_empty[slot]);
            issued_any = true;
            if (last) umma_commit(&q_empty[q_ring.slot()]);
          }
        } else {
          ok = wait_bar(&kv_full[slot], ring.parity(), fs);
          // the key threads zero the rows behind the last one
          if (ok && last && block_rows_at(args, item, item.j0 + j) < kBN) {
            *v_slot = slot;
            mbar_arrive(v_need);
          }
          ok = ok && wait_bar(p_full, p_n & 1, fs);
          if (ok) {
            tc_fence_after();
            const uint64_t vd = v_desc + slot * kTileStep;
#pragma unroll
            for (int kk = 0; kk < kBN / 16; ++kk)
              umma_f16_ss(o_tmem, vd + (uint64_t)(kk * 16 * 128 >> 4),
                          p_desc + kstep(kk, L::kRowsBox), kIdescO, (j | kk) != 0);
            umma_commit(p_done);
            umma_commit(&kv_empty[slot]);
            if (last) umma_commit(o_full);
          }
        }
      }
      ++ring.n;
      if (which == 0) {
        ++s_ring.n;
        if (last) ++q_ring.n;
      } else {
        ++p_n;
      }
      return __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
    });
    if (lane == 0 && issued_any) {
      // (complete already on the normal path)
      umma_commit(drain);
      const unsigned long long t0 = globaltimer_ns();
      while (!mbar_try_wait(drain, 0) && globaltimer_ns() - t0 < kWaitLimitNs) {
      }
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ Q
    // Copies the unit's rows (up to 16) into the K-major swizzled image; the
    // rows behind them stay as they are and reach only columns not used.
    Ring<2> q_ring;
    const Item* item;
#pragma unroll 1
    while ((item = get(it.n)) && item->request != kEnd) {
      if (item->blocks > 0) {
        constexpr int kChunks = D / 8;              // 16-byte chunks per row
        constexpr int kPer = NR * kChunks / 32;     // per lane
        const int group = args.group, chunks = item->ntok * group * kChunks;
        const __half* src =
            args.Q + (long long)item->tok0 * args.ldq + (long long)item->head * group * D;
        uint4 v[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int idx = i * 32 + lane;
          if (idx < chunks) {
            const int r = idx / kChunks, tok = r / group;
            v[i] = *reinterpret_cast<const uint4*>(src + tok * args.ldq + (r - tok * group) * D +
                                                   idx % kChunks * 8);
          }
        }
        // (the buffer's last unit may still be at work, for as long as it takes)
        if (!__all_sync(0xffffffffu, wait_bar(&q_empty[q_ring.slot()], q_ring.parity() ^ 1, fs,
                                              kLongWaitNs)))
          break;
        uint8_t* dst = smem + L::kOffQ + q_ring.slot() * L::kQBytes;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int idx = i * 32 + lane;
          const int r = idx / kChunks, ch = idx % kChunks;
          if (idx < chunks)
            *reinterpret_cast<uint4*>(dst + (ch >> 3) * L::kRowsBox + r * 128 +
                                      (((ch & 7) ^ (r & 7)) << 4)) = v[i];
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[q_ring.slot()]);
        ++q_ring.n;
      }
      release();
    }
  } else if (warp == 3) {
    if (lane == 0)
      announce<kNarItems, true>(args, share, share_smem, items, item_full, item_empty, fs);
  } else {
    // ------------------------------------------- key threads: softmax, epilogue
    // The four warps vote at fixed places, so a warp whose wait gave up tells
    // the others at the next one and all leave together.
    const int quarter = warp & 3;
    const int kl = quarter * 32 + lane;  // key of the block (S^T lane), d of O^T
    const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const float c = args.c;
    uint8_t* p_smem = smem + L::kOffP + (kl >> 6) * L::kRowsBox;
    const int p_chunk = (kl & 63) >> 3, p_in = (kl & 7) * 2;
    const int group = args.group;
    Ring<2> s_ring;
    uint32_t blocks_done = 0, items_done = 0, fixes = 0;
    bool bad = false;  // a wait of this warp gave up
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      bad = !__all_sync(0xffffffffu, wait_bar(bar, parity, fs)) || bad;
    };
#pragma unroll 1
    while (true) {
      const Item* next = get(it.n);
      bad = !next || bad;
      if (key_vote(bad)) break;
      const Item& item = *next;
      if (item.request == kEnd) break;
      const int rows = item.ntok * group, blocks = item.blocks, key00 = item.j0 * kBN;
      const int keys = item.keys, pos0 = item.pos0;
      float m_run[NR], l_part[NR];
#pragma unroll
      for (int q = 0; q < NR; ++q) {
        m_run[q] = -INFINITY;
        l_part[q] = 0.0f;
      }
      bool stop = false;
#pragma unroll 1
      for (int j = 0; j < blocks; ++j) {
        wait(&s_full[s_ring.slot()], s_ring.parity());
        tc_fence_after();
        uint32_t u[NR];
        tmem_ld_rows<NR>(lane_base + s_ring.slot() * kNarrowRows, u);
        tmem_wait_ld();
        ++s_ring.n;
        const int key = key00 + j * kBN + kl;
        float x[NR];
        bool need = false;
#pragma unroll
        for (int q = 0; q < NR; ++q) x[q] = __uint_as_float(u[q]) * c;
        if (key00 + j * kBN + kBN - 1 > min(keys - 1, pos0)) {  // not all rows see all keys
          int lim = pos0, head = 0;  // of row q
#pragma unroll
          for (int q = 0; q < NR; ++q) {
            if (key > min(keys - 1, lim)) x[q] = -INFINITY;
            if (++head == group) head = 0, ++lim;
          }
        }
        // (rows behind the unit's hold stale scores: they move nothing)
#pragma unroll
        for (int q = 0; q < NR; ++q) need |= q < rows && x[q] > m_run[q] + kMoveLog2;
        if (key_vote(need || bad)) {
          // the block maximum of every row over the 128 keys
          float* rd = red + (blocks_done & 1) * 64;
#pragma unroll
          for (int g = 0; g < NR; g += 4) {
            if (g >= rows) break;  // (uniform)
            const float4 mx = make_float4(warp_max(x[g]), warp_max(x[g + 1]), warp_max(x[g + 2]),
                                          warp_max(x[g + 3]));
            if (lane == 0) *reinterpret_cast<float4*>(rd + quarter * 16 + g) = mx;
          }
          // O^T of the block before is complete
          if (j > 0) wait(p_done, (blocks_done & 1) ^ 1);
          if (key_vote(bad)) { stop = true; break; }
          uint32_t o[NR];
          if (j > 0) {
            tc_fence_after();
            tmem_ld_rows<NR>(lane_base + 2 * kNarrowRows, o);
            tmem_wait_ld();
          }
#pragma unroll
          for (int q = 0; q < NR; ++q) {
            if (q % 4 == 0 && q >= rows) break;  // (uniform)
            const float m_new =
                fmaxf(m_run[q], fmaxf(fmaxf(rd[q], rd[16 + q]), fmaxf(rd[32 + q], rd[48 + q])));
            const float alpha = m_run[q] == -INFINITY ? 0.0f : ex2_approx(m_run[q] - m_new);
            l_part[q] *= alpha;
            m_run[q] = m_new;
            if (j > 0) o[q] = __float_as_uint(__uint_as_float(o[q]) * alpha);
          }
          if (j > 0) {
            tmem_st_rows<NR>(lane_base + 2 * kNarrowRows, o);
            tmem_wait_st();
          }
        }
        // the P image is free when the PV of the block before is complete
        if (blocks_done > 0) wait(p_done, (blocks_done & 1) ^ 1);
#pragma unroll
        for (int q = 0; q < NR; ++q) {
          if (q % 4 == 0 && q >= rows) break;  // (uniform)
          const float pv = ex2_approx(x[q] - (m_run[q] == -INFINITY ? 0.0f : m_run[q]));
          l_part[q] += pv;
          *reinterpret_cast<__half*>(p_smem + q * 128 + ((p_chunk ^ (q & 7)) << 4) + p_in) =
              __float2half_rn(pv);
        }
        ++blocks_done;
        const int live = keys - (key00 + j * kBN);
        if (live < kBN) {
          // zeros behind the last V row, once the tile has landed
          wait(v_need, fixes++ & 1);
          if (!bad) {
            // (behind the end of its cache block a tile is zeros already)
            const int P = 1 << args.rows_log2, end = min(kBN, (live + P - 1) & -P);
            uint8_t* tile = smem + L::kOffKV + *v_slot * kTileBytes;
            for (int i = live * 8 + kl; i < end * 8; i += 128)
#pragma unroll
              for (int b = 0; b < L::kBoxes; ++b)
                *reinterpret_cast<uint4*>(tile + b * kBoxBytes + i * 16) = make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(p_full);
      }
      if (stop) break;
      // ---------------------------------------------------------- epilogue
      float* rl = red + 128;
      const float l_sum = warp_sums<NR>(l_part, lane);
      if (lane % (32 / NR) == 0) rl[quarter * 16 + lane / (32 / NR)] = l_sum;
      uint32_t o[NR];
      if (blocks > 0) {
        wait(o_full, items_done++ & 1);
        tc_fence_after();
        tmem_ld_rows<NR>(lane_base + 2 * kNarrowRows, o);
        tmem_wait_ld();
        tc_fence_before();
      }
      if (key_vote(bad)) break;
      const int kind = item.request < 0, slot = item.slot;
      const bool direct = slot < 0 && args.prefix_len == 0;
      const int R = args.total_q * group;
      const int pr0 = item.tok0 * group;  // packed row of row 0
      const long long at0 = (long long)item.head * R + pr0;
      // element (row q, column kl) is at dst + q * 4
      float* dst = slot >= 0 ? args.cut_o[1] + ((long long)slot * D + (kl >> 2) * 4) * kNarrowRows
                             : args.whole_o[kind] +
                                   (((long long)item.head * (D / 4) + (kl >> 2)) * R + pr0) * 4;
      dst += kl & 3;
      __half* orow = args.O + (long long)item.tok0 * args.ldo + (long long)item.head * group * D + kl;
      const long long skip = args.ldo - (long long)group * D;
      int head = 0;  // of row q
#pragma unroll
      for (int q = 0; q < NR; ++q) {
        if (q < rows) {
          const float l = (rl[q] + rl[16 + q]) + (rl[32 + q] + rl[48 + q]);
          // (a sum of 0 is a row without visible keys, a NaN sum stays NaN)
          const float v = l == 0.0f ? 0.0f : __fdividef(__uint_as_float(o[q]), l);
          if (D == 128 || kl < D) {
            if (direct) *orow = __float2half_rn(v);
            else dst[q * 4] = v;
          }
          orow += D;
          if (++head == group) head = 0, orow += skip;
        }
      }
      // statistics of row kl
      if (kl < rows) {
        float mq = m_run[0];
#pragma unroll
        for (int q = 1; q < NR; ++q) mq = kl == q ? m_run[q] : mq;
        const float l = (rl[kl] + rl[16 + kl]) + (rl[32 + kl] + rl[48 + kl]);
        const float lse = l == 0.0f ? -INFINITY : mq + log2f(l);
        if (slot >= 0) args.cut_lse[1][slot * kNarrowRows + kl] = lse;
        else if (!direct) args.whole_lse[kind][at0 + kl] = lse;
        if (item.j0 == 0)
          args.info[kind][at0 + kl] =
              make_int2(item.first | kNarrowSlot, item.pieces | (kl << 16));
      }
      release();
    }
  }

  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, kNarTmemCols);
  }
  // (the combine kernel waits for this one, and so for the wide one)
  if (args.beside) pdl_wait();
}

}  // namespace hxb
