// The paged attention kernel for row units of up to 256 rows (rows on the TMEM
// lanes), in the tile scheme of attention.cu:
//   * S = Q K^T (tcgen05, operands in shared memory) lands in TMEM, a softmax
//     warpgroup (thread = row) writes P = 2^(S c - m) as f16 over S, and
//     O += P V accumulates in TMEM; the maximum moves only when it grows by
//     more than 2^8.
//   * a unit of more than one 128-row tile keeps its two tiles in flight
//     ("pair": both share every K/V block); a unit of one tile gives the two
//     softmax warpgroups alternate key blocks of the SAME tile ("solo") and
//     merges the two accumulators in the epilogue, so that short units do not
//     wait for one softmax chain per block.
// Bound: the tensor core and the exponentials, 2.05 to 2.15 us per 256 x 128 block
// at D = 128 (1.2 PFLOP/s), where the keys are many, 2.1 at D = 64 (the exponentials
// are the same); 2.6 us (D = 128) beside a narrow kernel that saturates HBM. One CTA
// per SM, persistent.
#pragma once

#include "paged_work.cuh"

namespace hxb {

constexpr int kThreads = 384;
constexpr int kItems = 4;  // items announced ahead of the roles
constexpr int kStagePitch = 80;  // 64 bytes of a row, and 16 against bank conflicts
// Register split of the 384 launch threads, as in attention.cu.
constexpr int kPagedRegsLaunch = 168;
constexpr int kPagedRegsControl = 104;
constexpr int kPagedRegsSoftmax = 200;
static_assert(kPagedRegsControl * 128 + kPagedRegsSoftmax * (kThreads - 128) <=
                  kPagedRegsLaunch * kThreads,
              "register split exceeds the launch allocation");

template <int D>
struct WideSmem {
  static_assert(D == 64 || D == 128, "head dimension 64 or 128");
  static constexpr int kBoxes = D / 64;
  static constexpr int kTileBytes = 128 * D * 2;
  static constexpr int kSlots = D == 64 ? 8 : 4;
  static constexpr int kOffQ = 0;
  static constexpr int kOffKV = kOffQ + 2 * kTileBytes;
  static constexpr int kOffML = kOffKV + kSlots * kTileBytes;  // [2][2][128] float2
  static constexpr int kOffStage = kOffML + 4 * 128 * 8;  // [8 warps][32 rows]
  static constexpr int kOffItems = kOffStage + 8 * 32 * kStagePitch;
  static constexpr int kOffBar = kOffItems + kItems * 64;
  // q_full, q_empty, kv_full[], kv_empty[], s_full[2], p_full[2], o_full,
  // o_free, v_need, v_ready, xsync, item_full[], item_empty[], drain
  static constexpr int kNumBars = 2 + 2 * kSlots + 4 + 5 + 2 * kItems + 1;
  static constexpr int kOffMisc = kOffBar + kNumBars * 8;
  static constexpr int kOffShare = kOffMisc + 16;
  static constexpr int kBytes = kOffShare + (int)sizeof(ShareSmem<kThreads>);
  static constexpr int kAlloc = kBytes + 1024;
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    attention_paged_wide_kernel(const __grid_constant__ CUtensorMap tmQ,
                                const __grid_constant__ CUtensorMap tmK,
                                const __grid_constant__ CUtensorMap tmV, const PagedArgs args) {
  using L = WideSmem<D>;
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
  volatile int* v_job = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 8);
  auto& share_smem = *reinterpret_cast<ShareSmem<kThreads>*>(smem + L::kOffShare);

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
      mbar_init(&item_empty[s], 2 + 8);  // producer, issuer, 8 softmax warps
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
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
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  // (in this order: a narrow kernel that runs beside this one does not wait)
  pdl_wait();
  pdl_trigger();
  const Share share = find_share(args, share_smem);
  if (share.lo >= share.hi) {  // no work: the SM is the next kernel's
    if (warp == 1) tmem_dealloc(tmem_base, 512);
    return;
  }

  // Reads the next item; false at the end and on failure.
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

  if (warp < 4) {
    reg_dealloc<kPagedRegsControl>();
    if (warp == 0) {
      // -------------------------------------------------------- TMA producer
      const TileLoader<D> loader(args, lane);
      Ring<kSlots> ring;
      uint32_t q_items = 0;
      bool ok = true;
      Item item;
      while (ok && next_item(item)) {
        if (item.blocks == 0) continue;
        const bool pair = item.ntok > args.tile_tok;
        const int la = pair ? 1 : 2;  // K blocks ahead of the V block
        // Q of the row unit (a second tile begins where the first one's boxes
        // end: tile_tok is a multiple of box_tok)
        if (!__all_sync(0xffffffffu, mbar_wait(q_empty, (q_items & 1) ^ 1, fs))) break;
        ++q_items;
        const int tile_boxes = args.tile_tok / args.box_tok;
        const int q_boxes = (item.ntok + args.box_tok - 1) / args.box_tok;
        const int box_bytes = args.box_tok * args.group * 128;
        if (lane == 0) mbar_arrive_expect_tx(q_full, q_boxes * L::kBoxes * box_bytes);
        __syncwarp();
        for (int i = lane; i < q_boxes * L::kBoxes; i += 32) {
          const int half = i % L::kBoxes, q = i / L::kBoxes;
          const int t = q >= tile_boxes, bx = q - t * tile_boxes;
          tma_load_3d(smem + L::kOffQ + t * kTileBytes + half * kBoxBytes + bx * box_bytes, &tmQ,
                      q_full, 64 * half, item.head * args.group, item.tok0 + q * args.box_tok);
        }
        // V block j behind K block j + la (the first la K blocks by themselves)
#pragma unroll 1
        for (int i = -2 * la; i < 2 * item.blocks && ok; ++i) {
          const int which = !(i & 1);  // V_j, then K_{j + la}
          const int j = which ? i >> 1 : (i >> 1) + la;
          if (j < 0 || j >= item.blocks) continue;
          const BlockOf at = block_at(args, item, item.j0 + j);
          // (the block id is on its way while the slot is waited for)
          const int block = loader.block_of(args, at.keys, at.table, at.j);
          const int slot = ring.slot();
          ok = __all_sync(0xffffffffu, mbar_wait(&kv_empty[slot], ring.parity() ^ 1, fs));
          if (!ok) break;
          loader.load(args, item.head, which ? &tmV : &tmK, smem + L::kOffKV + slot * kTileBytes,
                      &kv_full[slot], at.j, block);
          ++ring.n;
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
          const int nb = item.blocks, la = pair ? 1 : 2;
          // Step j: PV of block j and S of block j + la, for both tiles (pair) or
          // for stream j mod 2 (solo).
#pragma unroll 1
          for (int j = -la; j < nb && ok; ++j) {
            const bool more = j + la < nb;
            const int vslot = ring.slot();
            bool fix = false;
            if (j >= 0) {
              if (!(ok = mbar_wait(&kv_full[vslot], ring.parity(), fs))) break;
              ++ring.n;
              const int rows = block_rows_at(args, item, item.j0 + j);
              fix = rows < kBN;
              if (fix) {  // (zeroed while the softmax runs)
                *v_job = vslot << 8 | rows;
                mbar_arrive(v_need);
              }
              // both warpgroups have read the previous item's accumulators
              if (j == 0 && q_items && !(ok = mbar_wait(o_free, (q_items & 1) ^ 1, fs))) break;
            }
            const int kslot = ring.slot();
            bool k_here = false;
            const int t0 = pair ? 0 : j & 1, t1 = pair ? 1 : t0;
#pragma unroll 1
            for (int t = t0; t <= t1; ++t) {
              if (j >= 0) {
                if (!(ok = mbar_wait(&p_full[t], (p_par >> t) & 1, fs))) break;
                p_par ^= 1u << t;
                if (fix && t == t0 && !(ok = mbar_wait(v_ready, fixes++ & 1, fs))) break;
                tc_fence_after();
                const uint64_t vd = v_desc + vslot * kTileStep;
#pragma unroll
                for (int kk = 0; kk < kBN / 16; ++kk)
                  umma_f16_ts(tmem_base + 256 + t * D, tmem_base + t * 128 + 64 + kk * 8,
                              vd + (uint64_t)(kk * 16 * 128 >> 4), kIdescPV, j >= la || kk != 0);
                if (t == t1) umma_commit(&kv_empty[vslot]);
              }
              if (more) {
                if (!k_here && !(ok = mbar_wait(&kv_full[kslot], ring.parity(), fs))) break;
                k_here = true;
                tc_fence_after();
                const uint64_t qd = q_desc + (pair ? t : 0) * kTileStep;
                const uint64_t kd = k_desc + kslot * kTileStep;
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                  umma_f16_ss(tmem_base + t * 128, qd + kstep(kk), kd + kstep(kk), kIdescQK,
                              kk != 0);
                umma_commit(&s_full[t]);
                issued_any = true;
              }
            }
            if (!ok) break;
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
      if (lane == 0) {
        *v_job = -1;
        mbar_arrive(v_need);
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
      // the answer before its PV, so both barriers keep in step; a job of -1
      // is the end.
      uint32_t fixes = 0;
      while (__all_sync(0xffffffffu, mbar_wait_for(v_need, fixes++ & 1, fs, kLongWaitNs))) {
        const int job = *v_job;
        if (job < 0) break;
        uint8_t* tile = smem + L::kOffKV + (job >> 8) * kTileBytes;
        // (behind the end of its cache block a tile is zeros already)
        const int P = 1 << args.rows_log2, live = job & 255, end = min(kBN, (live + P - 1) & -P);
        for (int i = live * 8 + lane; i < end * 8; i += 32)
#pragma unroll
          for (int b = 0; b < L::kBoxes; ++b)
            *reinterpret_cast<uint4*>(tile + b * kBoxBytes + i * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_ready);
      }
    } else if (lane == 0) {
      announce<kItems, false>(args, share, share_smem, items, item_full, item_empty, fs);
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
    // parities of the next phases of s_full[t], o_full and xsync (one register:
    // a row of scores fills the others)
    constexpr uint32_t kS = 1, kO = 2, kX = 4;
    uint32_t ph = 0;
    auto cross_sync = [&]() -> bool {
      mbar_arrive(xsync);
      const bool ok = mbar_wait(xsync, (ph & kX) != 0, fs);
      ph ^= kX;
      return __all_sync(0xffffffffu, ok);
    };
    bool ok = true;
    // The first pass has no item: it runs the block's instructions once on
    // whatever the O columns hold (the first PV rewrites them), while the first
    // loads are under way, so that the first block does not wait for 12 KB of
    // instruction fetches.
    bool warm = true;
    // The item stays in shared memory while it is worked on (its registers
    // hold a row of scores) and is released at its end.
#pragma unroll 1
    while (ok) {
      const volatile Item& item = items[it.slot()];
      if (!warm) {
        if (!__all_sync(0xffffffffu, mbar_wait(&item_full[it.slot()], it.parity(), fs))) break;
        if (item.request == kEnd) break;
      }
      const bool pair = warm || item.ntok > args.tile_tok;
      // the row's token within the unit, and whether the tile has that row
      auto token = [&]() { return (pair ? t * args.tile_tok : 0) + r / args.group; };
      auto is_live = [&]() { return r < args.tile_tok * args.group && token() < item.ntok; };
      const bool warp_live = warm || __any_sync(0xffffffffu, is_live());
      const int nb = warm ? t + 1 : item.blocks;
      float m_run = -INFINITY;  // running max of S*c (log2 domain)
      float l_run = 0.0f;       // running sum of P against m_run
#pragma unroll 1
      for (int j = pair && !warm ? 0 : t; j < nb; j += pair ? 1 : 2) {
        if (!warm) {
          const bool ready = mbar_wait(&s_full[t], ph & kS, fs);
          ph ^= kS;
          if (!__all_sync(0xffffffffu, ready)) { ok = false; break; }
          tc_fence_after();
        }
        if (warp_live) {
          float s[kBN];
#pragma unroll
          for (int ch = 0; ch < 4; ++ch) {
            uint32_t u[32];
            tmem_ld_32x32b_x32(lane_base + (warm ? o_col : s_col) + ch * 32, u);
#pragma unroll
            for (int e = 0; e < 32; ++e) s[ch * 32 + e] = __uint_as_float(u[e]);
          }
          tmem_wait_ld();
          // keys of the block that all rows see, and (fewer) that this row sees
          const int jj = item.j0 + j - item.pre;
          int all = jj < 0 ? args.prefix_len - (jj + item.pre) * kBN
                           : min(item.keys - 1, item.pos0) + 1 - jj * kBN;
          if (all < kBN) {
            if (jj >= 0) all = min(item.keys - 1, item.pos0 + token()) + 1 - jj * kBN;
#pragma unroll
            for (int e = 0; e < kBN; ++e)
              if (e >= all) s[e] = -INFINITY;
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
            tmem_st_32x32b_x32(lane_base + (warm ? o_col : p_col) + h * 32, pk);
          }
          float sa, sb, sc2, sd;
          f2_unpack(acc2[0], sa, sb);
          f2_unpack(acc2[1], sc2, sd);
          l_run += (sa + sb) + (sc2 + sd);
          tmem_wait_st();
        }
        if (warm) break;
        tc_fence_before();
        mbar_arrive(&p_full[t]);
      }
      if (!ok) break;
      if (warm) {
        warm = false;
        continue;
      }
      // -------------------------------------------------------- epilogue
      const int blocks = item.blocks;
      const int tok = token();
      const bool live = is_live();
      if (blocks > 0) {
        const bool done = mbar_wait(o_full, (ph & kO) != 0, fs);
        ph ^= kO;
        if (!__all_sync(0xffffffffu, done)) { ok = false; break; }
        tc_fence_after();
      }
      // weights of the two accumulators a row may have (solo: both streams);
      // a sum of 0 is a row without visible keys, a NaN sum stays NaN
      float w0 = l_run == 0.0f ? 0.0f : 1.0f / l_run, w1 = 0.0f;
      float lse = l_run == 0.0f ? -INFINITY : m_run + log2f(l_run);
      uint32_t a0_col = o_col;
      int col0 = 0, cols = D;
      if (!pair) {
        float2* buf = ml + (ph & kX ? 256 : 0);
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
      const int kind = item.request < 0;
      const int slot = item.slot;
      const bool direct = slot < 0 && (args.prefix_len == 0 || item.pre > 0);
      const int prow = (pair ? t * kBM : 0) + r;
      const int R = args.total_q * args.group;
      const int pr = (item.tok0 + tok) * args.group + r % args.group;
      // float4 v of the row is at dst + v * pitch floats
      float* dst = nullptr;
      long long pitch = 0;
      if (live) {
        const long long at = (long long)item.head * R + pr;
        if (slot >= 0) {
          dst = args.cut_o[0] + (long long)slot * 256 * D + prow * 4;
          pitch = 256 * 4;
        } else if (!direct) {
          dst = args.whole_o[kind] + ((long long)item.head * (D / 4) * R + pr) * 4;
          pitch = (long long)R * 4;
        }
        if (pair || t == 0) {
          if (slot >= 0) args.cut_lse[0][slot * 256 + prow] = lse;
          else if (!direct) args.whole_lse[kind][at] = lse;
          if (item.j0 == 0)
            args.info[kind][at] = make_int2(item.first | (item.pre > 0 ? kWithPrefix : 0),
                                            item.pieces | (prow << 16));
        }
      }
      const __half* orow = args.O + ((long long)item.tok0 + tok) * args.ldo +
                           (long long)(item.head * args.group + r % args.group) * D + col0;
      // Finished rows go out through shared memory, so that a store writes 64
      // bytes of each of eight rows (a row per lane, 16 bytes at a time, took
      // 4 us for 256 rows of 128). Lane l then has chunk l % 4 of rows l / 4 + 8 q.
      uint8_t* stage = smem + L::kOffStage + (warp - 4) * 32 * kStagePitch;
      const unsigned live_rows = __ballot_sync(0xffffffffu, live);
      if (warp_live) {
#pragma unroll 1
        for (int ch = 0; ch < cols; ch += 16) {
          uint32_t u[16];
          float o[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = 0.0f;
          // (an accumulator whose row sum is 0 is 0: its weight may be 0)
          if (blocks > 0) {
            tmem_ld_32x32b_x16(lane_base + a0_col + col0 + ch, u);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __uint_as_float(u[e]) * w0;
          }
          if (!pair && blocks > 1) {
            tmem_ld_32x32b_x16(lane_base + 256 + D + col0 + ch, u);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = fmaf(__uint_as_float(u[e]), w1, o[e]);
          }
          if (direct) {
#pragma unroll
            for (int v = 0; v < 2; ++v) {
              uint4 x;
              x.x = pack_half2(o[v * 8 + 0], o[v * 8 + 1]);
              x.y = pack_half2(o[v * 8 + 2], o[v * 8 + 3]);
              x.z = pack_half2(o[v * 8 + 4], o[v * 8 + 5]);
              x.w = pack_half2(o[v * 8 + 6], o[v * 8 + 7]);
              *reinterpret_cast<uint4*>(stage + lane * kStagePitch + (ch & 16) * 2 + v * 16) = x;
            }
            if (ch & 16) {
              __syncwarp();
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const int from = q * 8 + (lane >> 2);
                __half* to = reinterpret_cast<__half*>(__shfl_sync(
                    0xffffffffu, reinterpret_cast<unsigned long long>(orow), from));
                const uint4 x =
                    *reinterpret_cast<const uint4*>(stage + from * kStagePitch + (lane & 3) * 16);
                if (live_rows >> from & 1)
                  *reinterpret_cast<uint4*>(to + ch - 16 + (lane & 3) * 8) = x;
              }
              __syncwarp();
            }
          } else if (live) {
            float* to = dst + (long long)((col0 + ch) / 4) * pitch;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              *reinterpret_cast<float4*>(to) =
                  make_float4(o[v * 4], o[v * 4 + 1], o[v * 4 + 2], o[v * 4 + 3]);
              to += pitch;
            }
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

}  // namespace hxb
