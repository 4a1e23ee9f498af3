// Tree attention with many query rows (nodes x query heads of a KV head) on
// the tcgen05 tensor cores; see tree_decode.cu for the operator and
// tree_work.cuh for the division of the work.
//
// With R rows per KV head each K/V byte is used for R products, so from some
// tens of rows on warp-level MMAs, not the cache's bytes, set the time.  Here a
// block of up to 128 rows (whole nodes: 128 / group of them) is the M of
// tcgen05.mma, S = Q.K^T and O += P.V accumulate in TMEM, P goes back over S's
// columns as 16-bit pairs (the schedule of prefill_head.cu).
//
// A thread's part of a tile (128 exponentials, and the waits and TMEM traffic
// around them) takes two to three times the tensor core's, so three warpgroups
// take the key tiles in turn, each with an S buffer of its own: while they work
// on tiles j to j + 2, PV(j) frees its buffer for QK(j + 3).  What ties the
// warpgroups is the running maximum: the warp of tile j publishes its rows'
// maximum before its exponentials, and the next warpgroup's warp of the same
// rows goes on from there with tile j + 1.  Each keeps the sum of its own tiles
// relative to the last maximum it used; they meet at the item's end.  S is read
// from TMEM twice (maximum, exponentials) in 64-column steps of a loop rather
// than held in 128 registers: that leaves room for the third warpgroup, and
// code that stays in the instruction cache.  Warps whose 32 rows hold no query
// only pass the barriers.
//
// 512 threads: warps 0 and 2 TMA producers (a box per page piece and 64
// columns, or one per tile where a page holds it), warp 1 TMEM owner and MMA
// issuer, warps 4-15 softmax (TMEM lane quarter = warp % 4).
// Measured, 16 x 32760 rows, bf16, 32/8 heads x 128, pages of 128: 32 rows 343 us
// (6.3 TB/s, HBM), 128 rows 363, 512 rows 1046 to 1080 (1020 to 1050 TFLOP/s, 0.62
// to 0.64 of the measured burst: the softmax chain and the issue of 16 MMAs a
// tile); pages of 16: 466, 472 to 493, 1662 to 1679, the boxes' issue.
// TMEM: S0 .. S2 (BN columns each), O (D columns).

#include <limits.h>

#include "b2a_common.cuh"
#include "tree_work.cuh"

namespace b2a {
namespace tree {

using prefill::Pack2;
using prefill::make_idesc;
using prefill::sw128_desc;
using prefill::tc_commit;
using prefill::tc_fence_after;
using prefill::tc_fence_before;
using prefill::tc_ld32;
using prefill::tc_mma;
using prefill::tc_mma_ts;
using prefill::tc_st16;
using prefill::tc_st32;
using prefill::tc_wait_ld;
using prefill::tc_wait_st;

constexpr int kWideThreads = 512;
constexpr int kWideGroups = 3;  // softmax warpgroups, each with an S buffer
constexpr int kWideM = 128;
constexpr int kMaxSlots = 16;

struct WideShared {
  uint64_t bar_qf, bar_qe, bar_oe, bar_last;  // bar_last: an item's last PV
  uint64_t bar_full[kMaxSlots], bar_empty[kMaxSlots];
  uint64_t bar_sf[kWideGroups], bar_pf[kWideGroups], bar_pv[2], bar_m[kWideGroups][4];
  Start start;
  uint32_t tmem;
  int special;  // the item's tree rows held infinities or NaN
  float x[kWideGroups][kWideM];  // maxima, at an item's end sums, between the warpgroups
};

template <int D>
struct WideCfg {
  static constexpr int kBN = D > 128 ? 64 : 128;      // keys per tile
  static constexpr int kS = kWideGroups;              // S buffers
  static constexpr int kBoxQ = kWideM * 128;          // 128 rows x 64 columns
  static constexpr int kBoxKV = kBN * 128;            // kBN rows x 64 columns
  static constexpr int kTileQ = (D / 64) * kBoxQ;
  static constexpr int kTileKV = (D / 64) * kBoxKV;   // one K or V tile
  // Q, the ring, then barriers and exchanged numbers: all in dynamic shared
  // memory, so that the ring gets what there is (the SM's 227 KB)
  static constexpr int kSlots = (227 * 1024 - sizeof(WideShared) - kTileQ) / kTileKV / 2 * 2;
  static constexpr int kRing = kTileQ;
  static constexpr int kShared = kRing + kSlots * kTileKV;
  static constexpr int kSmem = kShared + sizeof(WideShared);
  static_assert(kS * kBN + D <= 512, "TMEM columns");
  // a slot has the same producer on every use
  static_assert(kSlots % 2 == 0 && kSlots <= kMaxSlots && kSmem <= 227 * 1024, "ring");
};

template <typename T, int D>
__global__ void __launch_bounds__(kWideThreads, 1) tree_wide_kernel(
    const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
    const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Batch bt,
    const T* __restrict__ vc, long long page_stride, T* __restrict__ out, float* __restrict__ lse,
    float* __restrict__ part_o, float* __restrict__ part_ml, int piece_rows, float sscale) {
  using C = WideCfg<D>;
  constexpr int BN = C::kBN;
  constexpr int kSlots = C::kSlots;
  extern __shared__ __align__(1024) uint8_t smem[];
  WideShared& sh = *reinterpret_cast<WideShared*>(smem + C::kShared);
  uint64_t *bar_full = sh.bar_full, *bar_empty = sh.bar_empty;

  pdl_wait();
  if (smem_u32(smem) & 1023u) {  // swizzled tiles start on 1024-byte boundaries
    if (threadIdx.x == 0) set_dev_error(B2A_ERR_ALIGN, 0x3F000);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    const Start s = locate(bt, team_of(bt, blockIdx.x));
    if (lane == 0) sh.start = s;
  } else if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&sh.tmem)),
                 "r"(prefill::kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else if (warp == 2 && lane == 0) {
    mbar_init(&sh.bar_qf, 1);
    mbar_init(&sh.bar_qe, 1);
    mbar_init(&sh.bar_oe, 4 * kWideGroups);
    mbar_init(&sh.bar_last, 1);
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&bar_full[s], 1);
      mbar_init(&bar_empty[s], 1);
    }
    for (int b = 0; b < C::kS; ++b) {
      mbar_init(&sh.bar_sf[b], 1);
      mbar_init(&sh.bar_pf[b], 4);
    }
    for (int w = 0; w < kWideGroups; ++w)
      for (int i = 0; i < 4; ++i) mbar_init(&sh.bar_m[w][i], 1);
    mbar_init(&sh.bar_pv[0], 1);
    mbar_init(&sh.bar_pv[1], 1);
    fence_mbar_init();
    sh.special = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = sh.tmem;
  Walker wk;
  wk.start(bt, sh.start);
  Item it;

  constexpr uint32_t kOCol = C::kS * BN;
  const int block_nodes = bt.rows_per_block / bt.group;

  // a whole warp's wait on a barrier, with one answer for all lanes
  auto arrived = [](uint64_t* bar, uint32_t parity, int where) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, where)) != 0;
  };

  if (warp == 0 || warp == 2) {
    // ------------------------------ TMA producers --------------------------
    // Warp 0 loads Q and K, warp 2 V, so that a K tile never queues behind a V
    // tile whose slot is still in use.  Whole warps walk the loop and one
    // elected lane issues (see the MMA issuer).
    const int p = __shfl_sync(0xffffffffu, warp >> 1, 0);
    const CUtensorMap* map = p ? &tmV : &tmK;
    const bool whole = piece_rows == BN;
    const int bytes = piece_rows * 128 * (D / 64);  // of a page piece
    if (elect_one()) {
      if (p == 0) tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(map);
    }
    uint32_t slot = p, round = 0, items = 0;  // K tiles in the even slots, V tiles in the odd ones
    bool ok = true;
    const int mask = bt.table ? (1 << bt.page_shift) - 1 : INT_MAX;
    while (ok && wk.next(bt, it)) {
      const int rows = __shfl_sync(0xffffffffu, it.len + it.n, 0);
      const int t0 = __shfl_sync(0xffffffffu, it.t0, 0), t1 = __shfl_sync(0xffffffffu, it.t1, 0);
      const int kvh = __shfl_sync(0xffffffffu, it.kvh, 0);
      const int pieces = (min(rows, t1 * BN) - t0 * BN + piece_rows - 1) / piece_rows;
      // pages are looked up a warp's width of pieces at a time
      const int lane_row = t0 * BN + lane * piece_rows;
      int pgs = lane < pieces ? table_entry(bt, it.b, lane_row) : 0;
      if (p == 0) {
        if (items > 0) ok = arrived(&sh.bar_qe, (items - 1) & 1, 0x33000);
        if (!ok) break;
        const int node = __shfl_sync(0xffffffffu, it.node0 + it.blk * block_nodes, 0);
        if (elect_one()) {
          mbar_arrive_expect_tx(&sh.bar_qf, (D / 64) * bt.rows_per_block * 128);
#pragma unroll
          for (int b = 0; b < D / 64; ++b)
            tma_load_3d(smem + b * C::kBoxQ, &tmQ, &sh.bar_qf, b * 64, kvh * bt.group, node);
        }
        ++items;
      }
      int i = 0;  // piece of the item
      for (int t = t0; t < t1; ++t) {
        if (round > 0) ok = arrived(&bar_empty[slot], (round & 1) ^ 1, 0x34000);
        if (!ok) break;
        const int end = min(i + BN / piece_rows, pieces);
        uint8_t* dst = smem + C::kRing + slot * C::kTileKV;
        if (elect_one()) mbar_arrive_expect_tx(&bar_full[slot], (end - i) * bytes);
        for (; i < end; ++i, dst += piece_rows * 128) {
          const int pg = checked_page(bt, it.b, __shfl_sync(0xffffffffu, pgs, i & 31));
          if ((i & 31) == 31) {
            const int next = i + 1 + lane;
            pgs = next < pieces ? table_entry(bt, it.b, t0 * BN + next * piece_rows) : 0;
          }
          const int row = (t0 * BN + i * piece_rows) & mask;
          if (elect_one()) {
            if (whole) {
              tma_load_5d(dst, map, &bar_full[slot], 0, row, 0, kvh, pg);
            } else {
#pragma unroll
              for (int b = 0; b < D / 64; ++b)
                tma_load_5d(dst + b * C::kBoxKV, map, &bar_full[slot], 0, row, b, kvh, pg);
            }
          }
        }
        slot += 2;
        if (slot >= kSlots) {
          slot = p;
          ++round;
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------ MMA issuer -----------------------------
    // The whole warp walks the loop and one elected lane issues.  Everything a
    // tcgen05.mma takes is then the same in all lanes and stays in uniform
    // registers; computed by a single lane it has to be moved there for every
    // instruction, about 100 cycles each, longer than the product itself.
    constexpr uint32_t idesc_qk = make_idesc<T>(kWideM, BN, false, false);
    constexpr uint32_t idesc_pv = make_idesc<T>(kWideM, D, false, true);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint32_t base = smem_u32(smem);
    const uint64_t dQ = sw128_desc(base, 16, 1024);
    const uint64_t dK0 = sw128_desc(base + C::kRing, 16, 1024);
    const uint64_t dV0 = sw128_desc(base + C::kRing, C::kBoxKV, 1024);
    constexpr uint32_t kSlotStep = C::kTileKV >> 4;
    uint32_t kslot = 0, kround = 0, items = 0, pvg = 0;  // K(jj)'s slot; V(jj)'s is the next
    uint32_t pcnt = 0;  // bit b: parity of S buffer b's next P
    // QK of a tile into S buffer sb, from ring slot `slot`
    auto qk = [&](uint32_t sb, uint32_t slot) {
      const uint64_t dk = dK0 + slot * kSlotStep;
      const uint32_t d_tm = tm + sb * BN;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          constexpr int q64 = C::kBoxQ >> 4, k64 = C::kBoxKV >> 4;
          tc_mma(d_tm, dQ + (kk >> 2) * q64 + (kk & 3) * 2, dk + (kk >> 2) * k64 + (kk & 3) * 2,
                 idesc_qk, kk > 0);
        }
        tc_commit(&sh.bar_sf[sb]);
        tc_commit(&bar_empty[slot]);
      }
    };
    auto next_k = [&]() {
      kslot += 2;
      if (kslot >= kSlots) {
        kslot = 0;
        kround ^= 1;
      }
    };
    bool ok = true;
    while (ok && wk.next(bt, it)) {
      const int n = __shfl_sync(0xffffffffu, it.t1 - it.t0, 0);
      if (!arrived(&sh.bar_qf, items & 1, 0x36000)) break;
      uint32_t vslot = kslot + 1, vround = kround;
      for (int jj = 0; ok && jj < C::kS && jj < n; ++jj) {
        ok = arrived(&bar_full[kslot], kround, 0x35000);
        tc_fence_after();
        if (ok) qk(jj, kslot);
        next_k();
      }
      if (ok && n <= C::kS && elect_one()) tc_commit(&sh.bar_qe);
      uint32_t sb = 0;
      for (int jj = 0; ok && jj < n; ++jj) {
        const bool more = jj + C::kS < n;
        // A wait takes some 150 cycles even where there is nothing to wait for;
        // asked together, the three barriers (V, the next K, P) answer in one.
        uint64_t *bv = &bar_full[vslot], *bk = &bar_full[more ? kslot : vslot], *bp = &sh.bar_pf[sb];
        const uint32_t kpar = more ? kround : vround, ppar = (pcnt >> sb) & 1;
        const bool v_in = mbar_test(bv, vround), k_in = mbar_test(bk, kpar), p_in = mbar_test(bp, ppar);
        if (!__all_sync(0xffffffffu, v_in && k_in && p_in))
          ok = arrived(bv, vround, 0x39000) && arrived(bk, kpar, 0x35800) && arrived(bp, ppar, 0x37000);
        if (ok && jj == 0 && items > 0) ok = arrived(&sh.bar_oe, (items - 1) & 1, 0x38000);
        pcnt ^= 1u << sb;
        if (!ok) break;
        tc_fence_after();
        const uint64_t dv = dV0 + vslot * kSlotStep;
        const uint32_t tp = tm + sb * BN;  // P: 16 keys per 8 columns
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk)
            tc_mma_ts(tm + kOCol, tp + kk * 8, dv + kk * 128, idesc_pv, jj > 0 || kk > 0);
          tc_commit(&sh.bar_pv[pvg & 1]);
          tc_commit(&bar_empty[vslot]);
          if (jj + 1 == n) tc_commit(&sh.bar_last);
        }
        ++pvg;
        vslot += 2;
        if (vslot >= kSlots) {
          vslot = 1;
          vround ^= 1;
        }
        if (more) {
          qk(sb, kslot);
          next_k();
          if (jj + C::kS + 1 == n && elect_one()) tc_commit(&sh.bar_qe);
        }
        if (++sb == C::kS) sb = 0;
      }
      ++items;
    }
  } else if (warp >= 4) {
    // ------------------------------ softmax ----------------------------------
    const int w = (warp - 4) >> 2;                 // warpgroup: tiles jj % 3 == w, S buffer w
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;             // row of the block == TMEM lane
    const uint32_t tl = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t ts = tl + w * BN;
    const int before_w = w == 0 ? kWideGroups - 1 : w - 1;  // whose tile comes before
    uint32_t own = 0, theirs = 0;  // tiles this warpgroup and that one have done
    uint32_t pvbase = 0, kslot = 0, kround = 0, items = 0;
    bool dead = false;  // a wait ran out: no more waiting, the barriers go on
    auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
      if (!dead) dead = !__all_sync(0xffffffffu, mbar_wait(bar, parity, where));
      return !dead;
    };
    auto meet = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(128 * kWideGroups) : "memory"); };
    zero_unwritten<T, D>(bt, sh.start.left_out, out, lse, warp - 4, 4 * kWideGroups);
    while (wk.next(bt, it)) {
      const int n = it.t1 - it.t0;
      const int rows = it.len + it.n;
      const int row0 = it.blk * bt.rows_per_block;
      const int live = min(bt.rows_per_block, it.n * bt.group - row0);
      const bool busy = quarter * 32 < live;  // this warp holds query rows
      const bool good = r < live;
      const int node = good ? (row0 + r) / bt.group : 0;
      const int head = it.kvh * bt.group + (good ? row0 + r - node * bt.group : 0);
      // the nodes that this row's node sees
      uint32_t anc[kWords];
#pragma unroll
      for (int i = 0; i < kWords; ++i) anc[i] = 0u;
      if (busy && it.t1 * BN > it.len) {
        int at = node;
        while (true) {
#pragma unroll
          for (int i = 0; i < kWords; ++i)
            if ((at >> 5) == i) anc[i] |= 1u << (at & 31);
          const int up = bt.parents ? __ldg(bt.parents + it.node0 + at) : at - 1;
          if (up < 0 || up >= at) {
            if (up != -1) set_dev_error(B2A_ERR_POSITION, it.b);
            break;
          }
          at = up;
        }
      }
      // 32 scores whose first key is tree row j0 (negative: cached rows): bit j
      // of the node's ancestors says whether it sees row j
      auto hide = [&](float* s, int j0) {
        if (j0 <= -32) return;
        const int lo = j0 >> 5, sft = j0 & 31;  // floor
        uint32_t a = lo < 0 ? 0xffffffffu : 0u, b = 0u;
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          if (lo == i) a = anc[i];
          if (lo + 1 == i) b = anc[i];
        }
        const uint32_t vis = sft ? (a >> sft) | (b << (32 - sft)) : a;
#pragma unroll
        for (int e = 0; e < 32; ++e) s[e] = ((vis >> e) & 1u) ? s[e] : -INFINITY;
      };
      float m = -INFINITY, l = 0.f;
      for (int jj = w; jj < n; jj += kWideGroups) {
        const int t = it.t0 + jj;
        const int tree0 = t * BN - it.len;  // tree row of the tile's first key
        const bool tail = tree0 + BN > 0;
        const bool alive = wait(&sh.bar_sf[w], own & 1, 0x3A000);
        ++own;
        tc_fence_after();
        if (busy && alive) {
          float mxa = -INFINITY, mxb = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < BN; c += 64) {
            float s[64];
            tc_ld32(ts + c, s);
            tc_ld32(ts + c + 32, s + 32);
            tc_wait_ld();
            if (tail) {
              hide(s, tree0 + c);
              hide(s + 32, tree0 + c + 32);
            }
#pragma unroll
            for (int e = 0; e < 64; e += 4) {
              mxa = fmaxf(mxa, fmaxf(s[e], s[e + 1]));
              mxb = fmaxf(mxb, fmaxf(s[e + 2], s[e + 3]));
            }
          }
          const float mx = fmaxf(mxa, mxb) * sscale;
          // the reference maximum up to the tile before
          float before = -INFINITY;
          if (jj > 0) {
            const uint32_t idx = theirs + (w == 0 ? jj / kWideGroups - 1 : jj / kWideGroups);
            if (wait(&sh.bar_m[before_w][quarter], idx & 1, 0x3B000)) before = sh.x[before_w][r];
          }
          // It only follows when a row's maximum grew by more than 2^8 (exact:
          // sums and O are relative to the same number).
          const bool grow = __any_sync(0xffffffffu, mx > before + prefill::kRescaleThreshold);
          const float now = grow ? fmaxf(before, mx) : before;
          sh.x[w][r] = now;
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.bar_m[w][quarter]);
          const float mref = (now == -INFINITY) ? 0.f : now;
          l *= (m == -INFINITY) ? 0.f : fast_exp2(m - mref);
          m = now;
          float suma = 0.f, sumb = 0.f;
#pragma unroll 1
          for (int c = 0; c < BN; c += 64) {
            float s[64];
            tc_ld32(ts + c, s);
            tc_ld32(ts + c + 32, s + 32);
            tc_wait_ld();
            if (tail) {
              hide(s, tree0 + c);
              hide(s + 32, tree0 + c + 32);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t pk[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const float p0 = fast_exp2(fmaf(s[h * 32 + 2 * e], sscale, -mref));
                const float p1 = fast_exp2(fmaf(s[h * 32 + 2 * e + 1], sscale, -mref));
                if (e & 1) sumb += p0 + p1; else suma += p0 + p1;
                pk[e] = Pack2<T>::run(p0, p1);
              }
              tc_st16(ts + (c >> 1) + h * 16, pk);
            }
          }
          tc_wait_st();
          l += suma + sumb;
          if (jj > 0 && grow) {
            // O is relative to the maximum before: rescale it after PV(jj - 1)
            const uint32_t g = pvbase + jj - 1;
            if (wait(&sh.bar_pv[g & 1], (g >> 1) & 1, 0x3C000)) {
              const float alpha = (before == -INFINITY) ? 0.f : fast_exp2(before - mref);
              tc_fence_after();
#pragma unroll 1
              for (int cc = 0; cc < D / 32; ++cc) {
                float o[32];
                tc_ld32(tl + kOCol + cc * 32, o);
                tc_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] *= alpha;
                tc_st32(tl + kOCol + cc * 32, o);
              }
              tc_wait_st();
            }
          }
          tc_fence_before();
        } else if (lane == 0) {
          mbar_arrive(&sh.bar_m[w][quarter]);  // keeps the barrier's count of tiles
        }
        const int first = max(it.len - t * BN, 0), past = min(rows - t * BN, BN);  // tree rows
        if (past < BN || (it.n > 1 && first < past)) {
          // V rows past the request's last hold anything: their weight is 0,
          // but 0 * NaN is not, so they are cleared before the product, and the
          // infinities and NaN of the tree's rows with them
          // (the slot's use before this one has to be over: its PV is, by S's
          // buffer, unless the ring is shorter than the S buffers)
          if (kSlots / 2 < C::kS && jj >= kSlots / 2) {
            const uint32_t g = pvbase + jj - kSlots / 2;
            wait(&sh.bar_pv[g & 1], (g >> 1) & 1, 0x3D800);
          }
          uint32_t vslot = kslot + 1 + 2 * jj, vround = kround;
          vround ^= (vslot / kSlots) & 1;
          vslot %= kSlots;
          if (wait(&bar_full[vslot], vround, 0x3D000)) {
            uint8_t* vt = smem + C::kRing + vslot * C::kTileKV;
            auto chunk = [&](int from, int i) {  // 16 bytes i of the rows from `from` on
              const int row = from + i / (D / 8), c16 = i % (D / 8);
              return reinterpret_cast<uint4*>(vt + (c16 >> 3) * C::kBoxKV + sw128_off(row, c16 & 7));
            };
            for (int i = r; i < (BN - past) * (D / 8); i += 128)
              *chunk(past, i) = make_uint4(0u, 0u, 0u, 0u);
            if (it.n > 1)
              for (int i = r; i < (past - first) * (D / 8); i += 128) {
                uint4 u = *chunk(first, i);
                if (clear_special<T>(u)) {
                  *chunk(first, i) = u;
                  sh.special = 1;
                }
              }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.bar_pf[w]);
      }
      theirs += (n - before_w + kWideGroups - 1) / kWideGroups;
      // ---------------- the item's end: the warpgroups' sums meet -----------
      meet();  // the last tile's maximum is the one that O is relative to
      const float M = sh.x[(n - 1) % kWideGroups][r];
      const float mref = (M == -INFINITY) ? 0.f : M;
      const bool special = sh.special != 0;
      meet();
      sh.x[w][r] = (m == -INFINITY) ? 0.f : l * fast_exp2(m - mref);
      meet();
      const float L = (sh.x[0][r] + sh.x[1][r]) + sh.x[2][r];
      wait(&sh.bar_last, items & 1, 0x3E000);
      ++items;
      tc_fence_after();
      const int slot = part_slot(it, blockIdx.x);
      const size_t row = static_cast<size_t>(it.node0 + node) * bt.H + head;
      const float f = L > 0.f ? 1.f / L : 0.f;
      float* po = part_o + (static_cast<size_t>(max(slot, 0)) * bt.rows_per_block + r) * D;
      if (busy && !dead) {
        // the warpgroups write the columns in turn
#pragma unroll 1
        for (int col = w * 32; col < D; col += 32 * kWideGroups) {
          float o[32];
          tc_ld32(tl + kOCol + col, o);
          tc_wait_ld();
          if (good) {
            if (slot >= 0) {
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                *reinterpret_cast<float4*>(po + col + e) =
                    make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            } else {
#pragma unroll
              for (int e = 0; e < 32; e += 8) {
                uint4 u;
                u.x = Pack2<T>::run(o[e] * f, o[e + 1] * f);
                u.y = Pack2<T>::run(o[e + 2] * f, o[e + 3] * f);
                u.z = Pack2<T>::run(o[e + 4] * f, o[e + 5] * f);
                u.w = Pack2<T>::run(o[e + 6] * f, o[e + 7] * f);
                *reinterpret_cast<uint4*>(out + row * D + col + e) = u;
              }
            }
          }
        }
        if (special && good) {
          const uint4 sees = make_uint4(anc[0], anc[1], anc[2], anc[3]);
          const int lo = max(it.t0 * BN - it.len, 0), hi = min(it.t1 * BN - it.len, it.n);
          for (int col = w * 32; col < D; col += 32 * kWideGroups) {
            if (slot >= 0)
              add_special(bt, vc, page_stride, it.b, it.kvh, it.len, lo, hi, sees, po + col, D, col, 32);
            else
              add_special(bt, vc, page_stride, it.b, it.kvh, it.len, lo, hi, sees, out + row * D + col,
                          D, col, 32);
          }
        }
        if (good && w == 0) {
          if (slot >= 0) {
            float* ml = part_ml + (static_cast<size_t>(slot) * bt.rows_per_block + r) * 2;
            ml[0] = M;
            ml[1] = L;
          } else if (lse) {
            lse[row] = L > 0.f ? (M + log2f(L)) * kLn2 : -INFINITY;
          }
        }
      }
      pvbase += n;
      kslot += 2 * (n % (kSlots / 2));
      kround ^= (n / (kSlots / 2)) & 1;
      if (kslot >= kSlots) {
        kslot -= kSlots;
        kround ^= 1;
      }
      tc_fence_before();
      if (special && threadIdx.x == 128) sh.special = 0;  // (all have read it: meet() above)
      meet();  // the exchanged numbers and O are read
      if (lane == 0) mbar_arrive(&sh.bar_oe);
    }
  }
  // ------------------------------ teardown -----------------------------------
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(prefill::kTmemCols));
  }
}

}  // namespace tree
}  // namespace b2a
