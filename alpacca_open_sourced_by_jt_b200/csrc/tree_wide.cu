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
// around them) takes longer than the tensor core's, so two warpgroups take the
// key tiles in turn and three S buffers keep both supplied: while they work on
// tiles j and j + 1, QK(j + 2) is done, and PV(j) frees its buffer for
// QK(j + 3).  What ties the warpgroups is the running maximum: the warp of tile
// j publishes its rows' maximum before its exponentials, and the other
// warpgroup's warp of the same rows goes on from there with tile j + 1.  Each
// keeps the sum of its own tiles relative to the last maximum it used; they
// meet at the item's end.  Warps whose 32 rows hold no query only pass the
// barriers.  (Both warpgroups on every tile, half of its keys each: their
// exponentials then fall together on one SFU and wait together for the next
// tile, 2000 cycles a tile.)
//
// 384 threads: warps 0 and 2 TMA producers (a box per page piece and 64
// columns, or one per tile where a page holds it), warp 1 TMEM owner and MMA
// issuer, warps 4-11 softmax (TMEM lane quarter = warp % 4).
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

constexpr int kWideThreads = 384;
constexpr int kWideM = 128;
constexpr int kMaxSlots = 16;

struct WideShared {
  uint64_t bar_qf, bar_qe, bar_oe, bar_last;  // bar_last: an item's last PV
  uint64_t bar_full[kMaxSlots], bar_empty[kMaxSlots];
  uint64_t bar_sf[3], bar_pf[3], bar_pv[2], bar_m[2][4];
  Start start;
  uint32_t tmem;
  float m[2][kWideM], l[2][kWideM];  // maxima and sums between the warpgroups
};

// One lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

template <int D>
struct WideCfg {
  static constexpr int kBN = D > 128 ? 64 : 128;      // keys per tile
  static constexpr int kS = 3;                        // S buffers
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
    T* __restrict__ out, float* __restrict__ lse, float* __restrict__ part_o,
    float* __restrict__ part_ml, int piece_rows, float sscale) {
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
    mbar_init(&sh.bar_oe, 8);
    mbar_init(&sh.bar_last, 1);
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&bar_full[s], 1);
      mbar_init(&bar_empty[s], 1);
    }
    for (int b = 0; b < C::kS; ++b) {
      mbar_init(&sh.bar_sf[b], 1);
      mbar_init(&sh.bar_pf[b], 4);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&sh.bar_pv[w], 1);
      for (int i = 0; i < 4; ++i) mbar_init(&sh.bar_m[w][i], 1);
    }
    fence_mbar_init();
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

  if (warp == 0 || warp == 2) {
    // ------------------------------ TMA producers --------------------------
    // One lane per warp issues: warp 0 loads Q and K, warp 2 V, so that a K
    // tile never queues behind a V tile whose slot is still in use.
    const int p = warp >> 1;
    const CUtensorMap* map = p ? &tmV : &tmK;
    const int boxes = piece_rows == BN ? 1 : D / 64;   // boxes of a page piece
    const int bytes = piece_rows * 128 * (D / 64);     // of a piece
    if (lane == 0) {
      if (p == 0) tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(map);
      uint32_t slot = p, round = 0, items = 0;  // K tiles in the even slots, V tiles in the odd ones
      bool ok = true;
      const int mask = bt.table ? (1 << bt.page_shift) - 1 : INT_MAX;
      while (ok && wk.next(bt, it)) {
        const int rows = it.len + it.n;
        int pg = table_entry(bt, it.b, it.t0 * BN);  // looked up one piece ahead
        if (p == 0) {
          if (items > 0 && !mbar_wait(&sh.bar_qe, (items - 1) & 1, 0x33000)) break;
          mbar_arrive_expect_tx(&sh.bar_qf, (D / 64) * bt.rows_per_block * 128);
#pragma unroll
          for (int b = 0; b < D / 64; ++b)
            tma_load_3d(smem + b * C::kBoxQ, &tmQ, &sh.bar_qf, b * 64, it.kvh * bt.group,
                        it.node0 + it.blk * block_nodes);
          ++items;
        }
        const int row_end = min(rows, it.t1 * BN);
        for (int t = it.t0; t < it.t1; ++t) {
          const int row0 = t * BN;
          const int end = min(row0 + BN, rows);
          if (round > 0 && !mbar_wait(&bar_empty[slot], (round & 1) ^ 1, 0x34000 | slot)) {
            ok = false;
            break;
          }
          uint8_t* dst = smem + C::kRing + slot * C::kTileKV;
          mbar_arrive_expect_tx(&bar_full[slot], (end - row0 + piece_rows - 1) / piece_rows * bytes);
          for (int row = row0; row < end; row += piece_rows, dst += piece_rows * 128) {
            const int now = checked_page(bt, it.b, pg);
            if (row + piece_rows < row_end) pg = table_entry(bt, it.b, row + piece_rows);
            for (int b = 0; b < boxes; ++b)
              tma_load_5d(dst + b * C::kBoxKV, map, &bar_full[slot], 0, row & mask, b, it.kvh, now);
          }
          slot += 2;
          if (slot >= kSlots) {
            slot = p;
            ++round;
          }
        }
      }
    }
    __syncwarp();
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
    auto arrived = [&](uint64_t* bar, uint32_t parity, int where) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, where)) != 0;
    };
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
        // waits that do not depend on P(jj) come before the one that does
        ok = arrived(&bar_full[vslot], vround, 0x39000);
        if (ok && more) ok = arrived(&bar_full[kslot], kround, 0x35800);
        if (ok && jj == 0 && items > 0) ok = arrived(&sh.bar_oe, (items - 1) & 1, 0x38000);
        if (ok) ok = arrived(&sh.bar_pf[sb], (pcnt >> sb) & 1, 0x37000);
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
    const int w = (warp - 4) >> 2;                 // warpgroup: tiles jj % 2 == w
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;             // row of the block == TMEM lane
    const uint32_t tl = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    uint32_t scnt = 0;       // bit b: parity of S buffer b's next tile (all tiles of the CTA)
    uint32_t mdone[2] = {0, 0};  // tiles each warpgroup has done
    uint32_t pvbase = 0, kslot = 0, kround = 0, items = 0;
    bool dead = false;  // a wait ran out: no more waiting, the barriers go on
    auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
      if (!dead) dead = !__all_sync(0xffffffffu, mbar_wait(bar, parity, where));
      return !dead;
    };
    // rows past the last node (the padding of a captured step) become zeros
    if (blockIdx.x == 0) {
      const long long first = static_cast<long long>(max(bt.cu[bt.B], 0)) * bt.H;
      for (long long i = first + warp - 4; i < static_cast<long long>(bt.n_tok) * bt.H; i += 8) {
        for (int d = lane; d < D; d += 32) st_elem(out + i * D + d, 0.f);
        if (lse && lane == 0) lse[i] = -INFINITY;
      }
    }
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
      float m = -INFINITY, l = 0.f;
      int sb = 0;
      for (int jj = 0; jj < n; ++jj) {
        const uint32_t s_col = sb * BN;
        uint64_t *sf = &sh.bar_sf[sb], *pf = &sh.bar_pf[sb];
        const uint32_t sparity = (scnt >> sb) & 1;
        scnt ^= 1u << sb;
        if (++sb == C::kS) sb = 0;
        if ((jj & 1) != w) continue;
        const int t = it.t0 + jj;
        const bool alive = wait(sf, sparity, 0x3A000);
        tc_fence_after();
        if (busy && alive) {
          float s[BN];
#pragma unroll
          for (int q32 = 0; q32 < BN / 32; ++q32) tc_ld32(tl + s_col + q32 * 32, s + q32 * 32);
          tc_wait_ld();
          if ((t + 1) * BN > it.len) {
            // tree rows: bit j of the node's ancestors for key len + j
#pragma unroll
            for (int wd = 0; wd < BN / 32; ++wd) {
              const int j0 = t * BN + wd * 32 - it.len;  // node of the word's first key
              uint32_t vis = 0xffffffffu;
              if (j0 > -32) {
                const int lo = j0 >> 5, sft = j0 & 31;  // floor
                uint32_t a = lo < 0 ? 0xffffffffu : 0u, b = 0u;
#pragma unroll
                for (int i = 0; i < kWords; ++i) {
                  if (lo == i) a = anc[i];
                  if (lo + 1 == i) b = anc[i];
                }
                vis = sft ? (a >> sft) | (b << (32 - sft)) : a;
              }
#pragma unroll
              for (int e = 0; e < 32; ++e)
                s[wd * 32 + e] = ((vis >> e) & 1u) ? s[wd * 32 + e] : -INFINITY;
            }
          }
          float mxa = -INFINITY, mxb = -INFINITY, mxc = -INFINITY, mxd = -INFINITY;
#pragma unroll
          for (int cc = 0; cc < BN; cc += 4) {
            mxa = fmaxf(mxa, s[cc]);
            mxb = fmaxf(mxb, s[cc + 1]);
            mxc = fmaxf(mxc, s[cc + 2]);
            mxd = fmaxf(mxd, s[cc + 3]);
          }
          const float mx = fmaxf(fmaxf(mxa, mxb), fmaxf(mxc, mxd)) * sscale;
          // the reference maximum up to the tile before
          float before = -INFINITY;
          if (jj > 0) {
            const uint32_t theirs = mdone[w ^ 1] + ((jj - 1) >> 1);
            if (wait(&sh.bar_m[w ^ 1][quarter], theirs & 1, 0x3B000)) before = sh.m[w ^ 1][r];
          }
          // It only follows when a row's maximum grew by more than 2^8 (exact:
          // sums and O are relative to the same number).
          const bool grow = __any_sync(0xffffffffu, mx > before + prefill::kRescaleThreshold);
          const float now = grow ? fmaxf(before, mx) : before;
          sh.m[w][r] = now;
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.bar_m[w][quarter]);
          const float mref = (now == -INFINITY) ? 0.f : now;
          l *= (m == -INFINITY) ? 0.f : fast_exp2(m - mref);
          m = now;
          float suma = 0.f, sumb = 0.f;
#pragma unroll
          for (int qtr = 0; qtr < BN / 32; ++qtr) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float p0 = fast_exp2(fmaf(s[qtr * 32 + 2 * e], sscale, -mref));
              const float p1 = fast_exp2(fmaf(s[qtr * 32 + 2 * e + 1], sscale, -mref));
              if (e & 1) sumb += p0 + p1; else suma += p0 + p1;
              pk[e] = Pack2<T>::run(p0, p1);
            }
            tc_st16(tl + s_col + qtr * 16, pk);
          }
          tc_wait_st();
          l += suma + sumb;
          if (jj > 0 && grow) {
            // O is relative to the maximum before: rescale it after PV(jj - 1)
            const uint32_t g = pvbase + jj - 1;
            if (wait(&sh.bar_pv[g & 1], (g >> 1) & 1, 0x3C000)) {
              const float alpha = (before == -INFINITY) ? 0.f : fast_exp2(before - mref);
              tc_fence_after();
#pragma unroll
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
        if ((t + 1) * BN > rows) {
          // V rows past the request's last hold anything: their weight is 0,
          // but 0 * NaN is not, so they are cleared before the product
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
            const int bad = max(rows - t * BN, 0);
            uint8_t* vt = smem + C::kRing + vslot * C::kTileKV;
            for (int i = r; i < (BN - bad) * (D / 8); i += 128) {
              const int row = bad + i / (D / 8), c16 = i % (D / 8);
              *reinterpret_cast<uint4*>(vt + (c16 >> 3) * C::kBoxKV + sw128_off(row, c16 & 7)) =
                  make_uint4(0u, 0u, 0u, 0u);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(pf);
      }
      // ---------------- the item's end: both warpgroups' sums meet ----------
      sh.l[w][r] = l;
      sh.m[w][r] = m;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      const float ma = sh.m[0][r], mb = sh.m[1][r];
      const float M = fmaxf(ma, mb);
      const float mref = (M == -INFINITY) ? 0.f : M;
      const float L = sh.l[0][r] * fast_exp2(ma - mref) + sh.l[1][r] * fast_exp2(mb - mref);
      wait(&sh.bar_last, items & 1, 0x3E000);
      ++items;
      tc_fence_after();
      const int slot = part_slot(it, blockIdx.x);
      const size_t row = static_cast<size_t>(it.node0 + node) * bt.H + head;
      const float f = L > 0.f ? 1.f / L : 0.f;
      float* po = part_o + (static_cast<size_t>(max(slot, 0)) * bt.rows_per_block + r) * D;
      if (busy && !dead) {
        // each warpgroup writes half of the columns
#pragma unroll
        for (int cc = 0; cc < D / 64; ++cc) {
          const int col = w * (D / 2) + cc * 32;
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
      mdone[0] += (n + 1) >> 1;
      mdone[1] += n >> 1;
      pvbase += n;
      kslot += 2 * (n % (kSlots / 2));
      kround ^= (n / (kSlots / 2)) & 1;
      if (kslot >= kSlots) {
        kslot -= kSlots;
        kround ^= 1;
      }
      tc_fence_before();
      asm volatile("bar.sync 1, 256;" ::: "memory");  // m, l and O are read
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
