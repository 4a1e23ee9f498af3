// Tree attention over a 4-bit cache with many query rows (nodes x query heads of a KV
// head): the schedule of tree_wide.cu on tcgen05, with the tiles made from codes.
//
// A block of up to 128 rows is the M of tcgen05.mma; S = Q.K^T and O += P.V accumulate
// in TMEM, P goes over S's columns and Q stays in TMEM too, so that shared memory
// carries only the tiles.  Converting warps turn each granule of 16 keys into rows of the
// K and V tiles, 128-byte swizzled as the MMAs read them: a code at bits 6 to 9 of 0x4c00
// is the f16 16 + code, and (16 + code) d - 24 d, one fused operation, is d * (code - 8)
// exactly (24 d has 10 bits).  So both products are those of the cache's own values; q is
// scaled by a power of two to f16 as in tree_q4.cu, the weights are rounded to f16.
//
// 896 threads: warps 0-7 softmax (two warpgroups, tiles in turn, an S buffer each),
// 8-23 converters, 24 feeds them (as tree_q4_kernel's warps are fed, here by steps of 16
// keys), 25 owns TMEM and issues the MMAs.
// TMEM: S0, S1 (128 columns each), O (D), Q (D / 2).
//
// Bound by instructions and the waits between them (54 % of the issue slots used, no pipe
// above 40 %): a tile of 128 keys takes some 5700 with 32 rows, half for
// the conversion, which a block of 128 rows repeats, half for the softmax.  16 x 32760
// rows, 32/8 heads x 128: 32 rows 302 us (2.0 TB/s), 64 rows 354, 128 rows 451; 8 requests
// of 9K to 16K rows, up to 512 query rows a KV head: 366 us, 450 TFLOP/s.  With converters
// that bring their own steps a tenth more for 32 rows.

#include <limits.h>

#include <type_traits>

#include "b2a_common.cuh"
#include "q4.cuh"
#include "tree_work.cuh"

namespace b2a {
namespace tree {

constexpr int kQWGroups = 2;     // softmax warpgroups
constexpr int kQWConvert = 16;   // converting warps
constexpr int kQWPlan = 8 + kQWConvert, kQWIssue = kQWPlan + 1;  // the planning and the issuing warp
constexpr int kQWThreads = (kQWIssue + 3) * 32;  // whole warpgroups
// Registers: 896 x 72 at launch; softmax 104, converters 56, the last four warps 72.
constexpr int kQWSoftmaxRegs = 104, kQWConvertRegs = 56;
static_assert(256 * kQWSoftmaxRegs + kQWConvert * 32 * kQWConvertRegs + 128 * 72 <= kQWThreads * 72, "registers");
constexpr int kQWKeys = 128;     // keys per tile
constexpr int kQWSlots = 2;      // K tiles, and V tiles, in shared memory

template <int S>
struct alignas(128) QWShared {
  static constexpr int kStepKeys = 16, kTileSteps = kQWKeys / 16;  // a step is a granule
  uint64_t full[kQWConvert][S], empty[kQWConvert][S];  // a converter's stages
  uint64_t item_full[kQ4Queue], item_empty[kQ4Queue];  // feeding warp -> all others
  uint64_t k_full[kQWSlots], k_empty[kQWSlots], v_full[kQWSlots], v_empty[kQWSlots];
  uint64_t q_full, last;                               // an item's Q, its last PV
  uint64_t s_full[kQWGroups], p_full[kQWGroups], pv[2], bar_m[kQWGroups][4];
  uint32_t tmem;
  int special[8];  // an item's tree rows held NaN (converters are less than 8 items ahead)
  Q4Item item[kQ4Queue];
  float x[kQWGroups][128];  // maxima, at an item's end sums, between the warpgroups
  float o[128][33];         // rows of O, where several lanes share a query row
};

template <int D>
struct QWCfg {
  static constexpr int kGranule = q4::granule_bytes(D);
  static constexpr int kStage = kGranule;
  static constexpr int kBox = kQWKeys * 128;        // 128 rows x 64 columns
  static constexpr int kTile = (D / 64) * kBox;     // one K or V tile
  static constexpr int kTiles = 2 * kQWSlots * kTile;
  static constexpr int kFit = (227 * 1024 - kTiles - static_cast<int>(sizeof(QWShared<4>))) / (kQWConvert * kStage);
  static constexpr int kStages = kFit > 4 ? 4 : kFit;
  using Shared = QWShared<kStages>;
  static constexpr int kSmem = kTiles + kQWConvert * kStages * kStage + static_cast<int>(sizeof(Shared));
  static_assert(kStages >= 2 && kSmem <= 227 * 1024, "ring");
  // A converter takes every kQWConvert-th of all steps, so at least one of the tiles in
  // the slots: further apart, it could not tell the phase of a slot by its parity.
  static_assert(kQWConvert <= kQWSlots * Shared::kTileSteps, "converters");
};

// Does a tree row j in [lo, hi) that the node sees have a NaN scale in V's block?
__device__ __noinline__ bool q4_special(const Batch& bt, const q4::Pool& pool, int D, int b, int kvh, int len,
                                        int lo, int hi, uint4 anc, int block) {
  for (int j = lo; j < hi; ++j) {
    const uint32_t word = j < 32 ? anc.x : j < 64 ? anc.y : j < 96 ? anc.z : anc.w;
    if (!((word >> (j & 31)) & 1u)) continue;
    const int row = len + j;
    const int pg = checked_page(bt, b, table_entry(bt, b, row));
    if (pg >= bt.n_pages) continue;
    const int in_page = bt.table ? row & ((1 << bt.page_shift) - 1) : row;
    const unsigned char* g = q4::granule(pool, D, pg, kvh, in_page);
    const uint16_t h = *reinterpret_cast<const uint16_t*>(g + q4::v_scale(D, in_page & 15, block));
    if ((h & 0x7fffu) > 0x7c00u) return true;
  }
  return false;
}

// 8 values of a word: code places 0 to 3 give dims (0, 1), (2, 3), (4, 5), (6, 7).
template <bool kLarge>  // 24 d is past f16
__device__ __forceinline__ uint4 q4_values(uint32_t w, __half2 d, __half2 d24) {
  uint32_t x[4] = {((w << 6) & 0x03c003c0u) | 0x4c004c00u, ((w << 2) & 0x03c003c0u) | 0x4c004c00u,
                   ((w >> 2) & 0x03c003c0u) | 0x4c004c00u, ((w >> 6) & 0x03c003c0u) | 0x4c004c00u};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 c = *reinterpret_cast<const __half2*>(&x[i]);
    const __half2 y = kLarge ? __hmul2(__hsub2(c, __float2half2_rn(24.f)), d) : __hfma2(c, d, d24);
    x[i] = *reinterpret_cast<const uint32_t*>(&y);
  }
  return make_uint4(x[0], x[1], x[2], x[3]);
}

template <typename T, int D>
__global__ void __launch_bounds__(kQWThreads, 1) tree_q4_wide_kernel(
    const __grid_constant__ Batch bt, const __grid_constant__ q4::Pool pool, const T* __restrict__ q,
    long long q_stride, T* __restrict__ out, float* __restrict__ lse, float* __restrict__ part_o,
    float* __restrict__ part_ml, float scale_log2, int rep_shift) {
  using C = QWCfg<D>;
  constexpr int BN = kQWKeys, TS = C::Shared::kTileSteps, W = kQWConvert, NB = D / 32;
  constexpr uint32_t kOCol = kQWGroups * BN, kQCol = kOCol + D;
  static_assert(kQCol + D / 2 <= 512, "TMEM columns");
  extern __shared__ __align__(1024) uint8_t qw_smem[];
  typename C::Shared& sh = *reinterpret_cast<typename C::Shared*>(qw_smem + C::kTiles + W * C::kStages * C::kStage);

  pdl_wait();
  if (smem_u32(qw_smem) & 1023u) {  // swizzled tiles start on 1024-byte boundaries
    if (threadIdx.x == 0) set_dev_error(B2A_ERR_ALIGN, 0x3F800);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == kQWIssue) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&sh.tmem)),
                 "r"(prefill::kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else if (warp == kQWPlan && lane == 0) {
    for (int w = 0; w < W; ++w)
      for (int s = 0; s < C::kStages; ++s) {
        mbar_init(&sh.full[w][s], 1);
        mbar_init(&sh.empty[w][s], 1);
      }
    for (int i = 0; i < kQ4Queue; ++i) {
      mbar_init(&sh.item_full[i], 1);
      mbar_init(&sh.item_empty[i], 1 + 4 * kQWGroups + W);
    }
    for (int i = 0; i < kQWSlots; ++i) {
      mbar_init(&sh.k_full[i], TS);
      mbar_init(&sh.k_empty[i], 1);
      mbar_init(&sh.v_full[i], TS);
      mbar_init(&sh.v_empty[i], 1);
    }
    mbar_init(&sh.q_full, 4 * kQWGroups);
    mbar_init(&sh.last, 1);
    for (int w = 0; w < kQWGroups; ++w) {
      mbar_init(&sh.s_full[w], 1);
      mbar_init(&sh.p_full[w], 4);
      for (int i = 0; i < 4; ++i) mbar_init(&sh.bar_m[w][i], 1);
    }
    mbar_init(&sh.pv[0], 1);
    mbar_init(&sh.pv[1], 1);
    fence_mbar_init();
    for (int i = 0; i < 8; ++i) sh.special[i] = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = sh.tmem;
  // a whole warp's wait on a barrier, with one answer for all lanes
  auto arrived = [](uint64_t* bar, uint32_t parity, int where) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, where)) != 0;
  };

  if (warp == kQWPlan) {
    // ------------------------------ the plan, the copies --------------------
    q4_feed<W, C::kStages, D>(bt, pool, sh, qw_smem + C::kTiles, lane);
  } else if (warp == kQWIssue) {
    // ------------------------------ MMA issuer -----------------------------
    // (the whole warp walks, one elected lane issues: tree_wide.cu says why)
    constexpr uint32_t idesc_qk = make_idesc<__half>(128, BN, false, false);
    constexpr uint32_t idesc_pv = make_idesc<__half>(128, D, false, true);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint32_t base = smem_u32(qw_smem);
    const uint64_t dK0 = sw128_desc(base, 16, 1024);
    const uint64_t dV0 = sw128_desc(base + kQWSlots * C::kTile, C::kBox, 1024);
    constexpr uint32_t kSlotStep = C::kTile >> 4;
    uint32_t kt = 0, vt = 0;  // K and V tiles taken
    uint32_t items = 0, pvg = 0, pcnt = 0;
    auto qk = [&](uint32_t sb) {
      const uint32_t slot = kt % kQWSlots;
      const uint64_t dk = dK0 + slot * kSlotStep;
      const uint32_t d_tm = tm + sb * BN;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          constexpr int k64 = C::kBox >> 4;
          tc_mma_ts(d_tm, tm + kQCol + kk * 8, dk + (kk >> 2) * k64 + (kk & 3) * 2, idesc_qk, kk > 0);
        }
        tc_commit(&sh.s_full[sb]);
        tc_commit(&sh.k_empty[slot]);
      }
      ++kt;
    };
    bool ok = true;
    while (ok) {
      const int place = items % kQ4Queue;
      if (!arrived(&sh.item_full[place], (items / kQ4Queue) & 1, 0x3F810)) break;
      const int end = sh.item[place].end;
      const int n = __shfl_sync(0xffffffffu, sh.item[place].it.t1 - sh.item[place].it.t0, 0);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.item_empty[place]);
      if (end) break;
      if (!arrived(&sh.q_full, items & 1, 0x3F820)) break;
      tc_fence_after();
      for (int jj = 0; ok && jj < kQWGroups && jj < n; ++jj) {
        ok = arrived(&sh.k_full[kt % kQWSlots], (kt / kQWSlots) & 1, 0x3F830);
        tc_fence_after();
        if (ok) qk(jj);
      }
      uint32_t sb = 0;
      for (int jj = 0; ok && jj < n; ++jj) {
        const bool more = jj + kQWGroups < n;
        // asked together, the three barriers (V, the next K, P) answer in one
        const uint32_t vslot = vt % kQWSlots, vpar = (vt / kQWSlots) & 1, ppar = (pcnt >> sb) & 1;
        uint64_t* bk = more ? &sh.k_full[kt % kQWSlots] : &sh.v_full[vslot];
        const uint32_t kpar = more ? (kt / kQWSlots) & 1 : vpar;
        const bool v_in = mbar_test(&sh.v_full[vslot], vpar), k_in = mbar_test(bk, kpar),
                   p_in = mbar_test(&sh.p_full[sb], ppar);
        if (!__all_sync(0xffffffffu, v_in && k_in && p_in))
          ok = arrived(&sh.v_full[vslot], vpar, 0x3F840) && arrived(&sh.p_full[sb], ppar, 0x3F850);
        pcnt ^= 1u << sb;
        if (!ok) break;
        tc_fence_after();
        const uint64_t dv = dV0 + vslot * kSlotStep;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk)
            tc_mma_ts(tm + kOCol, tm + sb * BN + kk * 8, dv + kk * 128, idesc_pv, jj > 0 || kk > 0);
          tc_commit(&sh.pv[pvg & 1]);
          tc_commit(&sh.v_empty[vslot]);
          if (jj + 1 == n) tc_commit(&sh.last);
        }
        ++pvg;
        ++vt;
        if (more) {
          ok = arrived(bk, kpar, 0x3F860);
          tc_fence_after();
          if (ok) qk(sb);
        }
        if (++sb == kQWGroups) sb = 0;
      }
      ++items;
    }
  } else if (warp >= 8 && warp < kQWPlan) {
    // ------------------------------ converters -------------------------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kQWConvertRegs));
    const int cw = warp - 8;
    uint8_t* ring = qw_smem + C::kTiles + cw * C::kStages * C::kStage;
    uint32_t stage = 0, phase = 0, items = 0;
    bool ok = true;
    for (; ok; ++items) {
      const int place = items % kQ4Queue;
      if (!arrived(&sh.item_full[place], (items / kQ4Queue) & 1, 0x3F870)) break;
      const Q4Item& entry = sh.item[place];
      if (entry.end) break;
      const int len = entry.it.len, rows = len + entry.it.n, g0 = entry.g0;
      const int s0 = entry.it.t0 * TS, steps = entry.it.t1 * TS - s0;
      const bool tree = entry.it.n > 1;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.item_empty[place]);
      for (int i = (cw + W - g0 % W) % W; i < steps; i += W) {
        const int st = s0 + i;
        const uint32_t tile = (g0 + i) / TS;
        const uint32_t slot = tile % kQWSlots, round = tile / kQWSlots;
        if (!arrived(&sh.full[cw][stage], phase, 0x3F880)) {
          ok = false;
          break;
        }
        const int part = lane >> 4, r = lane & 15;   // two lanes to a row
        const uint8_t* g = ring + stage * C::kStage;
        const int at = st * 16 + r;                  // row of the cache
        const bool none = at >= rows;
        // the row in a tile, swizzled: chunk c is at `swz` with c & 7 in bits 4 to 6 flipped
        const uint32_t key = (st % TS) * 16 + r, swz = key * 128 + ((key & 7) << 4);
        // scales of K and V, [block] f16; of rows that are not there 0
        uint32_t dk[NB / 2], dv[NB / 2];
#pragma unroll
        for (int i = 0; i < NB / 2; ++i) {
          dk[i] = *reinterpret_cast<const uint32_t*>(g + 16 * D + r * (2 * NB) + i * 4);
          dv[i] = *reinterpret_cast<const uint32_t*>(g + 17 * D + r * (2 * NB) + i * 4);
        }
        if (st * 16 + 16 > len) {  // rows of the tree, or past the last
#pragma unroll
          for (int i = 0; i < NB / 2; ++i) {
            if (none) dk[i] = dv[i] = 0u;
            if (tree && at >= len) {
              // a NaN that some rows do not see: taken out here, put back at the item's end
              if ((dv[i] & 0x7fffu) > 0x7c00u) {
                dv[i] &= 0xffff0000u;
                sh.special[items & 7] = 1;
              }
              if ((dv[i] & 0x7fff0000u) > 0x7c000000u) {
                dv[i] &= 0x0000ffffu;
                sh.special[items & 7] = 1;
              }
            }
          }
        }
        __half2 most = __float2half2_rn(0.f);
#pragma unroll
        for (int i = 0; i < NB / 2; ++i) {
          most = __hmax2(most, __habs2(*reinterpret_cast<const __half2*>(&dk[i])));
          most = __hmax2(most, __habs2(*reinterpret_cast<const __half2*>(&dv[i])));
        }
        const bool large = __any_sync(0xffffffffu, !__hble2(most, __float2half2_rn(2048.f)));
        const __half2 m24 = __float2half2_rn(-24.f);
        auto scale_of = [](const uint32_t* d, int b) {
          const uint32_t u = __byte_perm(d[b >> 1], 0u, b & 1 ? 0x3232u : 0x1010u);
          return *reinterpret_cast<const __half2*>(&u);
        };
        auto convert_k = [&](uint8_t* kt, auto is_large) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int t = 2 * part + ((j + (r >> 1)) & 1);  // (rows begin at different words: fewer bank conflicts)
            uint32_t w[4];
            if constexpr (NB >= 4) {
              const uint4 u = *reinterpret_cast<const uint4*>(g + r * 64 + t * 16);
              w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
            } else {
              const uint2 u = *reinterpret_cast<const uint2*>(g + r * 32 + t * 8);
              w[0] = u.x; w[1] = u.y;
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              const __half2 d = scale_of(dk, b);  // (chunk 4 b + t of the row)
              *reinterpret_cast<uint4*>(kt + (b >> 1) * C::kBox + ((swz ^ (t << 4)) ^ ((b & 1) << 6))) =
                  q4_values<decltype(is_large)::value>(w[b], d, __hmul2(d, m24));
            }
          }
        };
        auto convert_v = [&](uint8_t* vt, auto is_large) {
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const __half2 d = scale_of(dv, b), d24 = __hmul2(d, m24);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int t = 2 * j + part;
              const uint32_t w = *reinterpret_cast<const uint32_t*>(g + 8 * D + (4 * b + t) * 64 + r * 4);
              *reinterpret_cast<uint4*>(vt + (b >> 1) * C::kBox + ((swz ^ (t << 4)) ^ ((b & 1) << 6))) =
                  q4_values<decltype(is_large)::value>(w, d, d24);
            }
          }
        };
        // ---- K ----
        if (round > 0 && !arrived(&sh.k_empty[slot], (round & 1) ^ 1, 0x3F890)) {
          ok = false;
          break;
        }
        uint8_t* kt = qw_smem + slot * C::kTile;
        if (large) convert_k(kt, std::true_type());
        else convert_k(kt, std::false_type());
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.k_full[slot]);
        // ---- V ----
        if (round > 0 && !arrived(&sh.v_empty[slot], (round & 1) ^ 1, 0x3F8A0)) {
          ok = false;
          break;
        }
        uint8_t* vt = qw_smem + (kQWSlots + slot) * C::kTile;
        if (large) convert_v(vt, std::true_type());
        else convert_v(vt, std::false_type());
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.v_full[slot]);
        // (the stage is read by then)
        if (lane == 0) mbar_arrive(&sh.empty[cw][stage]);
        if (++stage == C::kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp < 8) {
    // ------------------------------ softmax ----------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kQWSoftmaxRegs));
    const int w = warp >> 2;                       // warpgroup: tiles jj % 2 == w, S buffer w
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;             // row of the block == TMEM lane
    const uint32_t tl = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t ts = tl + w * BN;
    const int before_w = 1 - w;                    // whose tile comes before
    const int lanes_of = 128 >> rep_shift;         // query rows of a block
    const int rr = r & (lanes_of - 1);             // the lane's query row
    const int width = BN >> rep_shift, c0 = (r >> (7 - rep_shift)) * width;  // its keys of a tile
    uint32_t own = 0, theirs = 0;  // tiles this warpgroup and that one have done
    uint32_t pvbase = 0, items = 0;
    int end = 0;
    bool dead = false;  // a wait of this warp ran out: no more waiting, the barriers go on
    auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
      if (!dead) dead = !__all_sync(0xffffffffu, mbar_wait(bar, parity, where));
      return !dead;
    };
    auto meet = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(128 * kQWGroups) : "memory"); };
    // meet(), and whether one of the eight warps says so.  A wait may run out in some warps
    // only, so what decides which barriers follow is decided here, by all alike.
    auto any_of = [&](bool says) {
      uint32_t any;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\t"
          "setp.ne.u32 p, %1, 0;\n\t"
          "bar.red.or.pred q, 1, %2, p;\n\t"
          "selp.u32 %0, 1, 0, q;\n\t}"
          : "=r"(any)
          : "r"(static_cast<uint32_t>(says)), "n"(128 * kQWGroups)
          : "memory");
      return any != 0u;
    };
    while (true) {
      const int place = items % kQ4Queue;
      // (waited for whatever ran out before)
      if (any_of(!arrived(&sh.item_full[place], (items / kQ4Queue) & 1, 0x3F8B0))) break;
      end = sh.item[place].end;
      const Item it = sh.item[place].it;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.item_empty[place]);
      if (end) break;
      const int n = it.t1 - it.t0;
      const int row0 = it.blk * bt.rows_per_block;
      const int live = min(bt.rows_per_block, it.n * bt.group - row0);
      const bool busy = (rr & ~31) < live;  // this warp holds query rows
      const bool good = rr < live;
      const int node = good ? (row0 + rr) / bt.group : 0;
      const int head = it.kvh * bt.group + (good ? row0 + rr - node * bt.group : 0);
      // ---- the row of q, scaled to f16, into TMEM: half of it by each warpgroup -----------
      float sscale;
      {
        const T* qr = q + (it.node0 + node) * q_stride + head * D;
        float big = 0.f;
        if (good) {
#pragma unroll 4
          for (int d = 0; d < D; d += 8) {
            float x[8];
            paged::load8(qr + d, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(x[e]));
          }
        }
        int k = 0;  // big * 2^k in [2^14, 2^15); rows of zeros, infinities: 0
        if (big > 0.f && big < INFINITY) k = max(-126, min(126, 14 + 127 - static_cast<int>(__float_as_uint(big) >> 23)));
        const float up = __uint_as_float(static_cast<uint32_t>(127 + k) << 23);
        sscale = scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
#pragma unroll
        for (int c = 0; c < D / 2; c += 32) {  // 32 dims are 16 columns
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = 0.f;
            if (good) paged::load8(qr + w * (D / 2) + c + e * 8, x);
#pragma unroll
            for (int i = 0; i < 4; ++i) pk[e * 4 + i] = Pack2<__half>::run(x[2 * i] * up, x[2 * i + 1] * up);
          }
          tc_st16(tl + kQCol + (w * (D / 2) + c) / 2, pk);
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.q_full);
      }
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
      // 32 scores whose first key is tree row j0 (negative: cached rows): bit j of the
      // node's ancestors says whether it sees row j
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
      for (int jj = w; jj < n; jj += kQWGroups) {
        const int tree0 = (it.t0 + jj) * BN - it.len;  // tree row of the tile's first key
        const bool tail = tree0 + BN > 0;
        const bool alive = wait(&sh.s_full[w], own & 1, 0x3F8C0);
        ++own;
        tc_fence_after();
        if (busy && alive) {
          float mxa = -INFINITY, mxb = -INFINITY;
          float s[32];  // (the last 32 of the lane's keys, which are all of them for 4 lanes a row)
#pragma unroll 1
          for (int c = c0; c < c0 + width; c += 32) {
            tc_ld32(ts + c, s);
            tc_wait_ld();
            if (tail) hide(s, tree0 + c);
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              mxa = fmaxf(mxa, fmaxf(s[e], s[e + 1]));
              mxb = fmaxf(mxb, fmaxf(s[e + 2], s[e + 3]));
            }
          }
          const float mx = fmaxf(mxa, mxb) * sscale;
          // the reference maximum up to the tile before
          float before = -INFINITY;
          if (jj > 0) {
            const uint32_t idx = theirs + (w == 0 ? jj / kQWGroups - 1 : jj / kQWGroups);
            if (wait(&sh.bar_m[before_w][quarter], idx & 1, 0x3F8D0)) before = sh.x[before_w][r];
          }
          // It only follows when a row's maximum grew by more than 2^8 (exact: sums and O
          // are relative to the same number).
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
          for (int c = c0; c < c0 + width; c += 32) {
            if (width > 32) {
              tc_ld32(ts + c, s);
              tc_wait_ld();
              if (tail) hide(s, tree0 + c);
            }
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float p0 = fast_exp2(fmaf(s[2 * e], sscale, -mref));
              const float p1 = fast_exp2(fmaf(s[2 * e + 1], sscale, -mref));
              if (e & 1) sumb += p0 + p1; else suma += p0 + p1;
              pk[e] = Pack2<__half>::run(p0, p1);
            }
            tc_st16(ts + (c >> 1), pk);
          }
          if (rep_shift) {
            // the tile's other keys are other lanes': weight 0 here
            uint32_t zero[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) zero[e] = 0u;
#pragma unroll 1
            for (int c = 0; c < BN; c += 32)
              if (c < c0 || c >= c0 + width) tc_st16(ts + (c >> 1), zero);
          }
          tc_wait_st();
          l += suma + sumb;
          if (jj > 0 && grow) {
            // O is relative to the maximum before: rescale it after PV(jj - 1)
            const uint32_t g = pvbase + jj - 1;
            if (wait(&sh.pv[g & 1], (g >> 1) & 1, 0x3F8E0)) {
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
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_full[w]);
      }
      theirs += (n - before_w + kQWGroups - 1) / kQWGroups;
      // ---------------- the item's end: the warpgroups' sums meet -----------
      meet();  // the last tile's maximum is the one that O is relative to
      const float M = sh.x[(n - 1) % kQWGroups][r];
      const float mref = (M == -INFINITY) ? 0.f : M;
      meet();
      sh.x[w][r] = (m == -INFINITY) ? 0.f : l * fast_exp2(m - mref);
      wait(&sh.last, items & 1, 0x3F8F0);
      const bool lost = any_of(dead);
      dead = lost;
      const float L = sh.x[0][r] + sh.x[1][r];
      const uint32_t which = items & 7;
      ++items;
      tc_fence_after();
      const bool special = sh.special[which] != 0;  // (all of the item's tiles are converted)
      const int slot = part_slot(it, blockIdx.x);
      const size_t row = static_cast<size_t>(it.node0 + node) * bt.H + head;
      const float f = L > 0.f ? 1.f / L : 0.f;
      const int lo = max(it.t0 * BN - it.len, 0), hi = min(it.t1 * BN - it.len, it.n);
      const uint4 sees = make_uint4(anc[0], anc[1], anc[2], anc[3]);
      float* po = part_o + (static_cast<size_t>(max(slot, 0)) * bt.rows_per_block + r) * D;
      if (rep_shift == 0 && busy && !lost) {
        // the warpgroups write the columns in turn, 32 (a block) at a time
#pragma unroll 1
        for (int col = w * 32; col < D; col += 32 * kQWGroups) {
          float o[32];
          tc_ld32(tl + kOCol + col, o);
          tc_wait_ld();
          if (good) {
            if (special && q4_special(bt, pool, D, it.b, it.kvh, it.len, lo, hi,
                                      sees, col / 32)) {
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __uint_as_float(0x7fffffffu);
            }
            if (slot >= 0) {
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                *reinterpret_cast<float4*>(po + col + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] *= f;
#pragma unroll
              for (int e = 0; e < 32; e += 8) paged::store8(out + row * D + col + e, o + e);
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
      if (rep_shift) {
        // Several lanes share a query row, each with its own keys' sums relative to its own
        // maximum: they meet in shared memory, 32 columns at a time.
        meet();  // (L has been read)
        if (w == 0) {
          sh.x[0][r] = M;
          sh.x[1][r] = L;
        }
        meet();
        if (w == 0 && !lost) {
          float top = -INFINITY, sum = 0.f;
          for (int i = rr; i < 128; i += lanes_of) top = fmaxf(top, sh.x[0][i]);
          const float tref = top == -INFINITY ? 0.f : top;
          for (int i = rr; i < 128; i += lanes_of) sum = fmaf(sh.x[1][i], fast_exp2(sh.x[0][i] - tref), sum);
          const float mine = M == -INFINITY ? 0.f : fast_exp2(M - tref) * (slot >= 0 ? 1.f : (sum > 0.f ? 1.f / sum : 0.f));
#pragma unroll 1
          for (int col = 0; col < D; col += 32) {
            float o[32];
            tc_ld32(tl + kOCol + col, o);
            tc_wait_ld();
            const bool gone = special && good && q4_special(bt, pool, D, it.b, it.kvh, it.len, lo, hi, sees, col / 32);
#pragma unroll
            for (int e = 0; e < 32; ++e) sh.o[r][e] = gone ? __uint_as_float(0x7fffffffu) : o[e] * mine;
            asm volatile("bar.sync 2, 128;" ::: "memory");
            for (int i = threadIdx.x; i < live * 4; i += 128) {
              const int qr = i >> 2, at = (i & 3) * 8;
              float x[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = 0.f;
              for (int j = qr; j < 128; j += lanes_of) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] += sh.o[j][at + e];
              }
              const int nd = (row0 + qr) / bt.group;
              if (slot >= 0)
                paged::store8(part_o + (static_cast<size_t>(slot) * bt.rows_per_block + qr) * D + col + at, x);
              else
                paged::store8(out + (static_cast<size_t>(it.node0 + nd) * bt.H + it.kvh * bt.group + row0 + qr - nd * bt.group) * D + col + at, x);
            }
            asm volatile("bar.sync 2, 128;" ::: "memory");
          }
          if (good && r < lanes_of) {
            if (slot >= 0) {
              float* ml = part_ml + (static_cast<size_t>(slot) * bt.rows_per_block + rr) * 2;
              ml[0] = top;
              ml[1] = sum;
            } else if (lse) {
              lse[row] = sum > 0.f ? (top + log2f(sum)) * kLn2 : -INFINITY;
            }
          }
        }
      }
      pvbase += n;
      tc_fence_before();
      meet();  // the exchanged numbers and O are read
      if (special && threadIdx.x == 0) sh.special[which] = 0;
    }
    if (!dead) zero_unwritten<T, D>(bt, end == 2, out, lse, warp, 4 * kQWGroups);
  }
  // ------------------------------ teardown -----------------------------------
  tc_fence_before();
  __syncthreads();
  if (warp == kQWIssue) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(prefill::kTmemCols));
  }
}

}  // namespace tree
}  // namespace b2a

// ===========================================================================
// Host side
// ===========================================================================
namespace {

// Which kernel, by the most rows a KV head can have, and the rows of an item.  16 x 32760
// rows, 32/8 heads x 128: 16 rows 270 us with warp-level MMAs, 299 on tcgen05; 32 rows
// (two blocks of 16) 485 against 302.
bool tree_q4_is_wide(int rows, int D) { return rows > 16 && D <= 128; }
// (the wide kernel: as many lanes of 128 to a row as the most rows leave; 32 rows 428 us with
// one lane to a row, 339 with two, 302 with four; 64 rows 439, with two 354)
int tree_q4_rep(int rows) { return rows <= 32 ? 2 : rows <= 64 ? 1 : 0; }
int tree_q4_rows(int rows, int D, int group) {
  if (tree_q4_is_wide(rows, D)) return (128 >> tree_q4_rep(rows)) / group * group;
  return rows <= 8 || D > 128 ? 8 : 16;
}

template <typename T, int D, int NT>
int tree_q4_launch(const TreeArgs& a, const Q4::Pool& pool) {
  auto kern = TR::tree_q4_kernel<T, D, NT>;
  using C = TR::Q4Cfg<D, NT>;
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = allow_smem(kern, C::kSmem, done);
  if (e != cudaSuccess) return b2a_host::cuda_fail(e, "cudaFuncSetAttribute(tree_decode_q4)");
  e = b2a_host::launch(kern, dim3(a.grid), dim3(C::kThreads), C::kSmem, a.st, a.bt, pool,
                       static_cast<const T*>(a.q), a.q_stride, static_cast<T*>(a.out), a.lse, a.part_o,
                       a.part_ml, a.sscale);
  if (e != cudaSuccess) return b2a_host::cuda_fail(e, "tree_decode_q4 launch");
  return tree_merge<T, D>(a);
}

template <typename T, int D>
int tree_q4_wide_launch(const TreeArgs& a, const Q4::Pool& pool) {
  auto kern = TR::tree_q4_wide_kernel<T, D>;
  using C = TR::QWCfg<D>;
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = allow_smem(kern, C::kSmem, done);
  if (e != cudaSuccess) return b2a_host::cuda_fail(e, "cudaFuncSetAttribute(tree_decode_q4)");
  e = b2a_host::launch(kern, dim3(a.grid), dim3(TR::kQWThreads), C::kSmem, a.st, a.bt, pool,
                       static_cast<const T*>(a.q), a.q_stride, static_cast<T*>(a.out), a.lse, a.part_o,
                       a.part_ml, a.sscale, tree_q4_rep(a.bt.rows_per_block));
  if (e != cudaSuccess) return b2a_host::cuda_fail(e, "tree_decode_q4 wide launch");
  return tree_merge<T, D>(a);
}

template <typename T, int D>
int tree_q4_dispatch(const TreeArgs& a, const Q4::Pool& pool) {
  if constexpr (D <= 128) {
    if (a.bt.tile == TR::kQWKeys) return tree_q4_wide_launch<T, D>(a, pool);
    if (a.bt.rows_per_block == 16) return tree_q4_launch<T, D, 2>(a, pool);
  }
  return tree_q4_launch<T, D, 1>(a, pool);
}

template <typename T>
int tree_q4_type(const TreeArgs& a, const Q4::Pool& pool) {
  if (a.D == 64) return tree_q4_dispatch<T, 64>(a, pool);
  if (a.D == 128) return tree_q4_dispatch<T, 128>(a, pool);
  return tree_q4_dispatch<T, 256>(a, pool);
}

}  // namespace

extern "C" {

size_t b2a_tree_decode_q4_workspace_bytes(int max_nodes, int H, int KV, int D, int max_len) {
  if (max_nodes <= 0 || H <= 0 || KV <= 0 || D <= 0 || H % KV != 0) return 0;
  if (H / KV > 128 || tree_always_whole(max_len)) return 0;
  const int rb = tree_q4_rows(max_nodes * (H / KV), D, H / KV);
  return tree_part_o_bytes(D, KV, rb) + static_cast<size_t>(2) * tree_ctas(KV) * rb * 2 * sizeof(float);
}

int b2a_tree_decode_q4(const void* q, long long q_tok_stride, const void* pool, int n_pages,
                       int page_rows, long long page_bytes, const int* table_dev,
                       long long table_stride, int table_width, const int* lens_dev,
                       const int* cu_dev, const int* parents_dev, void* out, float* lse_out,
                       void* workspace, size_t workspace_bytes, int B, int n_tok, int max_nodes, int H,
                       int KV, int D, int dtype, float scale, int max_len, void* stream) {
  if (!q || !lens_dev || !cu_dev || !out) return fail(B2A_ERR_ARG, "tree_decode_q4: null pointer argument");
  if (B <= 0 || n_tok < 0 || H <= 0 || max_len <= 0)
    return fail(B2A_ERR_ARG, "tree_decode_q4: sizes must be positive (B=%d n_tok=%d H=%d max_len=%d)", B, n_tok, H, max_len);
  if (max_nodes <= 0 || max_nodes > B2A_TREE_MAX_NODES)
    return fail(B2A_ERR_ARG, "tree_decode_q4: max_nodes %d (1..%d)", max_nodes, B2A_TREE_MAX_NODES);
  const int rc = q4_pool_check("tree_decode_q4", pool, n_pages, page_rows, page_bytes, KV, D, table_dev != nullptr);
  if (rc) return rc;
  if (H % KV != 0) return fail(B2A_ERR_SHAPE, "tree_decode_q4: H=%d is not a multiple of KV=%d", H, KV);
  if (dtype != B2A_F16 && dtype != B2A_BF16) return fail(B2A_ERR_DTYPE, "tree_decode_q4: dtype %d", dtype);
  if (!(scale > 0.f) || !isfinite(scale)) return fail(B2A_ERR_ARG, "tree_decode_q4: scale must be positive");
  if (table_dev) {
    if (table_width <= 0 || table_stride < table_width ||
        static_cast<long long>(table_width) * page_rows < max_len)
      return fail(B2A_ERR_SHAPE, "tree_decode_q4: a table row of %d pages (stride %lld) does not hold max_len %d rows",
                  table_width, table_stride, max_len);
  } else if (n_pages < B || page_rows < max_len) {
    return fail(B2A_ERR_SHAPE, "tree_decode_q4: %d blocks of %d rows for %d sequences of up to %d",
                n_pages, page_rows, B, max_len);
  }
  if (q_tok_stride == 0) q_tok_stride = static_cast<long long>(H) * D;
  if (q_tok_stride < static_cast<long long>(H) * D)
    return fail(B2A_ERR_SHAPE, "tree_decode_q4: q_tok_stride %lld < H*D", q_tok_stride);
  if (!b2a_host::aligned16(q) || !b2a_host::aligned16(out) || !b2a_host::aligned16(workspace) ||
      (q_tok_stride * 2) % 16 != 0)
    return fail(B2A_ERR_ALIGN, "tree_decode_q4: q, its stride, out and workspace must be 16-byte aligned");
  if (n_tok == 0) return B2A_OK;
  const int group = H / KV;
  if (group > 128) return fail(B2A_ERR_UNSUPPORTED, "tree_decode_q4: group %d", group);

  TreeArgs a = {};
  const int rows = max_nodes * group;
  const bool wide = tree_q4_is_wide(rows, D);
  const int rb = tree_q4_rows(rows, D, group);
  const int tile = wide ? TR::kQWKeys : TR::kQ4Keys;
  a.bt = TR::Batch{lens_dev, cu_dev, parents_dev, table_dev, table_stride, B, n_tok, max_nodes, max_len,
                   n_pages, table_dev ? log2_of(page_rows) : 0, H, KV, group, rb, tile, 0, 1, 1, 1, 1};
  // Side by side in a team: the KV heads, or, where a request has several blocks of
  // query rows, those (b2a_tree_decode's rule)
  const long long avg_rows = static_cast<long long>(n_tok) * group / B;
  long long blks = (avg_rows + rb / 2) / rb;
  const int most = max_rows_blocks(rows, rb);
  if (blks > most || 4 * blks >= 3 * most) blks = most;
  if (blks > kTreeBlocks) blks = (blks + (blks + kTreeBlocks - 1) / kTreeBlocks - 1) / ((blks + kTreeBlocks - 1) / kTreeBlocks);
  a.bt.m_blks = blks > 1 ? static_cast<int>(blks) : 1;
  a.bt.m_heads = a.bt.m_blks > 1 ? 1 : KV;
  const int members = a.bt.m_heads * a.bt.m_blks;
  const long long max_tiles = (max_len + tile - 1) / tile;
  const long long items = static_cast<long long>(B) * (KV / a.bt.m_heads) * ((most + a.bt.m_blks - 1) / a.bt.m_blks);
  a.bt.by_item = tree_by_item(max_len, B, KV) ? 1 : 0;
  a.bt.min_units = a.bt.by_item ? 1 : wide ? 4 : 8;
  const long long units = (items * (a.bt.by_item ? 1 : max_tiles) + a.bt.min_units - 1) / a.bt.min_units;
  const int teams = b2a_host::sm_count() > members ? b2a_host::sm_count() / members : 1;
  a.bt.teams = static_cast<int>(units < teams ? units : teams);
  a.grid = a.bt.teams * members;
  a.merge = !a.bt.by_item;
  if (a.merge) {
    const size_t need = b2a_tree_decode_q4_workspace_bytes(max_nodes, H, KV, D, max_len);
    if (!workspace || workspace_bytes < need)
      return fail(B2A_ERR_WORKSPACE, "tree_decode_q4: workspace %zu bytes < %zu needed", workspace_bytes, need);
  }
  a.q = q;
  a.q_stride = q_tok_stride;
  a.out = out;
  a.lse = lse_out;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = workspace ? reinterpret_cast<float*>(static_cast<char*>(workspace) + tree_part_o_bytes(D, KV, rb)) : nullptr;
  a.D = D;
  a.dtype = dtype;
  a.sscale = scale * TR::kLog2e;
  a.st = static_cast<cudaStream_t>(stream);
  const Q4::Pool p = q4_pool_of(pool, n_pages, page_rows, page_bytes, D, table_dev != nullptr);
  if (dtype == B2A_BF16) return tree_q4_type<__nv_bfloat16>(a, p);
  return tree_q4_type<__half>(a, p);
}

}  // extern "C"
