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
// A thread's 128 exponentials take about twice the tensor core's time for a
// tile, so two warpgroups share every tile: warpgroup w takes half w of the
// tile's keys for all rows.  The two warps of a row exchange their maxima
// through shared memory (one 64-thread barrier a tile); each keeps the sum of
// its own keys.  With S double-buffered the tensor core runs QK(j + 1) and
// PV(j - 1) while both work on tile j.  Q lives in TMEM as 16-bit pairs (A of
// QK): reading it from shared memory for every product took as much of the
// shared-memory bandwidth as K, and its space is better used for tiles in
// flight.  Warps whose 32 rows hold no query only pass the barriers.
//
// 384 threads: warps 0, 2, 3 TMA producers (a box per page piece and 64
// columns, or one per tile where a page holds it), warp 1 TMEM owner and MMA
// issuer, warps 4-11 softmax (TMEM lane quarter = warp % 4).
// TMEM: S0 [0, BN), S1 [BN, 2 BN), O [2 BN, 2 BN + D), Q [2 BN + D, + D / 2).

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
using prefill::tc_mma_ts;
using prefill::tc_st16;
using prefill::tc_st32;
using prefill::tc_wait_ld;
using prefill::tc_wait_st;

constexpr int kWideThreads = 384;
constexpr int kWideM = 128;

template <int D>
struct WideCfg {
  static constexpr int kBN = D > 128 ? 64 : 128;      // keys per tile
  static constexpr int kBoxKV = kBN * 128;            // kBN rows x 64 columns
  static constexpr int kTileKV = (D / 64) * kBoxKV;   // one K or V tile
  static constexpr int kSlots = 192 * 1024 / kTileKV;
  static constexpr int kSmem = kSlots * kTileKV + 1024;
  static_assert(2 * kBN + D + D / 2 <= 512, "TMEM columns");
  // a K or V tile's slot has the same producer on every use, and the softmax
  // waits on a V slot only after K's of the same tile (see below)
  static_assert(kSlots % 2 == 0, "ring");
};

template <typename T, int D>
__global__ void __launch_bounds__(kWideThreads, 1) tree_wide_kernel(
    const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
    const __grid_constant__ Batch bt, const T* __restrict__ q, long long q_stride,
    T* __restrict__ out, float* __restrict__ lse, float* __restrict__ part_o,
    float* __restrict__ part_ml, int piece_rows, float sscale) {
  using C = WideCfg<D>;
  constexpr int BN = C::kBN;
  constexpr int kSlots = C::kSlots;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_qf, bar_oe;
  __shared__ __align__(8) uint64_t bar_full[kSlots], bar_empty[kSlots];
  __shared__ __align__(8) uint64_t bar_sf[2], bar_pf[2], bar_pv[2];
  __shared__ uint32_t s_tmem;
  __shared__ Start s_start;
  __shared__ float s_x[2][2][kWideM];  // maxima (and at the end sums) of a row's two warps

  pdl_wait();
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    const Start s = locate(bt, blockIdx.x / bt.KV);
    if (lane == 0) s_start = s;
  } else if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&s_tmem)),
                 "r"(prefill::kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else if (warp == 2 && lane == 0) {
    mbar_init(&bar_qf, 8);
    mbar_init(&bar_oe, 8);
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&bar_full[s], piece_rows == BN ? 1 : 3);
      mbar_init(&bar_empty[s], 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&bar_sf[w], 1);
      mbar_init(&bar_pf[w], 8);
      mbar_init(&bar_pv[w], 1);
    }
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = s_tmem;
  const int kvh = blockIdx.x % bt.KV;
  Walker wk;
  wk.start(bt, s_start);
  Item it;

  constexpr uint32_t kOCol = 2 * BN, kQCol = 2 * BN + D;

  if (warp < 4 && warp != 1) {
    // ------------------------------ TMA producers --------------------------
    // One lane per warp issues.  Where a page holds whole tiles warp 0 loads K
    // and warp 2 V, one box each; smaller pages are dealt to all three (an
    // issue takes a thread about a hundred cycles).
    const int p = warp > 0 ? warp - 1 : 0;
    const bool whole = piece_rows == BN;
    const int bytes = piece_rows * 128 * (D / 64);
    if (lane == 0 && (p < 2 || !whole)) {
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
      uint32_t slot = whole ? p : 0, round = 0;  // K tiles in the even slots, V tiles in the odd ones
      bool ok = true;
      const int mask = bt.table ? (1 << bt.page_shift) - 1 : INT_MAX;
      while (ok && wk.next(bt, it)) {
        const int rows = it.len + it.n;
        int pg = whole ? table_entry(bt, it.b, it.t0 * BN) : 0;
        for (int t = it.t0; ok && t < it.t1; ++t) {
          const int row0 = t * BN;
          if (whole) {
            const int now = checked_page(bt, it.b, pg);
            if (t + 1 < it.t1) pg = table_entry(bt, it.b, row0 + BN);
            if (round > 0 && !mbar_wait(&bar_empty[slot], (round & 1) ^ 1, 0x34000 | slot)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&bar_full[slot], bytes);
            tma_load_5d(smem + slot * C::kTileKV, p ? &tmV : &tmK, &bar_full[slot], 0, row0 & mask,
                        0, kvh, now);
            slot += 2;
          } else {
            // this warp's pieces of the tile, K then V
            const int pieces = (min(BN, rows - row0) + piece_rows - 1) / piece_rows;  // with rows
            const int n_mine = p < pieces ? (pieces - p + 2) / 3 : 0;
            for (int kv = 0; kv < 2; ++kv, ++slot) {
              if (round > 0 && !mbar_wait(&bar_empty[slot], (round & 1) ^ 1, 0x34000 | slot)) {
                ok = false;
                break;
              }
              mbar_arrive_expect_tx(&bar_full[slot], n_mine * bytes);
              for (int i = p; i < pieces; i += 3) {
                const int row = row0 + i * piece_rows;
                const int now = checked_page(bt, it.b, table_entry(bt, it.b, row));
#pragma unroll
                for (int b = 0; b < D / 64; ++b)
                  tma_load_5d(smem + slot * C::kTileKV + b * C::kBoxKV + i * piece_rows * 128,
                              kv ? &tmV : &tmK, &bar_full[slot], 0, row & mask, b, kvh, now);
              }
            }
          }
          if (slot >= kSlots) {
            slot -= kSlots;
            ++round;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------ MMA issuer -----------------------------
    if (lane == 0) {
      constexpr uint32_t idesc_qk = make_idesc<T>(kWideM, BN, false, false);
      constexpr uint32_t idesc_pv = make_idesc<T>(kWideM, D, false, true);
      const uint64_t dK0 = sw128_desc(smem_u32(smem), 16, 1024);
      const uint64_t dV0 = sw128_desc(smem_u32(smem), C::kBoxKV, 1024);
      constexpr uint64_t kSlotStep = C::kTileKV >> 4;
      uint32_t seq = 0, items = 0, pvg = 0;
      uint32_t pcnt[2] = {0, 0};
      bool ok = true;
      auto qk = [&](int jj, uint32_t ksq) {
        const uint32_t slot = ksq % kSlots;
        if (!mbar_wait(&bar_full[slot], (ksq / kSlots) & 1, 0x35000 | slot)) return false;
        tc_fence_after();
        const uint64_t dk = dK0 + slot * kSlotStep;
        const uint32_t d_tm = tmem + (jj & 1) * BN;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint64_t koff = (((kk >> 2) * C::kBoxKV) + (kk & 3) * 32) >> 4;
          tc_mma_ts(d_tm, tmem + kQCol + kk * 8, dk + koff, idesc_qk, kk > 0);
        }
        tc_commit(&bar_sf[jj & 1]);
        tc_commit(&bar_empty[slot]);
        return true;
      };
      while (ok && wk.next(bt, it)) {
        const int n = it.t1 - it.t0;
        if (!mbar_wait(&bar_qf, items & 1, 0x36000)) break;
        const uint32_t base = seq;  // K of tile jj at base + 2 jj, V behind it
        seq += 2 * n;
        for (int jj = 0; ok && jj < 2 && jj < n; ++jj) ok = qk(jj, base + 2 * jj);
        for (int jj = 0; ok && jj < n; ++jj) {
          const uint32_t vsq = base + 2 * jj + 1, slot = vsq % kSlots;
          uint32_t& pc = pcnt[jj & 1];
          ok = mbar_wait(&bar_pf[jj & 1], pc & 1, 0x37000);
          ++pc;
          if (ok && jj == 0 && items > 0) ok = mbar_wait(&bar_oe, (items - 1) & 1, 0x38000);
          if (ok) ok = mbar_wait(&bar_full[slot], (vsq / kSlots) & 1, 0x39000 | slot);
          if (!ok) break;
          tc_fence_after();
          const uint64_t dv = dV0 + slot * kSlotStep;
          const uint32_t tp = tmem + (jj & 1) * BN;  // P: 16 keys per 8 columns
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk)
            tc_mma_ts(tmem + kOCol, tp + kk * 8, dv + ((kk * 16 * 128) >> 4), idesc_pv,
                      jj > 0 || kk > 0);
          tc_commit(&bar_pv[pvg & 1]);
          ++pvg;
          tc_commit(&bar_empty[slot]);
          if (jj + 2 < n) ok = qk(jj + 2, base + 2 * (jj + 2));
        }
        ++items;
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ------------------------------ softmax ----------------------------------
    constexpr int HK = BN / 2;                     // keys of a thread
    const int w = (warp - 4) >> 2;                 // which half of a tile's keys
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;             // row of the block == TMEM lane
    const uint32_t tl = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    uint32_t cnt[2] = {0, 0};                      // tiles done in each S buffer
    uint32_t pvbase = 0, seq = 0;
    bool dead = false;  // a wait ran out: no more waiting, the barriers go on
    auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
      if (!dead) dead = !__all_sync(0xffffffffu, mbar_wait(bar, parity, where));
      return !dead;
    };
    auto meet = [&]() {  // the two warps of the same rows
      asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
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
      const int head = kvh * bt.group + (good ? row0 + r - node * bt.group : 0);
      // Q's row into TMEM, half of its columns by each warp (the last item's
      // products are complete: every warp waited for its last PV)
      if (busy) {
        const uint4* src = reinterpret_cast<const uint4*>(q + (it.node0 + node) * q_stride +
                                                          static_cast<long long>(head) * D + w * (D / 2));
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {  // 32 elements: 16 TMEM columns
          uint32_t u[16];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint4 x = good ? src[c * 4 + e] : make_uint4(0u, 0u, 0u, 0u);
            u[4 * e] = x.x;
            u[4 * e + 1] = x.y;
            u[4 * e + 2] = x.z;
            u[4 * e + 3] = x.w;
          }
          tc_st16(tl + kQCol + w * (D / 4) + c * 16, u);
        }
        tc_wait_st();
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_qf);
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
      for (int jj = 0; jj < n; ++jj) {
        const int t = it.t0 + jj;
        const uint32_t s_col = (jj & 1) * BN;
        wait(&bar_sf[jj & 1], (cnt[jj & 1] + (jj >> 1)) & 1, 0x3A000);
        tc_fence_after();
        if (busy) {
          float s[HK];
#pragma unroll
          for (int q32 = 0; q32 < HK / 32; ++q32)
            tc_ld32(tl + s_col + w * HK + q32 * 32, s + q32 * 32);
          tc_wait_ld();
          if ((t + 1) * BN > it.len) {
            // tree rows: bit j of the node's ancestors for key len + j
#pragma unroll
            for (int wd = 0; wd < HK / 32; ++wd) {
              const int j0 = t * BN + w * HK + wd * 32 - it.len;  // node of the word's first key
              uint32_t vis = 0xffffffffu;
              if (j0 > -32) {
                const int lo = j0 >> 5, sh = j0 & 31;  // floor
                uint32_t a = lo < 0 ? 0xffffffffu : 0u, b = 0u;
#pragma unroll
                for (int i = 0; i < kWords; ++i) {
                  if (lo == i) a = anc[i];
                  if (lo + 1 == i) b = anc[i];
                }
                vis = sh ? (a >> sh) | (b << (32 - sh)) : a;
              }
#pragma unroll
              for (int e = 0; e < 32; ++e)
                s[wd * 32 + e] = ((vis >> e) & 1u) ? s[wd * 32 + e] : -INFINITY;
            }
          }
          float mxa = -INFINITY, mxb = -INFINITY, mxc = -INFINITY, mxd = -INFINITY;
#pragma unroll
          for (int cc = 0; cc < HK; cc += 4) {
            mxa = fmaxf(mxa, s[cc]);
            mxb = fmaxf(mxb, s[cc + 1]);
            mxc = fmaxf(mxc, s[cc + 2]);
            mxd = fmaxf(mxd, s[cc + 3]);
          }
          float mx = fmaxf(fmaxf(mxa, mxb), fmaxf(mxc, mxd));
          s_x[jj & 1][w][r] = mx;
          // the other warp's P goes over columns of S that this one has read
          tc_fence_before();
          meet();
          tc_fence_after();
          mx = fmaxf(mx, s_x[jj & 1][w ^ 1][r]) * sscale;
          // The reference maximum only follows when it grew by more than 2^8
          // (exact: l and O share it); both warps see the same numbers.
          const float before = m;
          const bool grow = __any_sync(0xffffffffu, mx > before + prefill::kRescaleThreshold);
          if (grow) m = fmaxf(before, mx);
          const float mref = (m == -INFINITY) ? 0.f : m;
          float suma = 0.f, sumb = 0.f;
#pragma unroll
          for (int qtr = 0; qtr < HK / 32; ++qtr) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float p0 = fast_exp2(fmaf(s[qtr * 32 + 2 * e], sscale, -mref));
              const float p1 = fast_exp2(fmaf(s[qtr * 32 + 2 * e + 1], sscale, -mref));
              if (e & 1) sumb += p0 + p1; else suma += p0 + p1;
              pk[e] = Pack2<T>::run(p0, p1);
            }
            tc_st16(tl + s_col + w * (HK / 2) + qtr * 16, pk);
          }
          tc_wait_st();
          if (grow) {
            const float alpha = (before == -INFINITY) ? 0.f : fast_exp2(before - mref);
            l *= alpha;
            if (jj > 0) {
              // O is relative to the maximum before: rescale it after PV(jj - 1)
              const uint32_t g = pvbase + jj - 1;
              if (wait(&bar_pv[g & 1], (g >> 1) & 1, 0x3C000)) {
                tc_fence_after();
#pragma unroll
                for (int cc = 0; cc < D / 64; ++cc) {
                  float o[32];
                  tc_ld32(tl + kOCol + w * (D / 2) + cc * 32, o);
                  tc_wait_ld();
#pragma unroll
                  for (int e = 0; e < 32; ++e) o[e] *= alpha;
                  tc_st32(tl + kOCol + w * (D / 2) + cc * 32, o);
                }
                tc_wait_st();
              }
            }
          }
          l += suma + sumb;
          tc_fence_before();
        }
        if ((t + 1) * BN > rows) {
          // V rows past the request's last hold anything: their weight is 0,
          // but 0 * NaN is not, so they are cleared before the product
          const uint32_t vsq = seq + 2 * jj + 1, slot = vsq % kSlots;
          if (wait(&bar_full[slot], (vsq / kSlots) & 1, 0x3D000)) {
            const int bad = max(rows - t * BN, 0);
            uint8_t* vt = smem + slot * C::kTileKV;
            for (int i = w * 128 + r; i < (BN - bad) * (D / 8); i += 256) {
              const int row = bad + i / (D / 8), c16 = i % (D / 8);
              *reinterpret_cast<uint4*>(vt + (c16 >> 3) * C::kBoxKV + sw128_off(row, c16 & 7)) =
                  make_uint4(0u, 0u, 0u, 0u);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_pf[jj & 1]);
      }
      // ---------------- the item's end: both warps' sums meet ---------------
      float L = l;
      if (busy) {
        s_x[n & 1][w][r] = l;
        meet();
        L += s_x[n & 1][w ^ 1][r];
      }
      const uint32_t g = pvbase + n - 1;
      wait(&bar_pv[g & 1], (g >> 1) & 1, 0x3E000);
      tc_fence_after();
      const int slot = part_slot(it, blockIdx.x);
      const size_t row = static_cast<size_t>(it.node0 + node) * bt.H + head;
      const float f = L > 0.f ? 1.f / L : 0.f;
      float* po = part_o + (static_cast<size_t>(max(slot, 0)) * bt.rows_per_block + r) * D;
      if (busy && !dead) {
        // each warp writes half of the columns
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
            ml[0] = m;
            ml[1] = L;
          } else if (lse) {
            lse[row] = L > 0.f ? (m + log2f(L)) * kLn2 : -INFINITY;
          }
        }
      }
      cnt[0] += (n + 1) >> 1;
      cnt[1] += n >> 1;
      pvbase += n;
      seq += 2 * n;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_oe);
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
