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
// One softmax warpgroup needs about twice the tensor core's time for a tile
// (128 exponentials a thread), so two warpgroups take the key tiles in turn:
// warpgroup w owns S buffer w and tiles jj with jj % 2 = w.  What ties them is
// the running maximum: the warp of tile jj publishes its rows' maximum as soon
// as it has it, before its exponentials, and the other warpgroup's warp of the
// same rows goes on from there with tile jj + 1.  Each keeps the sum of its own
// tiles relative to the last maximum it used; they meet at the item's end.
// Warps whose 32 rows hold no query do nothing but pass the barriers.
//
// 384 threads: warp 0 TMA producer of Q and K, warp 2 of V (a box per page
// piece and 64 columns, or one per tile where a page holds it), warp 1 TMEM
// owner and MMA issuer, warps 4-11 softmax (TMEM lane quarter = warp % 4).
// TMEM: S0 [0, BN), S1 [BN, 2 BN), O [2 BN, 2 BN + D).

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

template <int D>
struct WideCfg {
  static constexpr int kBN = D > 128 ? 64 : 128;      // keys per tile
  static constexpr int kBoxQ = kWideM * 128;          // 128 rows x 64 columns
  static constexpr int kBoxKV = kBN * 128;
  static constexpr int kTileQ = (D / 64) * kBoxQ;
  static constexpr int kTileKV = (D / 64) * kBoxKV;   // one K or V tile
  static constexpr int kSlots = (225 * 1024 - kTileQ) / kTileKV > 10
                                    ? 10 : (225 * 1024 - kTileQ) / kTileKV - (D > 64 ? 1 : 0);
  static constexpr int kRing = kTileQ;
  static constexpr int kSmem = kTileQ + kSlots * kTileKV + 1024;
  static_assert(kSmem + 8192 <= 232448, "shared memory per CTA");
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
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_qf, bar_qe, bar_oe;
  __shared__ __align__(8) uint64_t bar_full[kSlots], bar_empty[kSlots];
  __shared__ __align__(8) uint64_t bar_sf[2], bar_pf[2], bar_pv[2], bar_m[2][4];
  __shared__ uint32_t s_tmem;
  __shared__ Start s_start;
  __shared__ int s_par[kMaxNodes];
  __shared__ uint32_t s_anc[kMaxNodes][kWords];
  __shared__ float s_m[2][kWideM], s_l[2][kWideM];

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
    mbar_init(&bar_qf, 1);
    mbar_init(&bar_qe, 1);
    mbar_init(&bar_oe, 8);
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&bar_full[s], 1);
      mbar_init(&bar_empty[s], 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&bar_sf[w], 1);
      mbar_init(&bar_pf[w], 4);
      mbar_init(&bar_pv[w], 1);
      for (int i = 0; i < 4; ++i) mbar_init(&bar_m[w][i], 1);
    }
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = s_tmem;
  const int kvh = blockIdx.x % bt.KV;
  const int block_nodes = bt.rows_per_block / bt.group;
  Walker wk;
  wk.start(bt, s_start);
  Item it;

  if (warp == 0 || warp == 2) {
    // ------------------------------ TMA producers --------------------------
    // one lane per warp issues: warp 0 loads Q and K, warp 2 loads V
    const int kv = warp >> 1;
    const CUtensorMap* map = kv ? &tmV : &tmK;
    const bool whole = piece_rows == BN;  // a page holds a tile: one box for it
    const int bytes = piece_rows * 128 * (whole ? D / 64 : 1);
    if (lane == 0) {
      if (kv == 0) tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(map);
      uint32_t seq = kv, qcnt = 0;  // K tiles take the ring's even numbers, V tiles the odd ones
      bool ok = true;
      const int mask = bt.table ? (1 << bt.page_shift) - 1 : INT_MAX;
      while (ok && wk.next(bt, it)) {
        const int rows = it.len + it.n;
        int next_pg = table_entry(bt, it.b, it.t0 * BN);
        if (kv == 0) {
          if (qcnt > 0 && !mbar_wait(&bar_qe, (qcnt - 1) & 1, 0x33000)) break;
          mbar_arrive_expect_tx(&bar_qf, (D / 64) * bt.rows_per_block * 128);
#pragma unroll
          for (int b = 0; b < D / 64; ++b)
            tma_load_3d(smem + b * C::kBoxQ, &tmQ, &bar_qf, b * 64, kvh * bt.group,
                        it.node0 + it.blk * block_nodes);
          ++qcnt;
        }
        for (int t = it.t0; t < it.t1; ++t, seq += 2) {
          const int row0 = t * BN;
          const int pieces = (min(BN, rows - row0) + piece_rows - 1) / piece_rows;  // with rows
          const int slot = seq % kSlots;
          if (seq >= kSlots && !mbar_wait(&bar_empty[slot], ((seq / kSlots) & 1) ^ 1, 0x34000 | slot)) {
            ok = false;
            break;
          }
          uint8_t* dst = smem + C::kRing + slot * C::kTileKV;
          mbar_arrive_expect_tx(&bar_full[slot], pieces * bytes * (whole ? 1 : D / 64));
          if (whole) {
            const int pg = checked_page(bt, it.b, next_pg);
            if (t + 1 < it.t1) next_pg = table_entry(bt, it.b, row0 + BN);
            tma_load_5d(dst, map, &bar_full[slot], 0, row0 & mask, 0, kvh, pg);
          } else {
            for (int i = 0; i < pieces; ++i) {
              const int pg = checked_page(bt, it.b, next_pg);
              const int row = row0 + i * piece_rows, next = row + piece_rows;
              if (next < rows && next < it.t1 * BN) next_pg = table_entry(bt, it.b, next);
#pragma unroll
              for (int b = 0; b < D / 64; ++b)
                tma_load_5d(dst + b * C::kBoxKV + i * piece_rows * 128, map, &bar_full[slot], 0,
                            row & mask, b, kvh, pg);
            }
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
      const uint64_t dQ = sw128_desc(smem_u32(smem), 16, 1024);
      const uint64_t dK0 = sw128_desc(smem_u32(smem + C::kRing), 16, 1024);
      const uint64_t dV0 = sw128_desc(smem_u32(smem + C::kRing), C::kBoxKV, 1024);
      constexpr uint64_t kSlotStep = C::kTileKV >> 4;
      uint32_t seq = 0, qcnt = 0, pvg = 0;
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
          const uint64_t qoff = (((kk >> 2) * C::kBoxQ) + (kk & 3) * 32) >> 4;
          const uint64_t koff = (((kk >> 2) * C::kBoxKV) + (kk & 3) * 32) >> 4;
          tc_mma(d_tm, dQ + qoff, dk + koff, idesc_qk, kk > 0);
        }
        tc_commit(&bar_sf[jj & 1]);
        tc_commit(&bar_empty[slot]);
        return true;
      };
      while (ok && wk.next(bt, it)) {
        const int n = it.t1 - it.t0;
        if (!mbar_wait(&bar_qf, qcnt & 1, 0x36000)) break;
        const uint32_t base = seq;  // K of tile jj at base + 2 jj, V behind it
        seq += 2 * n;
        for (int jj = 0; ok && jj < 2 && jj < n; ++jj) ok = qk(jj, base + 2 * jj);
        if (ok && n <= 2) tc_commit(&bar_qe);
        for (int jj = 0; ok && jj < n; ++jj) {
          const uint32_t vsq = base + 2 * jj + 1, slot = vsq % kSlots;
          uint32_t& pc = pcnt[jj & 1];
          ok = mbar_wait(&bar_pf[jj & 1], pc & 1, 0x37000);
          ++pc;
          if (ok && jj == 0 && qcnt > 0) ok = mbar_wait(&bar_oe, (qcnt - 1) & 1, 0x38000);
          if (ok) ok = mbar_wait(&bar_full[slot], (vsq / kSlots) & 1, 0x39000 | slot);
          if (!ok) break;
          tc_fence_after();
          const uint64_t dv = dV0 + slot * kSlotStep;
          const uint32_t tp = tmem + (jj & 1) * BN;  // P: 16 keys per 8 columns
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk)
            tc_mma_ts(tmem + 2 * BN, tp + kk * 8, dv + ((kk * 16 * 128) >> 4), idesc_pv,
                      jj > 0 || kk > 0);
          tc_commit(&bar_pv[pvg & 1]);
          ++pvg;
          tc_commit(&bar_empty[slot]);
          if (jj + 2 < n) {
            ok = qk(jj + 2, base + 2 * (jj + 2));
            if (ok && jj + 3 == n) tc_commit(&bar_qe);
          }
        }
        ++qcnt;
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ------------------------------ softmax ----------------------------------
    const int w = (warp - 4) >> 2;                 // warpgroup: tiles jj % 2 == w
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;             // row of the block == TMEM lane
    const uint32_t tl = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t s_col = w * BN, o_col = 2 * BN;
    uint32_t cnt[2] = {0, 0};                      // tiles each warpgroup has done
    uint32_t pvbase = 0, seq = 0;
    int anc_of = -1;
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
      if (it.t1 * BN > it.len && anc_of != it.b) {
        asm volatile("bar.sync 1, 256;");
        if (bt.parents)
          for (int i = threadIdx.x - 128; i < it.n; i += 256) s_par[i] = bt.parents[it.node0 + i];
        asm volatile("bar.sync 1, 256;");
        ancestor_masks(s_par, bt.parents == nullptr, it.n, s_anc, threadIdx.x - 128, 256, it.b);
        asm volatile("bar.sync 1, 256;");
        anc_of = it.b;
      }
      const int node = r < live ? (row0 + r) / bt.group : 0;
      float m = -INFINITY, l = 0.f;
      for (int jj = w; jj < n; jj += 2) {
        const int t = it.t0 + jj;
        const uint32_t own = cnt[w] + (jj >> 1);  // how many of this buffer's tiles came before
        const bool last_rows = (t + 1) * BN > rows;
        if (!wait(&bar_sf[w], own & 1, 0x3A000)) continue;
        tc_fence_after();
        if (busy) {
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
                const uint32_t* an = s_anc[node];
                const int lo = j0 >> 5, sh = j0 & 31;    // floor
                const uint32_t a = (lo >= 0 && lo < kWords) ? an[lo] : (lo < 0 ? 0xffffffffu : 0u);
                const uint32_t b = (lo + 1 >= 0 && lo + 1 < kWords) ? an[lo + 1] : 0u;
                vis = sh ? (a >> sh) | (b << (32 - sh)) : a;
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
          // the maximum up to the tile before
          float before = -INFINITY;
          if (jj > 0) {
            const uint32_t theirs = cnt[w ^ 1] + ((jj - 1) >> 1);
            if (wait(&bar_m[w ^ 1][quarter], theirs & 1, 0x3B000)) before = s_m[w ^ 1][r];
          }
          float mnew = before;
          const bool grow = __any_sync(0xffffffffu, mx > before + prefill::kRescaleThreshold);
          if (grow) mnew = fmaxf(before, mx);
          s_m[w][r] = mnew;
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar_m[w][quarter]);
          const float mref = (mnew == -INFINITY) ? 0.f : mnew;
          l *= (m == -INFINITY) ? 0.f : fast_exp2(m - mref);
          m = mnew;
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
            if (wait(&bar_pv[g & 1], (g >> 1) & 1, 0x3C000)) {
              const float alpha = (mnew == -INFINITY) ? 1.f : fast_exp2(before - mnew);
              tc_fence_after();
#pragma unroll
              for (int cc = 0; cc < D / 32; ++cc) {
                float o[32];
                tc_ld32(tl + o_col + cc * 32, o);
                tc_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] *= alpha;
                tc_st32(tl + o_col + cc * 32, o);
              }
              tc_wait_st();
            }
          }
          tc_fence_before();
        } else if (lane == 0) {
          mbar_arrive(&bar_m[w][quarter]);  // keeps the barrier's count of tiles
        }
        if (last_rows) {
          // V rows past the request's last hold anything: their weight is 0,
          // but 0 * NaN is not, so they are cleared before the product
          const uint32_t vsq = seq + 2 * jj + 1, slot = vsq % kSlots;
          if (wait(&bar_full[slot], (vsq / kSlots) & 1, 0x3D000)) {
            const int bad = max(rows - t * BN, 0);
            uint8_t* vt = smem + C::kRing + slot * C::kTileKV;
            for (int i = r; i < (BN - bad) * (D / 8); i += 128) {
              const int row = bad + i / (D / 8), c16 = i % (D / 8);
              *reinterpret_cast<uint4*>(vt + (c16 >> 3) * C::kBoxKV + sw128_off(row, c16 & 7)) =
                  make_uint4(0u, 0u, 0u, 0u);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_pf[w]);
      }
      // ---------------- the item's end: both warpgroups' sums meet ----------
      s_l[w][r] = l;
      s_m[w][r] = m;
      asm volatile("bar.sync 1, 256;");
      const float ma = s_m[0][r], mb = s_m[1][r];
      const float M = fmaxf(ma, mb);
      const float mref = (M == -INFINITY) ? 0.f : M;
      const float L = s_l[0][r] * fast_exp2(ma - mref) + s_l[1][r] * fast_exp2(mb - mref);
      const uint32_t g = pvbase + n - 1;
      wait(&bar_pv[g & 1], (g >> 1) & 1, 0x3E000);
      tc_fence_after();
      const int slot = part_slot(it, blockIdx.x);
      const bool good = r < live;
      const int head = kvh * bt.group + (good ? row0 + r - node * bt.group : 0);
      const size_t row = static_cast<size_t>(it.node0 + node) * bt.H + head;
      const float f = slot >= 0 ? 1.f : (L > 0.f ? 1.f / L : 0.f);
      float* po = part_o + (static_cast<size_t>(max(slot, 0)) * bt.rows_per_block + r) * D;
      if (busy && !dead) {
        // each warpgroup writes half of the columns
#pragma unroll
        for (int cc = 0; cc < D / 64; ++cc) {
          const int col = w * (D / 2) + cc * 32;
          float o[32];
          tc_ld32(tl + o_col + col, o);
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
      cnt[0] += (n + 1) >> 1;
      cnt[1] += n >> 1;
      pvbase += n;
      seq += 2 * n;
      tc_fence_before();
      asm volatile("bar.sync 1, 256;");  // s_m, s_l and O are read
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
