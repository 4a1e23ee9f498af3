// Attention of drafted tokens over a KV cache, split over the cached rows.
//
// Each request has a tree of n nodes (drafted tokens; one node is an ordinary
// decode token).  Its cache holds len rows of accepted tokens and, behind
// them, the nodes' own rows len .. len + n - 1.  Node i sees rows 0..len-1,
// its ancestors and itself:
//   out_i = sum_{s in S(i)} p_is V_s,  p_is = exp(scale q_i.K_s) / sum exp.
// The cache is a pool of pages reached through a block table, or one block
// per sequence (the layout b2a_decode reads).
//
// Three kernels share the work division of tree_work.cuh:
//   tree_mma_kernel   16-bit caches, few query rows (nodes x heads of a KV
//                     head): bound by reading K and V
//   tree_wide_kernel  16-bit caches, many rows: tcgen05 (tree_wide.cu)
//   tree_f32_kernel   f32 caches, f32 FMAs
// and tree_merge_kernel joins the parts of items cut between CTAs.

#include <limits.h>
#include <math.h>

#include <atomic>

#include "b2a_common.cuh"
#include "tree_work.cuh"

namespace b2a {
namespace tree {

// ---------------------------------------------------------------------------
// 16-bit caches, few rows: warp-level MMAs
// ---------------------------------------------------------------------------
// One persistent CTA per SM.  Producer warps stream 64-row K and V tiles into a
// ring with TMA: one box per page piece, all columns of its rows (a tile of
// 16-row pages takes 4 pieces x 2).
// Eight consumer warps run the decode kernel's fragments (decode.cu):
// S^T = K.Q^T with the query rows on the MMA's N axis, online softmax on the
// accumulators, O^T += V^T.P^T.  Warps 0-3 take the even
// tiles, 4-7 the odd ones; a warp takes 16 keys of a tile and all the query rows
// (up to 8 NT).
// P is rounded to the cache's type for the second product (its error, one
// part in 2^8 or 2^11 of each weight, is what the output's own rounding
// makes); scores, maxima, sums and accumulators are f32.  Q is not
// pre-scaled: the scale goes onto the f32 scores.  Measured, 16 x 32768 rows,
// 32/8 heads, 4 rows: bf16 x 128, pages of 64: 327 to 341 us (6.3 to 6.6 TB/s),
// one block per sequence 337; the decode kernel (decode.cu) takes 305 for the same
// rows on the same GPU (7.0 TB/s), and why this one is a tenth behind has not been
// found.  f16 x 64, pages of 64: 199 us (5.4 TB/s), pages of 16 220; the decode
// kernel 168 to 221 with its split of 2048 to 8192 rows.  There the warps' chain of a
// tile, not HBM, sets the time.
constexpr int kRows = 64;
constexpr int kConsumers = 8;
constexpr int kProducers = 4;
constexpr int kMmaThreads = (kConsumers + kProducers) * 32;

template <int D, int NT>
struct MmaCfg {
  static constexpr int kBoxes = D / 64;
  static constexpr int kTileBytes = kBoxes * kRows * 128;
  static constexpr int kStageBytes = 2 * kTileBytes;
  // four warps' states (o, m, l) while the warps of a CTA are joined
  static constexpr int kState = (D / 16 * NT * 4 + NT * 4) * 32 * 4;
  static constexpr int kMerge = 4 * kState;
  static constexpr int kFit = (232448 - 1024 - 4096 - kMerge) / kStageBytes;
  // A stage must always belong to the same half of the warps: a warp that
  // skipped a stage's last use could not tell its phase by the parity.  An even
  // ring keeps tile parity and stage parity together.
  static constexpr int kStages = kFit > 10 ? 10 : kFit & ~1;
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kMerge;
  static_assert(kStages >= 2, "ring");
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kMmaThreads, 1) tree_mma_kernel(
    const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
    const __grid_constant__ Batch bt, const T* __restrict__ q, long long q_stride,
    const T* __restrict__ vc, long long page_stride, T* __restrict__ out, float* __restrict__ lse,
    float* __restrict__ part_o, float* __restrict__ part_ml, int piece_rows, float sscale) {
  using C = MmaCfg<D, NT>;
  constexpr int KS = D / 16;
  constexpr int RB = 8 * NT;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[C::kStages];
  __shared__ __align__(8) uint64_t empty_bar[C::kStages];
  __shared__ Start s_start;
  __shared__ int s_special;  // the item's tree rows held infinities or NaN
  __shared__ int s_par[kMaxNodes];
  __shared__ uint32_t s_anc[kMaxNodes][kWords];

  pdl_wait();
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    const Start s = locate(bt, team_of(bt, blockIdx.x));
    if (lane == 0) s_start = s;
  } else if (warp == kConsumers && lane == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full_bar[s], min(kProducers, 2 * (kRows / piece_rows)));
      mbar_init(&empty_bar[s], kConsumers / 2);
    }
    fence_mbar_init();
    s_special = 0;
  }
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Walker wk;
  wk.start(bt, s_start);
  Item it;

  if (warp >= kConsumers) {
    // ---------------- producer warps --------------------------------------
    // A TMA issue takes a thread about a hundred cycles (its operands move to
    // uniform registers), so the boxes of a tile, K and V of each page piece,
    // are dealt to the producer warps; each warp's first lane issues its own.
    const int p = warp - kConsumers;
    const int boxes = 2 * (kRows / piece_rows);
    const int bytes = piece_rows * D * 2;
    if (p < boxes && lane == 0) {
      const CUtensorMap* map = (p & 1) ? &tmV : &tmK;
      tma_prefetch_desc(map);
      uint8_t* dst = smem + (p & 1) * C::kTileBytes;
      uint32_t s = 0, round = 0;
      bool ok = true;
      while (ok && wk.next(bt, it)) {
        const int rows = it.len + it.n;
        // the pages of the next tile are looked up while this one waits for room
        const int at0 = (p >> 1) * piece_rows, at1 = at0 + (kProducers / 2) * piece_rows;
        auto entry = [&](int t, int at) {
          const int row = t * kRows + at;
          return t < it.t1 && at < kRows && row < rows ? table_entry(bt, it.b, row) : 0;
        };
        int pg0 = entry(it.t0, at0), pg1 = entry(it.t0, at1);
        for (int t = it.t0; t < it.t1; ++t) {
          const int row0 = t * kRows + at0, row1 = t * kRows + at1;
          const bool live0 = row0 < rows, live1 = at1 < kRows && row1 < rows;
          const int now0 = live0 ? checked_page(bt, it.b, pg0) : 0;
          const int now1 = live1 ? checked_page(bt, it.b, pg1) : 0;
          pg0 = entry(t + 1, at0);
          pg1 = entry(t + 1, at1);
          if (round > 0 && !mbar_wait(&empty_bar[s], (round & 1) ^ 1, 0x31000 | s)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full_bar[s], (live0 ? bytes : 0) + (live1 ? bytes : 0));
          const int mask = bt.table ? (1 << bt.page_shift) - 1 : INT_MAX;
          uint8_t* at = dst + s * C::kStageBytes + (p >> 1) * bytes;
          if (live0) tma_load_5d(at, map, &full_bar[s], 0, row0 & mask, 0, it.kvh, now0);
          if (live1)
            tma_load_5d(at + (kProducers / 2) * bytes, map, &full_bar[s], 0, row1 & mask, 0, it.kvh, now1);
          if (++s == C::kStages) {
            s = 0;
            ++round;
          }
        }
      }
    }
    return;
  }

  // ---------------- consumer warps ----------------------------------------
  zero_unwritten<T, D>(bt, s_start.left_out, out, lse, warp, kConsumers);
  const int g = lane >> 2, t4 = lane & 3;
  const int slice = warp & 3, half = warp >> 2;
  const uint32_t ring = smem_u32(smem);
  float* merge = reinterpret_cast<float*>(smem + C::kStages * C::kStageBytes);
  // A tile is [piece][64-column box][row of the piece][128 bytes]; a warp's 16
  // rows lie in one piece.
  const int box_bytes = piece_rows * 128;
  const int slice_at = (slice * 16 / piece_rows) * piece_rows * D * 2 +
                       (slice * 16 % piece_rows) * 128;
  const int a_row = (lane & 7) + ((lane >> 3) & 1) * 8;  // K (non-trans)
  const int a_khalf = lane >> 4;
  const int v_row = (lane & 7) + ((lane >> 4) << 3);     // V (trans)
  const int v_dhalf = (lane >> 3) & 1;
  uint32_t seq = 0;
  int anc_of = -1;   // the request whose masks are in shared memory
  bool dead = false;  // a wait ran out: no more waiting, the barriers go on

  while (wk.next(bt, it)) {
    const int R = it.n * bt.group;
    const int row_lo = it.blk * RB;
    if (it.t1 * kRows > it.len && anc_of != it.b) {
      asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32));
      if (bt.parents)
        for (int i = threadIdx.x; i < it.n; i += kConsumers * 32)
          s_par[i] = bt.parents[it.node0 + i];
      asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32));
      ancestor_masks(s_par, bt.parents == nullptr, it.n, s_anc, threadIdx.x, kConsumers * 32, it.b);
      asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32));
      anc_of = it.b;
    }
    uint32_t qf[NT][KS][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = row_lo + nt * 8 + g;
      const bool valid = r < R;
      const int node = valid ? r / bt.group : 0;
      const int head = it.kvh * bt.group + (valid ? r - node * bt.group : 0);
      const T* qr = q + (it.node0 + node) * q_stride + head * D;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        qf[nt][ks][0] = valid ? *reinterpret_cast<const uint32_t*>(qr + ks * 16 + 2 * t4) : 0u;
        qf[nt][ks][1] = valid ? *reinterpret_cast<const uint32_t*>(qr + ks * 16 + 2 * t4 + 8) : 0u;
      }
    }
    float o[KS][NT][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int mt = 0; mt < KS; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[mt][nt][i] = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }
    const int rows = it.len + it.n;

    for (int t = it.t0; t < it.t1; ++t, ++seq) {
      if ((seq & 1u) != static_cast<uint32_t>(half)) continue;
      const int s = seq % C::kStages;
      if (!dead)
        dead = !__all_sync(0xffffffffu,
                           mbar_wait(&full_bar[s], (seq / C::kStages) & 1, 0x32000 | s));
      if (dead) continue;
      const uint32_t kt = ring + s * C::kStageBytes + slice_at;
      const uint32_t vt = kt + C::kTileBytes;

      const int slice0 = t * kRows + slice * 16;
      const bool tail = slice0 + 16 > it.len;  // tree rows, or rows past the last
      if (tail) {
        // Rows past the request's last hold anything (a pool's old rows, or
        // what the stage held before): their weight is 0, but 0 * NaN is not,
        // so their V rows are cleared, and infinities and NaN of tree rows too.
        const int first = max(it.len - slice0, 0), past = min(max(rows - slice0, 0), 16);
        uint8_t* vslice = smem + s * C::kStageBytes + C::kTileBytes + slice_at;
        auto chunk = [&](int from, int i) {  // 16 bytes i of the rows from `from` on
          const int row = from + i / (C::kBoxes * 8), rem = i % (C::kBoxes * 8);
          return reinterpret_cast<uint4*>(vslice + (rem >> 3) * box_bytes + sw128_off(row, rem & 7));
        };
        for (int i = lane; i < (16 - past) * C::kBoxes * 8; i += 32)
          *chunk(past, i) = make_uint4(0u, 0u, 0u, 0u);
        if (it.n > 1)
          for (int i = lane; i < (past - first) * C::kBoxes * 8; i += 32) {
            uint4 u = *chunk(first, i);
            if (clear_special<T>(u)) {
              *chunk(first, i) = u;
              s_special = 1;
            }
          }
        __syncwarp();
      }

      float sc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t a[4];
        ldsm_x4(kt + (ks >> 2) * box_bytes + sw128_off(a_row, ((ks & 3) << 1) + a_khalf), a[0],
                a[1], a[2], a[3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) MmaOp<T>::run(sc[nt], a, qf[nt][ks]);
      }
      if (tail) {
        // tree rows: visible to a query row whose node has them as ancestor
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = slice0 + g + e * 8 - it.len;  // tree node of this key
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int r = row_lo + nt * 8 + 2 * t4 + c;
              bool see = j < 0;
              if (j >= 0 && j < it.n && r < R)
                see = (s_anc[r / bt.group][j >> 5] >> (j & 31)) & 1u;
              if (!see) sc[nt][e * 2 + c] = -INFINITY;
            }
        }
      }

      uint32_t pb[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float p[4], alpha[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float mx = fmaxf(sc[nt][j], sc[nt][j + 2]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float mnew = fmaxf(m[nt][j], mx * sscale);
          const float mref = (mnew == -INFINITY) ? 0.f : mnew;
          alpha[j] = fast_exp2(m[nt][j] - mref);
          m[nt][j] = mnew;
          p[j] = fast_exp2(fmaf(sc[nt][j], sscale, -mref));
          p[j + 2] = fast_exp2(fmaf(sc[nt][j + 2], sscale, -mref));
          l[nt][j] = l[nt][j] * alpha[j] + (p[j] + p[j + 2]);
        }
#pragma unroll
        for (int mt = 0; mt < KS; ++mt) {
          o[mt][nt][0] *= alpha[0];
          o[mt][nt][1] *= alpha[1];
          o[mt][nt][2] *= alpha[0];
          o[mt][nt][3] *= alpha[1];
        }
        pb[nt][0] = movmatrix_trans(MmaOp<T>::pack(p[0], p[1]));
        pb[nt][1] = movmatrix_trans(MmaOp<T>::pack(p[2], p[3]));
      }
#pragma unroll
      for (int mt = 0; mt < KS; ++mt) {
        uint32_t a[4];
        const int dchunk = 2 * mt + v_dhalf;
        ldsm_x4_trans(vt + (dchunk >> 3) * box_bytes + sw128_off(v_row, dchunk & 7), a[0], a[1],
                      a[2], a[3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) MmaOp<T>::run(o[mt][nt], a, pb[nt]);
      }
      // the generic-proxy zeros come before the next TMA write of the stage
      if (tail) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty_bar[s]);
    }

    // ---------------- join the warps ---------------------------------------
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float x = l[nt][j];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        l[nt][j] = x;
      }
    // in each round the upper half of the remaining warps hands its state to
    // the lower half
#pragma unroll
    for (int left = 4; left > 0; left >>= 1) {
      const int rank = warp;
      float* st = merge + (rank & (left - 1)) * (C::kState / 4) + lane;
      if (rank >= left && rank < 2 * left) {
#pragma unroll
        for (int mt = 0; mt < KS; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) st[((mt * NT + nt) * 4 + i) * 32] = o[mt][nt][i];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            st[(KS * NT * 4 + nt * 4 + j * 2) * 32] = m[nt][j];
            st[(KS * NT * 4 + nt * 4 + j * 2 + 1) * 32] = l[nt][j];
          }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32));
      if (rank < left) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float a[2], c[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float m2 = st[(KS * NT * 4 + nt * 4 + j * 2) * 32];
            const float l2 = st[(KS * NT * 4 + nt * 4 + j * 2 + 1) * 32];
            const float mnew = fmaxf(m[nt][j], m2);
            const float mref = (mnew == -INFINITY) ? 0.f : mnew;
            a[j] = fast_exp2(m[nt][j] - mref);
            c[j] = fast_exp2(m2 - mref);
            m[nt][j] = mnew;
            l[nt][j] = l[nt][j] * a[j] + l2 * c[j];
          }
#pragma unroll
          for (int mt = 0; mt < KS; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              o[mt][nt][i] = o[mt][nt][i] * a[i & 1] + st[((mt * NT + nt) * 4 + i) * 32] * c[i & 1];
        }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32));
    }
    // the rows go through shared memory so that the stores are whole lines
    constexpr int kPad = D + 4;
    float* fin = merge;                // [RB][kPad]
    float* fml = merge + RB * kPad;    // [RB][2]
    static_assert((RB * (D + 4) + 2 * RB) * 4 <= C::kMerge, "final rows fit the merge buffer");
    const int slot = part_slot(it, blockIdx.x);
    if (warp == 0) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int r = nt * 8 + 2 * t4 + c;
          const float f = slot >= 0 ? 1.f : (l[nt][c] > 0.f ? 1.f / l[nt][c] : 0.f);
#pragma unroll
          for (int mt = 0; mt < KS; ++mt) {
            fin[r * kPad + mt * 16 + g] = o[mt][nt][c] * f;
            fin[r * kPad + mt * 16 + g + 8] = o[mt][nt][2 + c] * f;
          }
          if (g == 0) {
            fml[r * 2] = m[nt][c];
            fml[r * 2 + 1] = l[nt][c];
          }
        }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32));
    const bool special = s_special != 0;
    if (special) {
      asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32));
      if (threadIdx.x == 0) s_special = 0;
    }
    const int live = min(RB, R - it.blk * RB);
    // adds what was taken out of the V rows to n elements of row r from column d on
    auto put_back = [&](int r, int d, int n, auto* dst) {
      const uint32_t* a = s_anc[(it.blk * RB + r) / bt.group];
      add_special(bt, vc, page_stride, it.b, it.kvh, it.len, max(it.t0 * kRows - it.len, 0),
                  min(it.t1 * kRows - it.len, it.n), make_uint4(a[0], a[1], a[2], a[3]), dst, D, d, n);
    };
    if (slot >= 0) {
      float* po = part_o + static_cast<size_t>(slot) * RB * D;
      for (int i = threadIdx.x; i < live * (D / 4); i += kConsumers * 32) {
        const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
        *reinterpret_cast<float4*>(po + r * D + d) =
            *reinterpret_cast<const float4*>(fin + r * kPad + d);
        if (special) put_back(r, d, 4, po + r * D + d);
      }
      if (threadIdx.x < 2 * live) part_ml[static_cast<size_t>(slot) * RB * 2 + threadIdx.x] = fml[threadIdx.x];
    } else {
      for (int i = threadIdx.x; i < live * (D / 8); i += kConsumers * 32) {
        const int r = i / (D / 8), d = (i - r * (D / 8)) * 8;
        const int rr = it.blk * RB + r, node = rr / bt.group;
        const size_t row = static_cast<size_t>(it.node0 + node) * bt.H + it.kvh * bt.group + (rr - node * bt.group);
        const float* x = fin + r * kPad + d;
        uint4 u;
        u.x = MmaOp<T>::pack(x[0], x[1]);
        u.y = MmaOp<T>::pack(x[2], x[3]);
        u.z = MmaOp<T>::pack(x[4], x[5]);
        u.w = MmaOp<T>::pack(x[6], x[7]);
        *reinterpret_cast<uint4*>(out + row * D + d) = u;
        if (special) put_back(r, d, 8, out + row * D + d);
        if (lse && d == 0)
          lse[row] = fml[r * 2 + 1] > 0.f ? (fml[r * 2] + log2f(fml[r * 2 + 1])) * kLn2 : -INFINITY;
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32));
  }
}

// ---------------------------------------------------------------------------
// f32 caches: f32 products and sums on the CUDA cores
// ---------------------------------------------------------------------------
// 256 threads, items of 16 query rows, bound by the FMA pipe.  One K and one V
// buffer, filled by cp.async: K(t + 1) loads while softmax and P.V of tile t
// run, V(t + 1) while the scores of t + 1 do.  A thread forms the scores of 2
// rows x kTile/32 keys (32 FMAs per 6 shared 16-byte reads, which the pipes do
// in about the same time), a warp the softmax of 2 rows, a thread the output
// column(s) of its rows.  3 requests of 77 to 2049 rows, 1 to 12 nodes, 32/8
// heads x 128: 63 to 64 us (floor 7.3: the FMAs; with half the threads 88).
constexpr int kF32Threads = 256;
constexpr int kF32Rows = 16;

template <int D>
struct F32Cfg {
  static constexpr int kTile = D > 128 ? 64 : 128;
  static constexpr int kKStride = D + 4;
  static constexpr int kK = kTile * kKStride;
  static constexpr int kV = kTile * D;
  static constexpr int kQ = kF32Rows * kKStride;
  static constexpr int kP = kF32Rows * (kTile + 4);
  static constexpr int kSmem = (kK + kV + kQ + kP) * 4;
};

template <int D>
__global__ void __launch_bounds__(kF32Threads) tree_f32_kernel(
    const float* __restrict__ kc, const float* __restrict__ vc, long long page_stride,
    const __grid_constant__ Batch bt, const float* __restrict__ q, long long q_stride,
    float* __restrict__ out, float* __restrict__ lse, float* __restrict__ part_o,
    float* __restrict__ part_ml, float sscale) {
  using C = F32Cfg<D>;
  constexpr int TILE = C::kTile;
  constexpr int PS = TILE + 4;
  constexpr int kWarps = kF32Threads / 32;
  extern __shared__ __align__(16) float fsm[];
  __shared__ Start s_start;
  __shared__ int s_par[kMaxNodes];
  __shared__ uint32_t s_anc[kMaxNodes][kWords];
  __shared__ float s_m[kF32Rows], s_l[kF32Rows], s_alpha[kF32Rows];
  __shared__ int s_special;  // the item's tree rows held infinities or NaN
  pdl_wait();
  float* ks = fsm;
  float* vs = ks + C::kK;
  float* qs = vs + C::kV;
  float* ps = qs + C::kQ;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (warp == 0) {
    const Start s = locate(bt, team_of(bt, blockIdx.x));
    if (lane == 0) s_start = s;
  }
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  zero_unwritten<float, D>(bt, s_start.left_out, out, lse, warp, kWarps);
  Walker wk;
  wk.start(bt, s_start);
  Item it;
  constexpr int kCols = D > kF32Threads ? D / kF32Threads : 1;  // output columns of a thread
  constexpr int kShare = kF32Threads / (D / kCols);             // threads that share a column
  constexpr int kORows = kF32Rows / kShare;                     // rows of a thread
  const int oc = tid % (D / kCols);
  const int or0 = (tid / (D / kCols)) * kORows;

  while (wk.next(bt, it)) {
    const int R = it.n * bt.group;
    const int rows = it.len + it.n;
    // a K or V tile, rows past the end as zeros
    auto load = [&](const float* src, float* dst, int stride, int t) {
      for (int i = tid; i < TILE * (D / 4); i += kF32Threads) {
        const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
        const int row = t * TILE + r;
        size_t at = 0;
        int bytes = 0;
        if (row < rows) {
          const int pg = checked_page(bt, it.b, table_entry(bt, it.b, row));
          if (pg < bt.n_pages) {
            const int in_page = bt.table ? row & ((1 << bt.page_shift) - 1) : row;
            at = static_cast<size_t>(pg) * page_stride +
                 (static_cast<size_t>(in_page) * bt.KV + it.kvh) * D + d;
            bytes = 16;
          }
        }
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst + r * stride + d)),
                     "l"(src + at), "r"(bytes) : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    __syncthreads();  // the item before is done with every buffer
    load(kc, ks, C::kKStride, it.t0);
    load(vc, vs, D, it.t0);
    if (bt.parents)
      for (int i = tid; i < it.n; i += kF32Threads) s_par[i] = bt.parents[it.node0 + i];
    for (int i = tid; i < kF32Rows * (D / 4); i += kF32Threads) {
      const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
      const int rr = it.blk * kF32Rows + r;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (rr < R) {
        const int node = rr / bt.group, head = it.kvh * bt.group + rr - node * bt.group;
        x = *reinterpret_cast<const float4*>(q + (it.node0 + node) * q_stride + head * D + d);
      }
      *reinterpret_cast<float4*>(qs + r * C::kKStride + d) = x;
    }
    if (tid < kF32Rows) {
      s_m[tid] = -INFINITY;
      s_l[tid] = 0.f;
    }
    if (tid == 0) s_special = 0;
    __syncthreads();
    ancestor_masks(s_par, bt.parents == nullptr, it.n, s_anc, tid, kF32Threads, it.b);

    float o[kORows][kCols];
#pragma unroll
    for (int r = 0; r < kORows; ++r)
#pragma unroll
      for (int c = 0; c < kCols; ++c) o[r][c] = 0.f;
    for (int t = it.t0; t < it.t1; ++t) {
      asm volatile("cp.async.wait_group 1;" ::: "memory");  // K(t); V(t) may be on its way
      __syncthreads();
      {
        constexpr int KN = TILE / 32;
        const int r0 = (tid & 7) * 2, k0 = tid >> 3;
        float acc[2][KN];
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int b = 0; b < KN; ++b) acc[a][b] = 0.f;
#pragma unroll 8
        for (int d = 0; d < D; d += 4) {
          float4 qa[2];
#pragma unroll
          for (int a = 0; a < 2; ++a)
            qa[a] = *reinterpret_cast<const float4*>(qs + (r0 + a) * C::kKStride + d);
#pragma unroll
          for (int b = 0; b < KN; ++b) {
            const float4 kk = *reinterpret_cast<const float4*>(ks + (k0 + 32 * b) * C::kKStride + d);
#pragma unroll
            for (int a = 0; a < 2; ++a) {
              acc[a][b] = fmaf(qa[a].x, kk.x, acc[a][b]);
              acc[a][b] = fmaf(qa[a].y, kk.y, acc[a][b]);
              acc[a][b] = fmaf(qa[a].z, kk.z, acc[a][b]);
              acc[a][b] = fmaf(qa[a].w, kk.w, acc[a][b]);
            }
          }
        }
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int b = 0; b < KN; ++b) {
            const int row = t * TILE + k0 + 32 * b;
            const int r = it.blk * kF32Rows + r0 + a, j = row - it.len;
            bool see = j < 0;
            if (j >= 0 && j < it.n && r < R) see = (s_anc[r / bt.group][j >> 5] >> (j & 31)) & 1u;
            ps[(r0 + a) * PS + k0 + 32 * b] = see ? acc[a][b] * sscale : -INFINITY;
          }
      }
      __syncthreads();
      // K's buffer is free (an empty group keeps the count of groups)
      if (t + 1 < it.t1) load(kc, ks, C::kKStride, t + 1);
      else asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll
      for (int i = 0; i < kF32Rows / kWarps; ++i) {
        const int r = warp * (kF32Rows / kWarps) + i;
        float x[TILE / 32], mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < TILE / 32; ++e) {
          x[e] = ps[r * PS + lane + 32 * e];
          mx = fmaxf(mx, x[e]);
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        const float mo = s_m[r], mnew = fmaxf(mo, mx);
        const float mref = (mnew == -INFINITY) ? 0.f : mnew;
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < TILE / 32; ++e) {
          x[e] = exp2f(x[e] - mref);
          ps[r * PS + lane + 32 * e] = x[e];
          sum += x[e];
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        __syncwarp();
        if (lane == 0) {
          const float al = exp2f(mo - mref);
          s_alpha[r] = al;
          s_l[r] = s_l[r] * al + sum;
          s_m[r] = mnew;
        }
      }
      asm volatile("cp.async.wait_group 1;" ::: "memory");  // V(t)
      __syncthreads();
      if (it.n > 1 && (t + 1) * TILE > it.len) {
        const int first = max(it.len - t * TILE, 0), past = min(rows - t * TILE, TILE);
        for (int i = tid; i < (past - first) * (D / 4); i += kF32Threads) {
          uint4* at = reinterpret_cast<uint4*>(vs + first * D) + i;
          uint4 u = *at;
          if (clear_special<float>(u)) {
            *at = u;
            s_special = 1;
          }
        }
        __syncthreads();
      }
#pragma unroll
      for (int r = 0; r < kORows; ++r) {
        const float al = s_alpha[or0 + r];
#pragma unroll
        for (int c = 0; c < kCols; ++c) o[r][c] *= al;
      }
#pragma unroll 4
      for (int k = 0; k < TILE; k += 4) {
        float v[4][kCols];
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int c = 0; c < kCols; ++c) v[e][c] = vs[(k + e) * D + oc + c * kF32Threads];
#pragma unroll
        for (int r = 0; r < kORows; ++r) {
          const float4 p = *reinterpret_cast<const float4*>(ps + (or0 + r) * PS + k);
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            o[r][c] = fmaf(p.x, v[0][c], o[r][c]);
            o[r][c] = fmaf(p.y, v[1][c], o[r][c]);
            o[r][c] = fmaf(p.z, v[2][c], o[r][c]);
            o[r][c] = fmaf(p.w, v[3][c], o[r][c]);
          }
        }
      }
      __syncthreads();
      if (t + 1 < it.t1) load(vc, vs, D, t + 1);
      else asm volatile("cp.async.commit_group;" ::: "memory");
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    const int live = min(kF32Rows, R - it.blk * kF32Rows);
    const int slot = part_slot(it, blockIdx.x);
    const bool special = s_special != 0;
    // adds what was taken out of the V rows to column d of row rr
    auto put_back = [&](int rr, int d, float* dst) {
      const uint32_t* a = s_anc[(it.blk * kF32Rows + rr) / bt.group];
      add_special(bt, vc, page_stride, it.b, it.kvh, it.len, max(it.t0 * TILE - it.len, 0),
                  min(it.t1 * TILE - it.len, it.n), make_uint4(a[0], a[1], a[2], a[3]), dst, D, d, 1);
    };
#pragma unroll
    for (int r = 0; r < kORows; ++r) {
      const int rr = or0 + r;
      if (rr >= live) continue;
      const float l = s_l[rr];
      if (slot >= 0) {
        float* po = part_o + (static_cast<size_t>(slot) * kF32Rows + rr) * D;
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          po[oc + c * kF32Threads] = o[r][c];
          if (special) put_back(rr, oc + c * kF32Threads, po + oc + c * kF32Threads);
        }
        if (oc == 0) {
          part_ml[(static_cast<size_t>(slot) * kF32Rows + rr) * 2] = s_m[rr];
          part_ml[(static_cast<size_t>(slot) * kF32Rows + rr) * 2 + 1] = l;
        }
      } else {
        const int gr = it.blk * kF32Rows + rr, node = gr / bt.group;
        const size_t row = static_cast<size_t>(it.node0 + node) * bt.H + it.kvh * bt.group + (gr - node * bt.group);
        const float f = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          out[row * D + oc + c * kF32Threads] = o[r][c] * f;
          if (special) put_back(rr, oc + c * kF32Threads, out + row * D + oc + c * kF32Threads);
        }
        if (lse && oc == 0) lse[row] = l > 0.f ? (s_m[rr] + log2f(l)) * kLn2 : -INFINITY;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Joins the parts of cut items
// ---------------------------------------------------------------------------
// Block (c, y) looks at the last item of CTA c's range: if the item goes on
// past the range and does not begin before it, its parts are CTA c's slot
// 2c + 1, the same slot of its fellows in the later teams that the item fills,
// and slot 2e of the one, e, where it ends.  One warp per query row.
constexpr int kMergeWarps = 8;

template <typename T, int D>
__global__ void __launch_bounds__(kMergeWarps * 32) tree_merge_kernel(
    const __grid_constant__ Batch bt, const float* __restrict__ part_o,
    const float* __restrict__ part_ml, T* __restrict__ out, float* __restrict__ lse) {
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x;
  const Start s = locate(bt, team_of(bt, c));
  if (s.left < s.chunk) return;  // an empty range, or the list's last
  // the item that holds the range's last tile
  int b = s.b, n, len;
  long long off = s.off + s.left - 1;  // the range's last tile, counted in request b
  request(bt, b, n, len, s.left_out);
  long long u = units_of(bt, n, len);
  while (off >= u) {
    off -= u;
    if (++b >= bt.B) return;
    request(bt, b, n, len, s.left_out);
    u = units_of(bt, n, len);
  }
  const int tiles = (len + n + bt.tile - 1) / bt.tile;
  const int idx = static_cast<int>(off / tiles);
  const int at = static_cast<int>(off - static_cast<long long>(idx) * tiles);
  const int after = tiles - 1 - at;  // tiles past the range
  int kvh, blk;
  if (after == 0 || at >= s.chunk || !member_item(bt, c, idx, blocks_of(bt, n), kvh, blk)) return;
  const int whole = static_cast<int>(after / s.chunk);  // later ranges the item fills
  const int rest = static_cast<int>(after - whole * s.chunk);
  const int parts = 1 + whole + (rest > 0 ? 1 : 0);
  const int RB = bt.rows_per_block;
  const int live = min(RB, n * bt.group - blk * RB);
  const int node0 = bt.cu[b];
  // A part that ends exactly with its CTA's range is that CTA's slot 2e.
  auto slot = [&](int i) {
    return 2 * (c + i * bt.m_heads * bt.m_blks) + ((i == parts - 1) ? 0 : 1);
  };
  for (int r = blockIdx.y * kMergeWarps + warp; r < live; r += gridDim.y * kMergeWarps) {
    float M = -INFINITY;
    for (int i = lane; i < parts; i += 32)
      M = fmaxf(M, part_ml[(static_cast<size_t>(slot(i)) * RB + r) * 2]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float mref = (M == -INFINITY) ? 0.f : M;
    float L = 0.f;
    float acc[D / 32];
#pragma unroll
    for (int e = 0; e < D / 32; ++e) acc[e] = 0.f;
    for (int i0 = 0; i0 < parts; i0 += 32) {
      const int k = min(32, parts - i0);
      float w = 0.f, lw = 0.f;
      if (lane < k) {
        const float2 ml = *reinterpret_cast<const float2*>(part_ml + (static_cast<size_t>(slot(i0 + lane)) * RB + r) * 2);
        w = exp2f(ml.x - mref);
        lw = ml.y * w;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) lw += __shfl_xor_sync(0xffffffffu, lw, o);
      L += lw;
#pragma unroll 4
      for (int i = 0; i < k; ++i) {
        const float wi = __shfl_sync(0xffffffffu, w, i);
        const float* po = part_o + (static_cast<size_t>(slot(i0 + i)) * RB + r) * D;
        if constexpr (D == 64) {
          const float2 x = *reinterpret_cast<const float2*>(po + lane * 2);
          acc[0] = fmaf(x.x, wi, acc[0]);
          acc[1] = fmaf(x.y, wi, acc[1]);
        } else {
#pragma unroll
          for (int e = 0; e < D / 128; ++e) {
            const float4 x = *reinterpret_cast<const float4*>(po + e * 128 + lane * 4);
            acc[e * 4] = fmaf(x.x, wi, acc[e * 4]);
            acc[e * 4 + 1] = fmaf(x.y, wi, acc[e * 4 + 1]);
            acc[e * 4 + 2] = fmaf(x.z, wi, acc[e * 4 + 2]);
            acc[e * 4 + 3] = fmaf(x.w, wi, acc[e * 4 + 3]);
          }
        }
      }
    }
    const float f = L > 0.f ? 1.f / L : 0.f;
    const int rr = blk * RB + r, node = rr / bt.group;
    const size_t row = static_cast<size_t>(node0 + node) * bt.H + kvh * bt.group + (rr - node * bt.group);
    T* dst = out + row * D;
    if constexpr (D == 64) {
      st_elem(dst + lane * 2, acc[0] * f);
      st_elem(dst + lane * 2 + 1, acc[1] * f);
    } else {
#pragma unroll
      for (int e = 0; e < D / 128; ++e)
#pragma unroll
        for (int k = 0; k < 4; ++k) st_elem(dst + e * 128 + lane * 4 + k, acc[e * 4 + k] * f);
    }
    if (lse && lane == 0) lse[row] = L > 0.f ? (M + log2f(L)) * kLn2 : -INFINITY;
  }
}

}  // namespace tree
}  // namespace b2a

// ===========================================================================
// Host side
// ===========================================================================
namespace {

namespace TR = b2a::tree;

// Launch as a programmatic dependent of the kernel just launched on the
// stream: only for a second kernel of the same call, which waits
// (griddepcontrol.wait) before it reads what the first one wrote.
template <typename... KArgs, typename... Args>
cudaError_t launch_second(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem,
                          cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

// Dynamic shared memory above 48 KB needs the attribute once per kernel and
// device; `done` is the kernel's own flag word (one bit per device).
template <typename K>
cudaError_t allow_smem(K kern, int smem, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && (done.load(std::memory_order_relaxed) >> dev) & 1ull) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return e;
}

// Which kernel, by type and by the most rows a KV head can have.  16 x 32K rows,
// 8 KV heads, bf16, pages of 64, tree_mma against tree_wide, us: D = 64, 4 rows
// 199 / 224, 16 rows 219 / 226; D = 128, 4 rows 330 / 335, 16 rows 324 / 342; D =
// 256, 8 rows 640 / 700 (16 rows do not fit tree_mma's registers).  From 17 rows on
// tree_mma would read the cache once more per 16 rows: 32 rows of D = 128 took 623
// / 346.  In short contexts tree_wide's set-up shows too: one request of 64 rows
// 8.3 / 12.9, 16 of 1024 14.7 / 22.
enum TreeKernel { kTreeF32, kTreeMma, kTreeWide };

TreeKernel tree_kernel(int dtype, int rows, int D) {
  if (dtype == B2A_F32) return kTreeF32;
  return rows <= (D > 128 ? 8 : 16) ? kTreeMma : kTreeWide;
}

// Query rows of an item and keys of a tile.
int tree_rows_per_block(TreeKernel k, int rows, int group) {
  if (k == kTreeF32) return TR::kF32Rows;
  if (k == kTreeWide) return TR::kWideM / group * group;
  return rows <= 8 ? 8 : 16;
}
int tree_tile(TreeKernel k, int D) {
  if (k == kTreeF32 || k == kTreeWide) return D > 128 ? 64 : 128;
  return TR::kRows;
}
// Whole items per CTA, one launch without parts to join, or items cut evenly
// over the CTAs.  Cutting costs some 12 us (division of the work by tiles, the
// parts, the second kernel).  Whole against cut, 32/8 heads x 64, f16, pages of
// 16, one node, us: 1 request of 512 rows 9.5 / 13.4, of 1024 12.7 / 13.6, of 2048
// 19.5 / 14.1; 4 of 1024 12.9 / 17.6, of 4000 32 / 22; 16 of 1024 13.5 / 26.5, of
// 4000 35.5 / 45; 64 of 200 to 2047 55 / 80, of 4000 123 / 128.  tree_wide, bf16 x
// 128, 8 nodes: 1 of 1000 15.6 / 19.3, 16 of 1000 17.5 / 35.4, of 4000 49 / 77.  So:
// short contexts, and middling ones where the items alone nearly fill the SMs.
// Where the rule is behind: requests that do not divide by the teams (19 of 4000
// rows 63 / 52: two rounds of items for ten teams of 18) and few short f32 requests
// (1 of 1000 rows 95 / 25, 16 of 1000 97 / 106: one item's tiles in series).
bool tree_always_whole(int max_len) { return max_len <= 1024; }
bool tree_by_item(int max_len, int B, int KV) {
  return tree_always_whole(max_len) ||
         (max_len <= 4096 && static_cast<long long>(B) * KV * 4 >= 3LL * b2a_host::sm_count());
}
int max_rows_blocks(int rows, int rows_per_block) { return (rows + rows_per_block - 1) / rows_per_block; }

struct TreeArgs {
  const void *q, *k, *v;
  long long q_stride, page_stride;
  void* out;
  float *lse, *part_o, *part_ml;
  int D, dtype, page_rows, grid;
  TreeKernel kernel;
  float sscale;
  bool merge;
  TR::Batch bt;
  cudaStream_t st;
};

template <typename T, int D>
int tree_merge(const TreeArgs& a) {
  if (!a.merge) return B2A_OK;
  const int gy = (a.bt.rows_per_block + TR::kMergeWarps - 1) / TR::kMergeWarps;
  const cudaError_t e = launch_second(TR::tree_merge_kernel<T, D>, dim3(a.grid, gy),
                                      dim3(TR::kMergeWarps * 32), 0, a.st, a.bt,
                                      const_cast<const float*>(a.part_o),
                                      const_cast<const float*>(a.part_ml),
                                      static_cast<T*>(a.out), a.lse);
  return e == cudaSuccess ? B2A_OK : b2a_host::cuda_fail(e, "tree_decode merge launch");
}

// Tensor map of a pool for boxes of box_rows rows x box_cols x 64 columns,
// written as [64-column box][row][128 bytes]: 64 columns, rows of a page, column
// boxes, KV heads, pages.  L2 fetches no more than a row of one head (128
// bytes for D = 64): the next head's bytes are another CTA's.
int tree_map(CUtensorMap* m, const TreeArgs& a, const void* base, int box_rows, int box_cols) {
  const uint64_t dims[5] = {64, static_cast<uint64_t>(a.page_rows), static_cast<uint64_t>(a.D / 64),
                            static_cast<uint64_t>(a.bt.KV), static_cast<uint64_t>(a.bt.n_pages)};
  const uint64_t strides[4] = {static_cast<uint64_t>(a.bt.KV) * a.D * 2, 128,
                               static_cast<uint64_t>(a.D) * 2,
                               static_cast<uint64_t>(a.page_stride) * 2};
  const uint32_t box[5] = {64, static_cast<uint32_t>(box_rows), static_cast<uint32_t>(box_cols), 1, 1};
  return b2a_host::make_tmap(m,
                             a.dtype == B2A_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                             5, const_cast<void*>(base), dims, strides, box,
                             CU_TENSOR_MAP_SWIZZLE_128B,
                             a.D > 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B
                                      : CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
}

template <typename T, int D, int NT>
int tree_mma(const TreeArgs& a) {
  auto kern = TR::tree_mma_kernel<T, D, NT>;
  constexpr int smem = TR::MmaCfg<D, NT>::kSmem;
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = allow_smem(kern, smem, done);
  if (e != cudaSuccess) return b2a_host::cuda_fail(e, "cudaFuncSetAttribute(tree_decode)");
  const int piece = a.bt.table && a.page_rows < TR::kRows ? a.page_rows : TR::kRows;
  CUtensorMap tk, tv;
  int rc = tree_map(&tk, a, a.k, piece, D / 64);
  if (rc == B2A_OK) rc = tree_map(&tv, a, a.v, piece, D / 64);
  if (rc) return rc;
  e = b2a_host::launch(kern, dim3(a.grid), dim3(TR::kMmaThreads), smem, a.st, tk, tv, a.bt,
                       static_cast<const T*>(a.q), a.q_stride, static_cast<const T*>(a.v),
                       a.page_stride, static_cast<T*>(a.out), a.lse, a.part_o, a.part_ml, piece,
                       a.sscale);
  if (e != cudaSuccess) return b2a_host::cuda_fail(e, "tree_decode launch");
  return tree_merge<T, D>(a);
}

template <typename T, int D>
int tree_wide(const TreeArgs& a) {
  auto kern = TR::tree_wide_kernel<T, D>;
  using C = TR::WideCfg<D>;
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = allow_smem(kern, C::kSmem, done);
  if (e != cudaSuccess) return b2a_host::cuda_fail(e, "cudaFuncSetAttribute(tree_wide)");
  const int piece = a.bt.table && a.page_rows < C::kBN ? a.page_rows : C::kBN;
  const int cols = piece == C::kBN ? D / 64 : 1;
  CUtensorMap tq, tk, tv;
  int rc = tree_map(&tk, a, a.k, piece, cols);
  if (rc == B2A_OK) rc = tree_map(&tv, a, a.v, piece, cols);
  // q as nodes of [H][D]: a box is the rows of one KV head's group x the
  // block's nodes
  const uint64_t dims[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(a.bt.H),
                            static_cast<uint64_t>(a.bt.n_tok)};
  const uint64_t strides[2] = {static_cast<uint64_t>(D) * 2, static_cast<uint64_t>(a.q_stride) * 2};
  const uint32_t box[3] = {64, static_cast<uint32_t>(a.bt.group),
                           static_cast<uint32_t>(a.bt.rows_per_block / a.bt.group)};
  if (rc == B2A_OK)
    rc = b2a_host::make_tmap(&tq, a.dtype == B2A_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                      : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                             3, const_cast<void*>(a.q), dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  e = b2a_host::launch(kern, dim3(a.grid), dim3(TR::kWideThreads), C::kSmem, a.st, tq, tk, tv, a.bt,
                       static_cast<const T*>(a.v), a.page_stride, static_cast<T*>(a.out), a.lse, a.part_o, a.part_ml, piece, a.sscale);
  if (e != cudaSuccess) return b2a_host::cuda_fail(e, "tree_wide launch");
  return tree_merge<T, D>(a);
}

template <typename T, int D>
int tree_16bit(const TreeArgs& a) {
  if (a.kernel == kTreeWide) return tree_wide<T, D>(a);
  if constexpr (D <= 128) {
    if (a.bt.rows_per_block == 16) return tree_mma<T, D, 2>(a);
  }
  return tree_mma<T, D, 1>(a);
}

template <int D>
int tree_f32(const TreeArgs& a) {
  auto kern = TR::tree_f32_kernel<D>;
  constexpr int smem = TR::F32Cfg<D>::kSmem;
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = allow_smem(kern, smem, done);
  if (e != cudaSuccess) return b2a_host::cuda_fail(e, "cudaFuncSetAttribute(tree_f32)");
  e = b2a_host::launch(kern, dim3(a.grid), dim3(TR::kF32Threads), smem, a.st,
                       static_cast<const float*>(a.k), static_cast<const float*>(a.v),
                       a.page_stride, a.bt, static_cast<const float*>(a.q), a.q_stride,
                       static_cast<float*>(a.out), a.lse, a.part_o, a.part_ml, a.sscale);
  if (e != cudaSuccess) return b2a_host::cuda_fail(e, "tree_f32 launch");
  return tree_merge<float, D>(a);
}

template <int D>
int tree_dispatch(const TreeArgs& a) {
  if (a.kernel == kTreeF32) return tree_f32<D>(a);
  if (a.dtype == B2A_BF16) return tree_16bit<__nv_bfloat16, D>(a);
  return tree_16bit<__half, D>(a);
}

// Most CTAs of a grid of teams (a team has a CTA per KV head, or up to
// kTreeBlocks).
constexpr int kTreeBlocks = 8;
int tree_ctas(int KV) {
  const int sms = b2a_host::sm_count();
  return KV > sms ? KV : sms;
}

size_t tree_part_o_bytes(int D, int KV, int rows_per_block) {
  return static_cast<size_t>(2) * tree_ctas(KV) * rows_per_block * D * sizeof(float);
}

int log2_of(int x) {
  int s = 0;
  while ((1 << s) < x) ++s;
  return s;
}

bool power_of_two(int x) { return x > 0 && (x & (x - 1)) == 0; }

}  // namespace

extern "C" {

size_t b2a_tree_decode_workspace_bytes(int max_nodes, int H, int KV, int D, int dtype, int max_len) {
  if (max_nodes <= 0 || H <= 0 || KV <= 0 || D <= 0 || H % KV != 0) return 0;
  if (tree_always_whole(max_len)) return 0;
  const int rows = max_nodes * (H / KV);
  const int rb = tree_rows_per_block(tree_kernel(dtype, rows, D), rows, H / KV);
  return tree_part_o_bytes(D, KV, rb) + static_cast<size_t>(2) * tree_ctas(KV) * rb * 2 * sizeof(float);
}

int b2a_tree_decode(const void* q, long long q_tok_stride, const void* k_cache,
                    const void* v_cache, int n_pages, int page_rows, long long page_stride,
                    const int* table_dev, long long table_stride, int table_width,
                    const int* lens_dev, const int* cu_dev, const int* parents_dev, void* out,
                    float* lse_out, void* workspace, size_t workspace_bytes, int B, int n_tok,
                    int max_nodes, int H, int KV, int D, int dtype, float scale, int max_len,
                    void* stream) {
  if (!q || !k_cache || !v_cache || !lens_dev || !cu_dev || !out)
    return fail(B2A_ERR_ARG, "tree_decode: null pointer argument");
  if (B <= 0 || n_tok < 0 || H <= 0 || KV <= 0 || D <= 0 || n_pages <= 0 || page_rows <= 0 ||
      max_len <= 0)
    return fail(B2A_ERR_ARG, "tree_decode: sizes must be positive (B=%d n_tok=%d H=%d KV=%d D=%d "
                "n_pages=%d page_rows=%d max_len=%d)", B, n_tok, H, KV, D, n_pages, page_rows, max_len);
  if (max_nodes <= 0 || max_nodes > B2A_TREE_MAX_NODES)
    return fail(B2A_ERR_ARG, "tree_decode: max_nodes %d (1..%d)", max_nodes, B2A_TREE_MAX_NODES);
  if (H % KV != 0) return fail(B2A_ERR_SHAPE, "tree_decode: H=%d is not a multiple of KV=%d", H, KV);
  const int es = b2a_host::elem_size(dtype);
  if (es == 0) return fail(B2A_ERR_DTYPE, "tree_decode: dtype %d", dtype);
  if (D != 64 && D != 128 && D != 256)
    return fail(B2A_ERR_UNSUPPORTED, "tree_decode: head_dim %d (64/128/256)", D);
  if (!(scale > 0.f) || !isfinite(scale)) return fail(B2A_ERR_ARG, "tree_decode: scale must be positive");
  const long long page_elems = static_cast<long long>(page_rows) * KV * D;
  if (page_stride == 0) page_stride = page_elems;
  if (page_stride < page_elems)
    return fail(B2A_ERR_SHAPE, "tree_decode: page_stride %lld < page_rows*KV*D %lld", page_stride, page_elems);
  if (table_dev) {
    if (!power_of_two(page_rows) || page_rows < 16)
      return fail(B2A_ERR_SHAPE, "tree_decode: page_rows %d must be a power of two from 16 up", page_rows);
    if (table_width <= 0 || table_stride < table_width ||
        static_cast<long long>(table_width) * page_rows < max_len)
      return fail(B2A_ERR_SHAPE, "tree_decode: a table row of %d pages (stride %lld) does not hold max_len %d rows",
                  table_width, table_stride, max_len);
  } else if (n_pages < B || page_rows < max_len) {
    return fail(B2A_ERR_SHAPE, "tree_decode: %d blocks of %d rows for %d sequences of up to %d",
                n_pages, page_rows, B, max_len);
  }
  if (q_tok_stride == 0) q_tok_stride = static_cast<long long>(H) * D;
  if (q_tok_stride < static_cast<long long>(H) * D)
    return fail(B2A_ERR_SHAPE, "tree_decode: q_tok_stride %lld < H*D", q_tok_stride);
  if (!b2a_host::aligned16(q) || !b2a_host::aligned16(k_cache) || !b2a_host::aligned16(v_cache) ||
      !b2a_host::aligned16(out) || !b2a_host::aligned16(workspace) || (q_tok_stride * es) % 16 != 0 ||
      (page_stride * es) % 16 != 0)
    return fail(B2A_ERR_ALIGN, "tree_decode: q, caches, out, workspace and their strides must be 16-byte aligned");
  if (n_tok == 0) return B2A_OK;
  const int group = H / KV;
  if (group > 128 || static_cast<long long>(max_nodes) * group > 16384)
    return fail(B2A_ERR_UNSUPPORTED, "tree_decode: group %d", group);

  TreeArgs a = {};
  const int rows = max_nodes * group;
  a.kernel = tree_kernel(dtype, rows, D);
  const int rb = tree_rows_per_block(a.kernel, rows, group);
  const int tile = tree_tile(a.kernel, D);
  a.bt = TR::Batch{lens_dev, cu_dev, parents_dev, table_dev, table_stride, B, n_tok, max_nodes,
                   max_len, n_pages, table_dev ? log2_of(page_rows) : 0, H, KV, group, rb, tile, 0, 1, 1, 1, 1};
  // Side by side in a team: the KV heads, or, where a request has several
  // blocks of query rows, those (as many as the average request has, or as the
  // largest where that is not much more; a request with more goes round again).
  // 16 x 32K rows, bf16, 32/8 heads x 128, 128 nodes (4 blocks), before
  // tree_wide's third softmax warpgroup: 1465 us with the heads side by side (every
  // block reads K and V from HBM again), 1170 with the blocks.
  const long long avg_rows = static_cast<long long>(n_tok) * group / B;
  long long blks = (avg_rows + rb / 2) / rb;
  const int most = max_rows_blocks(rows, rb);
  if (blks > most || 4 * blks >= 3 * most) blks = most;
  if (blks > kTreeBlocks) blks = (blks + (blks + kTreeBlocks - 1) / kTreeBlocks - 1) / ((blks + kTreeBlocks - 1) / kTreeBlocks);
  a.bt.m_blks = blks > 1 && a.kernel == kTreeWide ? static_cast<int>(blks) : 1;
  a.bt.m_heads = a.bt.m_blks > 1 ? 1 : KV;
  const int members = a.bt.m_heads * a.bt.m_blks;
  // A list's tiles are cut evenly over the teams, at least 4 to a team (one of
  // f32, where a tile is work enough).
  const long long max_tiles = (max_len + tile - 1) / tile;
  const long long items = static_cast<long long>(B) * (KV / a.bt.m_heads) *
                          ((max_rows_blocks(rows, rb) + a.bt.m_blks - 1) / a.bt.m_blks);
  a.bt.by_item = tree_by_item(max_len, B, KV) ? 1 : 0;
  a.bt.min_units = a.bt.by_item || a.kernel == kTreeF32 ? 1 : 4;
  const long long units = (items * (a.bt.by_item ? 1 : max_tiles) + a.bt.min_units - 1) / a.bt.min_units;
  const int teams = b2a_host::sm_count() > members ? b2a_host::sm_count() / members : 1;
  a.bt.teams = static_cast<int>(units < teams ? units : teams);
  a.grid = a.bt.teams * members;
  a.merge = !a.bt.by_item;
  if (a.merge) {
    const size_t need = b2a_tree_decode_workspace_bytes(max_nodes, H, KV, D, dtype, max_len);
    if (!workspace || workspace_bytes < need)
      return fail(B2A_ERR_WORKSPACE, "tree_decode: workspace %zu bytes < %zu needed", workspace_bytes, need);
  }
  a.q = q;
  a.k = k_cache;
  a.v = v_cache;
  a.q_stride = q_tok_stride;
  a.page_stride = page_stride;
  a.out = out;
  a.lse = lse_out;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = workspace ? reinterpret_cast<float*>(static_cast<char*>(workspace) + tree_part_o_bytes(D, KV, rb)) : nullptr;
  a.D = D;
  a.dtype = dtype;
  a.page_rows = page_rows;
  a.sscale = scale * TR::kLog2e;
  a.st = static_cast<cudaStream_t>(stream);
  if (D == 64) return tree_dispatch<64>(a);
  if (D == 128) return tree_dispatch<128>(a);
  return tree_dispatch<256>(a);
}

}  // extern "C"
