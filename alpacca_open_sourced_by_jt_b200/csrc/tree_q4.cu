// Tree attention (tree_decode.cu has the operator, tree_work.cuh the division of
// the work) over a 4-bit cache (q4.cuh has its layout).
//
// A cached row is 1.125 D bytes for K and V together, 0.28 of a 16-bit row's, so
// that what warps do with a row weighs as much as reading it.  Nothing is
// converted: a code is a f16 subnormal as it stands in its word (mask, no
// arithmetic), the block scales go onto f32 numbers.
//   scores    S = Q.K^T on m16n8k16 MMAs, block by block of 32 dims:
//             s += d_k[key][block] * (sum q c - 8 sum q), the second term as the
//             MMA's initial accumulator.  Codes of odd word places are 16 times
//             larger (2^-20): q is 16 times smaller there.  Each row of q is
//             scaled by a power of two to a largest element in [2^14, 2^15), so
//             f16 holds bf16 q's too; elements 2^28 times smaller than the row's
//             largest lose bits.
//   output    O^T += V^T.W^T with w = p d_v[key][block] rounded to f16 once: one
//             operand per block.  -8 sum w comes from an MMA of its own per block
//             (ones in row `block` of A: all blocks share four accumulators).
//             f16 w: 2^-12 of each weight, as tree_mma_kernel's P for f16 caches.
// The softmax runs relative to a number per query row that is at least (within
// 2^8) the largest score + log2 |d_v|, so w neither overflows nor, where it counts,
// falls under f16 whatever the scales are.  Scores, sums and accumulators are
// f32.  Hidden keys have w = 0 whatever their bytes say.
//
// S has the queries on its rows, so an accumulator is already the B operand of the
// second product (no transposition), and a lane's four keys of a granule are rows
// 4t .. 4t + 3, side by side in the pool.
//
// One persistent CTA per SM.  One warp plans: it walks the CTA's items and looks up
// their pages, segment by segment, into a queue in shared memory.  The others take
// the steps (32 keys) of a segment in turn.  Each brings its own steps, one bulk
// copy or two where pages have 16 rows, through a ring of its own, so they meet only
// at an item's end.
#include <limits.h>
#include <math.h>

#include "b2a_common.cuh"
#include "q4.cuh"
#include "tree_work.cuh"

namespace b2a {
namespace tree {

constexpr int kQ4Keys = 32;  // keys of a step (and of a tile of the work division)

// What the planning warp hands on: steps t0 .. t1 - 1 of an item and their pages.
constexpr int kQ4Rounds = 8;  // steps of a warp in a segment
constexpr int kQ4Queue = 4;

template <int W>
struct Q4Seg {
  Item it;
  int t0, t1;
  int last;      // the item ends with it
  int end;       // nothing follows (1, with requests left out 2)
  int gone;      // some granule has no page
  int g0;        // number of step t0 among all of the CTA's
  int pages[2][kQ4Rounds * W];  // of a step's two granules, -1: none
};

template <int W, int S>
struct alignas(128) Q4Shared {  // (the rings stand behind it)
  static constexpr int kStepKeys = kQ4Keys, kTileSteps = 1;  // a step's keys, a tile's steps
  static constexpr bool kItems = false;            // the items go by a queue of their own, too
  uint64_t full[W][S];                             // a warp's stages
  uint64_t seg_full[kQ4Queue], seg_empty[kQ4Queue];
  uint64_t handed, joined, read;                   // at an item's end
  uint4 sees[W][16];                               // the nodes that a warp's rows see
  Q4Seg<W> seg[kQ4Queue];
};

template <int D, int NT>
struct Q4Cfg {
  static constexpr int NB = D / 32;
  static constexpr int kGranule = q4::granule_bytes(D);
  static constexpr int kStage = 2 * kGranule;
  static constexpr int kWarps = NT == 1 && D <= 128 ? 15 : 7;
  static constexpr int RB = 8 * NT;
  static constexpr int kPad = D + 4;
  static constexpr int kMerge = (kWarps + 1) / 2 * RB * (kPad + 2) * 4;  // half the warps' rows, maxima and sums
  static constexpr int kFit = (227 * 1024 - static_cast<int>(sizeof(Q4Shared<kWarps, 6>)) - kMerge) / (kWarps * kStage);
  static constexpr int kStages = kFit > 6 ? 6 : kFit;
  using Shared = Q4Shared<kWarps, kStages>;
  static constexpr int kSmem = kWarps * kStages * kStage + kMerge + static_cast<int>(sizeof(Shared));
  static constexpr int kThreads = (kWarps + 1) * 32;
  static_assert(kStages >= 2 && kSmem <= 227 * 1024, "ring");
};

// One bulk copy (both addresses and the size multiples of 16 bytes).
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// (No volatile asm: the compiler moves loads and products of a step past one
// another; what orders the ring is in the waits.)
__device__ __forceinline__ void mma_f16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1, const float* c) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]),
        "f"(c[3]));
}

// The planning warp.  Requests are looked at 32 at a time, one by each lane.
template <int W, typename Shared>
__device__ __forceinline__ void q4_plan(const Batch& bt, Shared& sh, int lane) {
  constexpr int TS = Shared::kTileSteps, SK = Shared::kStepKeys;
  const Start start = locate(bt, team_of(bt, blockIdx.x));
  long long off = start.off, left = start.left;
  int b = start.b, base = -32, slot = 0, items = 0, steps = 0;
  uint32_t round = 0;
  int n32 = 0, len32 = 0, node32 = 0;  // of request base + lane
  const bool split = bt.table && bt.page_shift == 4;
  auto room = [&]() {  // a free place in the queue
    return round == 0 ||
           __all_sync(0xffffffffu, mbar_wait(&sh.seg_empty[slot], (round & 1) ^ 1, 0x3F200)) != 0;
  };
  auto hand_on = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.seg_full[slot]);
    if (++slot == kQ4Queue) {
      slot = 0;
      ++round;
    }
  };
  while (left > 0 && b < bt.B) {
    if (b - base >= 32) {
      base = b & ~31;
      n32 = len32 = node32 = 0;
      if (base + lane < bt.B) {
        request(bt, base + lane, n32, len32, start.left_out);
        node32 = bt.cu[base + lane];
      }
    }
    Item it;
    it.b = b;
    it.n = __shfl_sync(0xffffffffu, n32, b - base);
    it.len = __shfl_sync(0xffffffffu, len32, b - base);
    it.node0 = __shfl_sync(0xffffffffu, node32, b - base);
    it.tiles = (it.len + it.n + TS * SK - 1) / (TS * SK);
    const long long u = units_of(bt, it.n, it.len);
    if (off >= u) {
      off -= u;
      ++b;
      continue;
    }
    // (as Walker::next)
    const int per = bt.by_item ? 1 : it.tiles;
    const int idx = (off >> 31) == 0 ? static_cast<int>(static_cast<uint32_t>(off) / static_cast<uint32_t>(per))
                                     : static_cast<int>(off / per);
    const int at = static_cast<int>(off - static_cast<long long>(idx) * per);
    int take = per - at;
    if (take > left) take = static_cast<int>(left);
    it.t0 = bt.by_item ? 0 : at;
    it.t1 = bt.by_item ? it.tiles : at + take;
    off += take;
    left -= take;
    if (!member_item(bt, blockIdx.x, idx, blocks_of(bt, it.n), it.kvh, it.blk)) continue;
    const int rows = it.len + it.n;
    if constexpr (Shared::kItems) {
      const int place = items % kQ4Queue;
      if (items >= kQ4Queue && !__all_sync(0xffffffffu, mbar_wait(&sh.item_empty[place], (items / kQ4Queue - 1) & 1, 0x3F210)))
        return;
      if (lane == 0) {
        sh.item[place] = it;
        sh.item_end[place] = 0;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.item_full[place]);
      ++items;
    }
    for (int t0 = it.t0 * TS; t0 < it.t1 * TS; t0 += kQ4Rounds * W) {
      if (!room()) return;
      Q4Seg<W>& seg = sh.seg[slot];
      const int t1 = min(t0 + kQ4Rounds * W, it.t1 * TS);
      bool gone = false;
#pragma unroll 4
      for (int i = lane; i < t1 - t0; i += 32) {
        const int row = (t0 + i) * SK;
        const bool one = row < rows, two = SK > 16 && row + 16 < rows;  // (a tile's last steps may hold nothing)
        const int e0 = one ? table_entry(bt, it.b, row) : 0;
        const int e1 = split && two ? table_entry(bt, it.b, row + 16) : e0;
        const int p0 = checked_page(bt, it.b, e0), p1 = checked_page(bt, it.b, e1);
        seg.pages[0][i] = one && p0 < bt.n_pages ? p0 : -1;
        seg.pages[1][i] = two && p1 < bt.n_pages ? p1 : -1;
        gone |= p0 >= bt.n_pages || p1 >= bt.n_pages;
      }
      gone = __any_sync(0xffffffffu, gone);
      if (lane == 0) {
        seg.it = it;
        seg.t0 = t0;
        seg.t1 = t1;
        seg.last = t1 == it.t1 * TS;
        seg.end = 0;
        seg.gone = gone;
        seg.g0 = steps;
      }
      steps += t1 - t0;
      hand_on();
    }
  }
  if constexpr (Shared::kItems) {
    const int place = items % kQ4Queue;
    if (items >= kQ4Queue && !__all_sync(0xffffffffu, mbar_wait(&sh.item_empty[place], (items / kQ4Queue - 1) & 1, 0x3F210)))
      return;
    if (lane == 0) sh.item_end[place] = start.left_out ? 2 : 1;
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.item_full[place]);
  }
  if (!room()) return;
  if (lane == 0) sh.seg[slot].end = start.left_out ? 2 : 1;
  hand_on();
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(Q4Cfg<D, NT>::kThreads, 1) tree_q4_kernel(
    const __grid_constant__ Batch bt, const __grid_constant__ q4::Pool pool, const T* __restrict__ q,
    long long q_stride, T* __restrict__ out, float* __restrict__ lse, float* __restrict__ part_o,
    float* __restrict__ part_ml, float scale_log2) {
  using C = Q4Cfg<D, NT>;
  constexpr int NB = C::NB, W = C::kWarps, RB = C::RB, H = (W + 1) / 2;  // H: the lower half of the warps
  extern __shared__ __align__(128) uint8_t q4_smem[];
  typename C::Shared& sh = *reinterpret_cast<typename C::Shared*>(q4_smem);
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x < W) {
    for (int s = 0; s < C::kStages; ++s) mbar_init(&sh.full[threadIdx.x][s], 1);
  } else if (threadIdx.x == W * 32) {
    for (int i = 0; i < kQ4Queue; ++i) {
      mbar_init(&sh.seg_full[i], 1);
      mbar_init(&sh.seg_empty[i], W);
    }
    mbar_init(&sh.handed, W / 2);
    mbar_init(&sh.joined, (W + 1) / 2);
    mbar_init(&sh.read, W);
  }
  fence_mbar_init();
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (warp == W) {
    q4_plan<W>(bt, sh, lane);
    return;
  }
  const int g = lane >> 2, t = lane & 3;
  uint8_t* ring = q4_smem + sizeof(typename C::Shared) + warp * C::kStages * C::kStage;
  float* merge = reinterpret_cast<float*>(q4_smem + sizeof(typename C::Shared) + W * C::kStages * C::kStage);
  float* merge_ml = merge + H * RB * C::kPad;
  // A whole warp's wait, with one answer for all lanes.  After one that ran out the
  // warp leaves; the others' waits for it run out too.
  auto arrived = [](uint64_t* bar, uint32_t parity, int where) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, where)) != 0;
  };

  // ---- this warp's copies, ahead of its products -----------------------------------------
  uint32_t f_seg = 0;       // segments taken by the copies
  int f_step = 0, f_t1 = 0; // the next step, the segment's end (none taken: equal)
  uint32_t f_stage = 0, in_ring = 0;
  uint32_t bad = 0;         // bit 2 s + i: granule i of stage s has no page
  bool f_end = false;
  const bool split = bt.table && bt.page_shift == 4;  // a step's granules lie in two pages
  const int page_mask = bt.table ? (1 << bt.page_shift) - 1 : INT_MAX;
  // Brings the warp's next step if the plan is that far.
  auto bring = [&]() {
    while (f_step >= f_t1) {
      if (f_end || !mbar_test(&sh.seg_full[f_seg % kQ4Queue], (f_seg / kQ4Queue) & 1)) return;
      const Q4Seg<W>& seg = sh.seg[f_seg % kQ4Queue];
      f_end = seg.end != 0;
      if (f_end) return;
      f_step = seg.t0 + warp;
      f_t1 = seg.t1;
      ++f_seg;
    }
    const Q4Seg<W>& seg = sh.seg[(f_seg - 1) % kQ4Queue];
    const int i = f_step - seg.t0;
    const int p0 = seg.pages[0][i], p1 = seg.pages[1][i];
    if (seg.gone) {
      bad = (bad & ~(3u << (2 * f_stage))) | ((p0 < 0 ? 1u : 0u) | (p1 < 0 ? 2u : 0u)) << (2 * f_stage);
    } else {
      bad &= ~(3u << (2 * f_stage));
    }
    if (lane == 0) {
      uint64_t* bar = &sh.full[warp][f_stage];
      uint8_t* dst = ring + f_stage * C::kStage;
      const int row = (f_step * kQ4Keys) & page_mask, row1 = (f_step * kQ4Keys + 16) & page_mask;
      mbar_arrive_expect_tx(bar, ((p0 >= 0 ? 1 : 0) + (p1 >= 0 ? 1 : 0)) * C::kGranule);
      const unsigned char* src = q4::granule(pool, D, p0, seg.it.kvh, row);
      if (p0 >= 0) bulk_load(dst, src, p1 >= 0 && !split ? 2 * C::kGranule : C::kGranule, bar);
      if (p1 >= 0 && split)
        bulk_load(dst + C::kGranule, q4::granule(pool, D, p1, seg.it.kvh, row1), C::kGranule, bar);
    }
    f_step += W;
    ++in_ring;
    if (++f_stage == C::kStages) f_stage = 0;
  };

  uint32_t stage = 0, phase = 0, items = 0;
  int end = 0;
  // the lane's K words of keys 2j, 2j + 1 of each four (their partners two rows on)
  const int k_at = (4 * (g >> 1) + (g & 1)) * (16 * (NB < 4 ? NB : 4)) + t * (4 * (NB < 4 ? NB : 4));
  const uint32_t sel = g < 4 ? 0x5410u : 0x7632u;  // even dims stand in a word's low half
  // an item's state
  // A operands.  Two row tiles: [block][places 0, 2 | 1, 3 of the words].  One: both in
  // one operand, places 1, 3 on rows 8 to 15; of each product half the rows count.
  uint32_t qa[NB][NT][4];
  float qc[NB][NT];       // -8 sum q of a block
  float sscale[NT];
  float o[2 * NB][NT][4], ws[NT][4], m[NT], l[NT];
  uint32_t spoilt[NT];    // blocks with a NaN scale that the row sees
  bool have_anc = false;
  for (uint32_t c_seg = 0;; ++c_seg) {
    if (!arrived(&sh.seg_full[c_seg % kQ4Queue], (c_seg / kQ4Queue) & 1, 0x3F100)) return;
    const Q4Seg<W>& seg = sh.seg[c_seg % kQ4Queue];
    end = seg.end;
    if (end) break;
    while (in_ring < C::kStages) {
      const uint32_t before = in_ring;
      bring();
      if (in_ring == before) break;
    }
    const Item& it = seg.it;
    const int R = it.n * bt.group, row_lo = it.blk * RB;
    if (seg.t0 == it.t0) {
      // ---- the item's rows of q, scaled, and -8 sum q of each block -----------------
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = row_lo + nt * 8 + g;
        const bool valid = r < R;
        const int node = valid ? r / bt.group : 0;
        const int head = it.kvh * bt.group + (valid ? r - node * bt.group : 0);
        const T* qr = q + (it.node0 + node) * q_stride + head * D + 8 * t;
        float x[NB][8];
        float big = 0.f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[b][e] = 0.f;
          if (valid) paged::load8(qr + 32 * b, x[b]);
#pragma unroll
          for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(x[b][e]));
        }
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        // 2^k with big * 2^k in [2^14, 2^15); rows of zeros, infinities: k = 0
        int k = 0;
        if (big > 0.f && big < INFINITY) k = max(-126, min(126, 14 + 127 - static_cast<int>(__float_as_uint(big) >> 23)));
        const float up = __uint_as_float(static_cast<uint32_t>(127 + k) << 23);
        sscale[nt] = scale_log2 * 16777216.f * __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // word place i: dims 2i, 2i + 1
            const float f = i & 1 ? up * 0.0625f : up;
            const __half2 h = __floats2half2_rn(x[b][2 * i] * f, x[b][2 * i + 1] * f);
            if constexpr (NT == 1) qa[b][0][(i >> 1) * 2 + (i & 1)] = *reinterpret_cast<const uint32_t*>(&h);
            else qa[b][i & 1][(i >> 1) * 2 + nt] = *reinterpret_cast<const uint32_t*>(&h);
            const float2 y = __half22float2(h);
            sum += (y.x + y.y) * (i & 1 ? 16.f : 1.f);
          }
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          qc[b][nt] = sum * (-8.f / 16777216.f);
        }
      }
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][nt][e] = 0.f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m[nt] = -INFINITY;
        l[nt] = 0.f;
        spoilt[nt] = 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) ws[nt][e] = 0.f;
      }
      have_anc = false;
    }

    for (int st = seg.t0 + warp; st < seg.t1; st += W) {
      if (in_ring == 0) bring();  // (its segment is the products', so it is there)
      if (!arrived(&sh.full[warp][stage], phase, 0x3F000 | warp)) return;
      const uint8_t* base = ring + stage * C::kStage;
      int row0 = st * kQ4Keys;
      const bool tail = row0 + kQ4Keys > it.len;
      const uint32_t no_page = (bad >> (2 * stage)) & 3u;
      if (tail && !have_anc) {
        // the nodes that the rows see: a lane per row
        have_anc = true;
        if (lane < RB) {
          const int node = min((row_lo + lane) / bt.group, it.n - 1);
          uint32_t anc[kWords];
#pragma unroll
          for (int w = 0; w < kWords; ++w) {
            const int k = node + 1 - w * 32;
            anc[w] = bt.parents ? 0u : k >= 32 ? 0xffffffffu : (k > 0 ? (1u << k) - 1u : 0u);
          }
          if (bt.parents) {
            int at = node;
            while (true) {
#pragma unroll
              for (int w = 0; w < kWords; ++w)
                if ((at >> 5) == w) anc[w] |= 1u << (at & 31);
              const int up = __ldg(bt.parents + it.node0 + at);
              if (up < 0 || up >= at) {
                if (up != -1) set_dev_error(B2A_ERR_POSITION, it.b);
                break;
              }
              at = up;
            }
          }
          sh.sees[warp][lane] = make_uint4(anc[0], anc[1], anc[2], anc[3]);
        }
        __syncwarp();
      }

      // (a granule at a time: both at once need more registers than 15 warps have)
#pragma unroll 1
      for (int gr = 0; gr < 2; ++gr, base += C::kGranule, row0 += 16) {
        // ---- scores ----------------------------------------------------------------
        uint32_t dk[NB * 2];  // [key][block] f16
#pragma unroll
        for (int i = 0; i < NB / 2; ++i) {
          const uint4 u = *reinterpret_cast<const uint4*>(base + 16 * D + t * (8 * NB) + i * 16);
          dk[4 * i] = u.x; dk[4 * i + 1] = u.y; dk[4 * i + 2] = u.z; dk[4 * i + 3] = u.w;
        }
        float2 s[NT][2];  // of keys 4t, 4t + 1 | 4t + 2, 4t + 3
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = make_float2(0.f, 0.f);
        constexpr int NBP = NB < 4 ? NB : 4;
#pragma unroll
        for (int pl = 0; pl < NB / NBP; ++pl) {
          uint32_t kw[2][NBP];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint8_t* at = base + pl * (256 * NBP) + k_at + h * (32 * NBP);
            if constexpr (NBP == 4) {
              const uint4 u = *reinterpret_cast<const uint4*>(at);
              kw[h][0] = u.x; kw[h][1] = u.y; kw[h][2] = u.z; kw[h][3] = u.w;
            } else {
              const uint2 u = *reinterpret_cast<const uint2*>(at);
              kw[h][0] = u.x; kw[h][1] = u.y;
            }
          }
#pragma unroll
          for (int bp = 0; bp < NBP; ++bp) {
            const int b = pl * NBP + bp;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t w = kw[h][bp], w8 = w >> 8;
              float acc[4], odd[4];
              const float zero[4] = {0.f, 0.f, 0.f, 0.f};
              mma_f16(acc, qa[b][0], w & 0x000f000fu, w8 & 0x000f000fu, zero);
              if constexpr (NT == 1) mma_f16(odd, qa[b][0], w & 0x00f000f0u, w8 & 0x00f000f0u, zero);
              else mma_f16(acc, qa[b][NT - 1], w & 0x00f000f0u, w8 & 0x00f000f0u, acc);
              // keys 4t + 2h, 4t + 2h + 1
              const __half* hk = reinterpret_cast<const __half*>(dk) + 2 * h * NB + b;
              const float2 d = make_float2(__half2float(hk[0]), __half2float(hk[NB]));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                s[nt][h] = fma2(d, make_float2(qc[b][nt], qc[b][nt]), s[nt][h]);
                s[nt][h] = fma2(d, make_float2(acc[2 * nt], acc[2 * nt + 1]), s[nt][h]);
                if constexpr (NT == 1) s[nt][h] = fma2(d, make_float2(odd[2], odd[3]), s[nt][h]);
              }
            }
          }
        }
        // ---- softmax ----------------------------------------------------------------
        uint32_t dv[NB * 2];  // [key][block] f16
#pragma unroll
        for (int i = 0; i < NB / 2; ++i) {
          const uint4 u = *reinterpret_cast<const uint4*>(base + 17 * D + t * (8 * NB) + i * 16);
          dv[4 * i] = u.x; dv[4 * i + 1] = u.y; dv[4 * i + 2] = u.z; dv[4 * i + 3] = u.w;
        }
        if (tail || no_page) {
          // keys that are not there, or that only some rows see, may hold anything
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = row0 + 4 * t + i - it.len;
            bool any = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              bool see = j < 0;
              if (j >= 0 && j < it.n && row_lo + nt * 8 + g < R)
                see = reinterpret_cast<const uint32_t*>(&sh.sees[warp][nt * 8 + g])[j >> 5] >> (j & 31) & 1u;
              if ((no_page >> gr) & 1u) see = false;
              float& x = i & 1 ? s[nt][i >> 1].y : s[nt][i >> 1].x;
              if (!see) x = -INFINITY;
              any |= see;
            }
            if (!any)
#pragma unroll
              for (int b = 0; b < NB / 2; ++b) dv[i * (NB / 2) + b] = 0u;
          }
        }
        auto top_scale = [&]() {  // the largest |d_v| of the lane's keys, a NaN before all
          __half2 top = __float2half2_rn(0.f);
#pragma unroll
          for (int i = 0; i < NB * 2; ++i)
            top = __hmax2_nan(top, __habs2(*reinterpret_cast<const __half2*>(&dv[i])));
          const uint32_t bits = *reinterpret_cast<const uint32_t*>(&top);
          return max(bits & 0x7fffu, bits >> 16 & 0x7fffu);
        };
        uint32_t top16 = top_scale();
        if (__any_sync(0xffffffffu, top16 > 0x7c00u)) {
          // A NaN scale of a key that is seen: its block's outputs become NaN at the
          // item's end; here it counts as zero.
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              uint32_t& u = dv[i * (NB / 2) + (b >> 1)];
              const uint32_t half = b & 1 ? u >> 16 : u & 0xffffu;
              if ((half & 0x7fffu) <= 0x7c00u) continue;
              u &= b & 1 ? 0x0000ffffu : 0xffff0000u;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                if ((i & 1 ? s[nt][i >> 1].y : s[nt][i >> 1].x) != -INFINITY) spoilt[nt] |= 1u << b;
            }
          top16 = top_scale();
        }
        // A power of two (its exponent) that is at least the largest |d_v| of the lane's
        // keys: with whole exponents the weight of a row's only key is exact.
        const float far = static_cast<float>(min(static_cast<int>(top16 >> 10), 30) - 14);
        bool grow = false;
        float mx[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float x = fmaxf(fmaxf(s[nt][0].x, s[nt][0].y), fmaxf(s[nt][1].x, s[nt][1].y));
          x = fmaf(x, sscale[nt], far);
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
          mx[nt] = x;
          grow |= x > m[nt] + 8.f;
        }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float now = fmaxf(m[nt], mx[nt]);
            const float alpha = now == -INFINITY ? 0.f : fast_exp2(m[nt] - now);
            m[nt] = now;
            l[nt] *= alpha;
            const float a0 = __shfl_sync(0xffffffffu, alpha, 8 * t), a1 = __shfl_sync(0xffffffffu, alpha, 8 * t + 4);
#pragma unroll
            for (int i = 0; i < 2 * NB; ++i) {
              o[i][nt][0] *= a0;
              o[i][nt][1] *= a1;
              o[i][nt][2] *= a0;
              o[i][nt][3] *= a1;
            }
            ws[nt][0] *= a0;
            ws[nt][1] *= a1;
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float mref = m[nt] == -INFINITY ? 0.f : m[nt];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 x = fma2(s[nt][h], make_float2(sscale[nt], sscale[nt]), make_float2(-mref, -mref));
            s[nt][h] = make_float2(fast_exp2(x.x), fast_exp2(x.y));  // the weights, unscaled
          }
          l[nt] += (s[nt][0].x + s[nt][0].y) + (s[nt][1].x + s[nt][1].y);
        }
        // ---- output -----------------------------------------------------------------
        const uint8_t* vb = base + 8 * D + (g & 3) * 64 + t * 16;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          uint32_t w[NT][2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const __half* hv = reinterpret_cast<const __half*>(dv) + 2 * h * NB + b;
            const float2 d = make_float2(__half2float(hv[0]), __half2float(hv[NB]));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const float2 x = mul2(s[nt][h], d);
              w[nt][h] = MmaOp<__half>::pack(x.x, x.y);
            }
          }
          const uint4 u = *reinterpret_cast<const uint4*>(vb + b * 256);
          const uint32_t lo = __byte_perm(u.x, u.y, sel), hi = __byte_perm(u.z, u.w, sel);
          const uint32_t lo8 = lo >> 8, hi8 = hi >> 8;
          const uint32_t a0[4] = {lo & 0x000f000fu, lo & 0x00f000f0u, hi & 0x000f000fu, hi & 0x00f000f0u};
          const uint32_t a1[4] = {lo8 & 0x000f000fu, lo8 & 0x00f000f0u, hi8 & 0x000f000fu, hi8 & 0x00f000f0u};
          const uint32_t one = g == b ? 0x3c003c00u : 0u;
          const uint32_t ones[4] = {one, one, one, one};  // (rows 8 to 15 are not used)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_f16(o[2 * b][nt], a0, w[nt][0], w[nt][1], o[2 * b][nt]);
            mma_f16(o[2 * b + 1][nt], a1, w[nt][0], w[nt][1], o[2 * b + 1][nt]);
            mma_f16(ws[nt], ones, w[nt][0], w[nt][1], ws[nt]);
          }
        }
      }
      // the stage is read: a next step
      __syncwarp();
      --in_ring;
      bring();
      if (++stage == C::kStages) {
        stage = 0;
        phase ^= 1;
      }
    }
    if (!seg.last) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.seg_empty[c_seg % kQ4Queue]);
      continue;
    }

    // ---------------- join the warps ---------------------------------------------------
    // the upper half hands its rows to the lower, whose rows are then added up
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      l[nt] += __shfl_xor_sync(0xffffffffu, l[nt], 1);
      l[nt] += __shfl_xor_sync(0xffffffffu, l[nt], 2);
      const bool seen_nan = __any_sync(0xffffffffu, spoilt[nt] != 0);
      if (seen_nan) {
        spoilt[nt] |= __shfl_xor_sync(0xffffffffu, spoilt[nt], 1);
        spoilt[nt] |= __shfl_xor_sync(0xffffffffu, spoilt[nt], 2);
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float w0 = -8.f * __shfl_sync(0xffffffffu, ws[nt][0], b * 4 + t);
        float w1 = -8.f * __shfl_sync(0xffffffffu, ws[nt][1], b * 4 + t);
        if (seen_nan) {
          if (__shfl_sync(0xffffffffu, spoilt[nt], 8 * t) >> b & 1u) w0 = __uint_as_float(0x7fffffffu);
          if (__shfl_sync(0xffffffffu, spoilt[nt], 8 * t + 4) >> b & 1u) w1 = __uint_as_float(0x7fffffffu);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float* x = o[2 * b + i][nt];
          x[0] = fmaf(x[0], 16777216.f, w0);
          x[1] = fmaf(x[1], 16777216.f, w1);
          x[2] = fmaf(x[2], 1048576.f, w0);
          x[3] = fmaf(x[3], 1048576.f, w1);
        }
      }
    }
    const int half = warp % H;
    float* mine = merge + half * RB * C::kPad + 2 * t * C::kPad + 8 * (g & 3) + (g >> 2);
    float* mine_ml = merge_ml + half * RB * 2;
    auto put = [&]() {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (t == 0) {
          mine_ml[(nt * 8 + g) * 2] = m[nt];
          mine_ml[(nt * 8 + g) * 2 + 1] = l[nt];
        }
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) {
          float* to = mine + nt * 8 * C::kPad + 32 * (i >> 1) + 4 * (i & 1);
          to[0] = o[i][nt][0];
          to[C::kPad] = o[i][nt][1];
          to[2] = o[i][nt][2];
          to[C::kPad + 2] = o[i][nt][3];
        }
      }
    };
    // (the item before has been read)
    if (items > 0 && !arrived(&sh.read, (items - 1) & 1, 0x3F300)) return;
    if (warp >= H) {
      put();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.handed);
    } else {
      if (!arrived(&sh.handed, items & 1, 0x3F400)) return;
#pragma unroll
      for (int nt = 0; nt < NT && warp + H < W; ++nt) {
        const float m2 = mine_ml[(nt * 8 + g) * 2], l2 = mine_ml[(nt * 8 + g) * 2 + 1];
        const float now = fmaxf(m[nt], m2), mref = now == -INFINITY ? 0.f : now;
        const float a = fast_exp2(m[nt] - mref), c = fast_exp2(m2 - mref);
        m[nt] = now;
        l[nt] = l[nt] * a + l2 * c;
        const float a0 = __shfl_sync(0xffffffffu, a, 8 * t), a1 = __shfl_sync(0xffffffffu, a, 8 * t + 4);
        const float c0 = __shfl_sync(0xffffffffu, c, 8 * t), c1 = __shfl_sync(0xffffffffu, c, 8 * t + 4);
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) {
          const float* from = mine + nt * 8 * C::kPad + 32 * (i >> 1) + 4 * (i & 1);
          o[i][nt][0] = o[i][nt][0] * a0 + from[0] * c0;
          o[i][nt][1] = o[i][nt][1] * a1 + from[C::kPad] * c1;
          o[i][nt][2] = o[i][nt][2] * a0 + from[2] * c0;
          o[i][nt][3] = o[i][nt][3] * a1 + from[C::kPad + 2] * c1;
        }
      }
      __syncwarp();
      put();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.joined);
    }
    if (!arrived(&sh.joined, items & 1, 0x3F500)) return;
    ++items;
    const int slot = part_slot(it, blockIdx.x);
    const int live = min(RB, R - row_lo);
    // warps that had no step have m = -inf and l = 0
    for (int i = threadIdx.x; i < live * (D / 8); i += W * 32) {
      const int r = i / (D / 8), d = (i - r * (D / 8)) * 8;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < H; ++w) M = fmaxf(M, merge_ml[(w * RB + r) * 2]);
      const float mref = M == -INFINITY ? 0.f : M;
      float L = 0.f, x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 0.f;
#pragma unroll 4
      for (int w = 0; w < H; ++w) {
        const float f = fast_exp2(merge_ml[(w * RB + r) * 2] - mref);
        L += merge_ml[(w * RB + r) * 2 + 1] * f;
        const float4 y0 = *reinterpret_cast<const float4*>(merge + (w * RB + r) * C::kPad + d);
        const float4 y1 = *reinterpret_cast<const float4*>(merge + (w * RB + r) * C::kPad + d + 4);
        x[0] = fmaf(y0.x, f, x[0]); x[1] = fmaf(y0.y, f, x[1]); x[2] = fmaf(y0.z, f, x[2]); x[3] = fmaf(y0.w, f, x[3]);
        x[4] = fmaf(y1.x, f, x[4]); x[5] = fmaf(y1.y, f, x[5]); x[6] = fmaf(y1.z, f, x[6]); x[7] = fmaf(y1.w, f, x[7]);
      }
      if (slot >= 0) {
        paged::store8(part_o + (static_cast<size_t>(slot) * RB + r) * D + d, x);
        if (d == 0) {
          part_ml[(static_cast<size_t>(slot) * RB + r) * 2] = M;
          part_ml[(static_cast<size_t>(slot) * RB + r) * 2 + 1] = L;
        }
      } else {
        const int rr = row_lo + r, nd = rr / bt.group;
        const size_t row = static_cast<size_t>(it.node0 + nd) * bt.H + it.kvh * bt.group + (rr - nd * bt.group);
        const float f = 1.f / L;  // a node sees itself: L > 0
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= f;
        paged::store8(out + row * D + d, x);
        if (lse && d == 0) lse[row] = (M + log2f(L)) * kLn2;
      }
    }
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(&sh.read);
      mbar_arrive(&sh.seg_empty[c_seg % kQ4Queue]);
    }
  }
  zero_unwritten<T, D>(bt, end == 2, out, lse, warp, W);
}

}  // namespace tree
}  // namespace b2a
