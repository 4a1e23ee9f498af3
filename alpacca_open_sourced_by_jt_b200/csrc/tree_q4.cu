// Tree attention (tree_decode.cu has the operator, tree_work.cuh the division of
// the work) over a 4-bit cache (q4.cuh has its layout).
//
// A cached row is 1.125 D bytes for K and V together, 0.28 of a 16-bit row's, so
// that what warps do with a row weighs as much as reading it.  Nothing is
// converted: a code is a f16 subnormal as it stands in its word (mask, no
// arithmetic), the block scales go onto f32 numbers.
//   scores    S = Q.K^T on m16n8k16 MMAs, block by block of 32 dims:
//             s += d_k[key][block] (sum q c) + d_k[key][block] (-8 sum q), two keys
//             in an operation.  Codes of odd word places are 16 times
//             larger (2^-20): q is 16 times smaller there.  Each row of q is
//             scaled by a power of two to a largest element in [2^14, 2^15), so
//             f16 holds bf16 q's too; elements 2^28 times smaller than the row's
//             largest lose bits.
//   output    O^T += V^T.W^T with w = p d_v[key][block] rounded to f16 once: one
//             operand per block.  -8 sum w comes from an MMA of its own per block
//             (ones in row `block` of A: all blocks share four accumulators).
//             f16 w: 2^-12 of each weight, as tree_mma_kernel's P for f16 caches.
// The weights p are relative to a number m per query row, and those of a block of V,
// p d_v, are held times a power of two c of the row and block.  Both follow only where
// a w would pass 2^15 (or a row's p 2^60): m then goes to the largest score, by whole
// exponents, and c to where the block's largest product is in [1/2, 1), or to where the
// products so far had theirs if that is lower.  So no w overflows, and one is under f16's
// normal numbers, off by up to 2^-25, only if it is 2^13 times smaller than the largest of
// its own block: what the blocks beside it hold does not matter.  Scores, sums and
// accumulators are f32.  Hidden keys have w = 0 whatever their bytes say.
//
// Subnormals cost bits of the sums: the MMA lines its products up by the exponents that
// they are encoded with, 2^-14, and cuts what lies 2^23 below.  In codes that is 2^-13 (places
// 0 and 2) or 2^-17 of sum w for 16 products, at worst and towards zero; a sum is off by
// 2^-18 of its terms on average (measured).  So an output element is off by up to 2^-13 of
// sum p d, some 2^-12 of what its codes leave out, and a score by as much of sum |q| d_k.
// Normal numbers (64 + code, with 72 sum w to take off) come out no better and take 200
// us instead of 162.
//
// S has the queries on its rows, so an accumulator is already the B operand of the
// second product (no transposition), and a lane's four keys of a granule are rows
// 4t .. 4t + 3, side by side in the pool.
//
// One persistent CTA per SM.  One warp feeds the others: it walks the CTA's items, looks
// up their pages and brings the steps (32 keys) in by bulk copies, one a step or two where
// pages have 16 rows, a step a lane.  The others take the steps in turn, each through a
// ring of its own, so they meet only at an item's end.
//
// Bound by latency with the 15 warps that the registers leave, behind HBM by a factor of
// 1.7: 367 instructions a granule at head_dim 128 (28 of them MMAs), 52 % of the issue slots
// used and no pipe above 36 %.  16 x 32760 rows, 32/8 heads x 128, bf16: one node 162 us (3.7
// TB/s; the 16-bit cache's kernel takes 327), 16 query rows 270; x 64 103 us and 162; 64
// requests of 200 to 8000 rows x 64, pages of 16: 94 us, an item's end and begin (join, q,
// first data) 4 us each.  With each warp looking after its own copies a fifth more.
#include <limits.h>
#include <math.h>

#include <cfloat>

#include "b2a_common.cuh"
#include "q4.cuh"
#include "tree_work.cuh"

namespace b2a {
namespace tree {

constexpr int kQ4Keys = 32;  // keys of a step (and of a tile of the work division)

constexpr int kQ4Queue = 4;

// What the feeding warp hands on.
struct Q4Item {
  Item it;
  int g0;   // number of its first step among all of the CTA's
  int end;  // nothing follows (1, with requests left out 2)
};

template <int W, int S>
struct alignas(128) Q4Shared {  // (the rings stand behind it)
  static constexpr int kStepKeys = kQ4Keys, kTileSteps = 1;  // a step's keys, a tile's steps
  uint64_t full[W][S], empty[W][S];                // a warp's stages
  uint64_t item_full[kQ4Queue], item_empty[kQ4Queue];
  uint64_t handed, joined, read;                   // at an item's end
  uint4 sees[W][16];                               // the nodes that a warp's rows see
  Q4Item item[kQ4Queue];
};

template <int D, int NT>
struct Q4Cfg {
  static constexpr int NB = D / 32;
  static constexpr int kGranule = q4::granule_bytes(D);
  static constexpr int kStage = 2 * kGranule;
  // (15 warps have 128 registers each, 7 have 255: one node 16 x 32760 rows 162 us and 209)
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

// Powers of two, exponents of floats (normal ones; exponent_bits: any, not negative).
constexpr int kQ4Top = 100;
__device__ __forceinline__ int exponent_bits(float x) { return static_cast<int>(__float_as_uint(x) >> 23); }
__device__ __forceinline__ int exponent_of(float x) { return exponent_bits(x) - 127; }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// The walk over a CTA's items by a whole warp.  Requests are looked at 32 at a time, one by
// each lane.
struct Q4Walk {
  long long off, left;
  int b, base, n32, len32, node32;  // of request base + lane
  bool left_out;
  __device__ __forceinline__ explicit Q4Walk(const Start& start)
      : off(start.off), left(start.left), b(start.b), base(-32), n32(0), len32(0), node32(0),
        left_out(start.left_out) {}
  // (as Walker::next)
  __device__ __forceinline__ bool next(const Batch& bt, int lane, int tile_keys, Item& it) {
    while (left > 0 && b < bt.B) {
      if (b - base >= 32) {
        base = b & ~31;
        n32 = len32 = node32 = 0;
        if (base + lane < bt.B) {
          request(bt, base + lane, n32, len32, left_out);
          node32 = bt.cu[base + lane];
        }
      }
      it.b = b;
      it.n = __shfl_sync(0xffffffffu, n32, b - base);
      it.len = __shfl_sync(0xffffffffu, len32, b - base);
      it.node0 = __shfl_sync(0xffffffffu, node32, b - base);
      it.tiles = (it.len + it.n + tile_keys - 1) / tile_keys;
      const long long u = units_of(bt, it.n, it.len);
      if (off >= u) {
        off -= u;
        ++b;
        continue;
      }
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
      if (member_item(bt, blockIdx.x, idx, blocks_of(bt, it.n), it.kvh, it.blk)) return true;
    }
    return false;
  }
};

// Zeros for a granule's scales: its rows are then zeros, whatever its codes.
template <int D>
__device__ __forceinline__ void q4_blank(uint8_t* granule) {
#pragma unroll 1
  for (int i = 0; i < D / 8; ++i) reinterpret_cast<uint4*>(granule + 16 * D)[i] = make_uint4(0u, 0u, 0u, 0u);
}

// The feeding warp: items to the queue, and each step's granules to the ring of the warp
// that takes it, a step a lane.  Step number g goes to warp g % W; the slots of a batch of
// steps are all different, so no lane waits for a copy that another is to make.
template <int W, int S, int D, typename Shared>
__device__ __forceinline__ void q4_feed(const Batch& bt, const q4::Pool& pool, Shared& sh, uint8_t* rings, int lane) {
  constexpr int TS = Shared::kTileSteps, SK = Shared::kStepKeys;
  constexpr int kBatch = W * S < 32 ? W * S : 32, kGranule = q4::granule_bytes(D);
  const Start start = locate(bt, team_of(bt, blockIdx.x));
  Q4Walk walk(start);
  uint32_t items = 0;
  int g = 0;
  const bool split = bt.table && bt.page_shift == 4;  // a step's granules lie in two pages
  const int page_mask = bt.table ? (1 << bt.page_shift) - 1 : INT_MAX;
  auto hand_on = [&](const Item& it, int end) {
    const int place = items % kQ4Queue;
    if (items >= kQ4Queue &&
        !__all_sync(0xffffffffu, mbar_wait(&sh.item_empty[place], (items / kQ4Queue - 1) & 1, 0x3F210)))
      return false;
    if (lane == 0) {
      sh.item[place] = Q4Item{it, g, end};
      mbar_arrive(&sh.item_full[place]);
    }
    ++items;
    return true;
  };
  Item it = {};
  while (walk.next(bt, lane, TS * SK, it)) {
    if (!hand_on(it, 0)) return;
    const int rows = it.len + it.n, steps = (it.t1 - it.t0) * TS;
    for (int i0 = 0; i0 < steps; i0 += kBatch) {
      const int i = i0 + lane;
      bool ok = true;
      if (lane < kBatch && i < steps) {
        const int row = (it.t0 * TS + i) * SK;
        const bool one = row < rows, two = SK > 16 && row + 16 < rows;  // (a tile's last steps may hold nothing)
        const int e0 = one ? table_entry(bt, it.b, row) : 0;
        const int e1 = split && two ? table_entry(bt, it.b, row + 16) : e0;
        const int p0 = checked_page(bt, it.b, e0), p1 = checked_page(bt, it.b, e1);
        const bool has0 = one && p0 < bt.n_pages, has1 = two && p1 < bt.n_pages;
        const uint32_t turn = static_cast<uint32_t>(g + i), w = turn % W, use = turn / W, s = use % S;
        if (use >= S) ok = mbar_wait(&sh.empty[w][s], (use / S - 1) & 1, 0x3F200) != 0;
        if (ok) {
          uint64_t* bar = &sh.full[w][s];
          uint8_t* dst = rings + (w * S + s) * (SK / 16 * kGranule);
          if (one != has0 || two != has1) {
            // rows of a page outside the pool: zeros for their scales, with whatever codes
            if (one != has0) q4_blank<D>(dst);
            if (two != has1) q4_blank<D>(dst + kGranule);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (copies come here again)
          }
          mbar_arrive_expect_tx(bar, (has0 + has1) * kGranule);
          if (has0)
            bulk_load(dst, q4::granule(pool, D, p0, it.kvh, row & page_mask), has1 && !split ? 2 * kGranule : kGranule, bar);
          if (has1 && split)
            bulk_load(dst + kGranule, q4::granule(pool, D, p1, it.kvh, (row + 16) & page_mask), kGranule, bar);
        }
      }
      if (!__all_sync(0xffffffffu, ok)) return;
    }
    g += steps;
  }
  hand_on(it, start.left_out ? 2 : 1);
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
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&sh.full[threadIdx.x][s], 1);
      mbar_init(&sh.empty[threadIdx.x][s], 1);
    }
  } else if (threadIdx.x == W * 32) {
    for (int i = 0; i < kQ4Queue; ++i) {
      mbar_init(&sh.item_full[i], 1);
      mbar_init(&sh.item_empty[i], W);
    }
    mbar_init(&sh.handed, W / 2);
    mbar_init(&sh.joined, (W + 1) / 2);
    mbar_init(&sh.read, W);
  }
  fence_mbar_init();
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (warp == W) {
    q4_feed<W, C::kStages, D>(bt, pool, sh, q4_smem + sizeof(typename C::Shared), lane);
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
  float c[NT][NB];        // a block's weights are held times this power of two
  uint32_t spoilt[NT];    // blocks with a NaN scale that the row sees
  bool have_anc = false;
  while (true) {
    if (!arrived(&sh.item_full[items % kQ4Queue], (items / kQ4Queue) & 1, 0x3F100)) return;
    const Q4Item& entry = sh.item[items % kQ4Queue];
    end = entry.end;
    if (end) break;
    const Item& it = entry.it;
    const int R = it.n * bt.group, row_lo = it.blk * RB, steps = it.t1 - it.t0;
    {
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
        m[nt] = -FLT_MAX;
        l[nt] = 0.f;
        spoilt[nt] = 0u;
#pragma unroll
        for (int b = 0; b < NB; ++b) c[nt][b] = power_of_two(kQ4Top);
#pragma unroll
        for (int e = 0; e < 4; ++e) ws[nt][e] = 0.f;
      }
      have_anc = false;
    }

    int i_step = warp - entry.g0 % W;
    for (i_step += i_step < 0 ? W : 0; i_step < steps; i_step += W) {
      if (!arrived(&sh.full[warp][stage], phase, 0x3F000 | warp)) return;
      const uint8_t* base = ring + stage * C::kStage;
      int row0 = (it.t0 + i_step) * kQ4Keys;
      const bool tail = row0 + kQ4Keys > it.len;
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
        uint32_t shown = 0xfu;  // which of the lane's keys a row sees
        if (tail) {
          // keys that are not there, or that only some rows see, may hold anything
          shown = 0u;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const int j0 = row0 + 4 * t - it.len, at = j0 >> 5;  // tree row of the first key, its word
            const uint32_t* words = reinterpret_cast<const uint32_t*>(&sh.sees[warp][nt * 8 + g]);
            const uint32_t w0 = at < 0 ? ~0u : at < kWords ? words[at] : 0u,
                           w1 = at + 1 < 0 ? ~0u : at + 1 < kWords ? words[at + 1] : 0u;
            const uint32_t vis = __funnelshift_r(w0, w1, j0 & 31);
            if (!(vis & 1u)) s[nt][0].x = -INFINITY;
            if (!(vis & 2u)) s[nt][0].y = -INFINITY;
            if (!(vis & 4u)) s[nt][1].x = -INFINITY;
            if (!(vis & 8u)) s[nt][1].y = -INFINITY;
            shown |= vis;
          }
        }
        uint32_t dv[NB * 2];  // [key][block] f16
#pragma unroll
        for (int i = 0; i < NB / 2; ++i) {
          const uint4 u = *reinterpret_cast<const uint4*>(base + 17 * D + t * (8 * NB) + i * 16);
          dv[4 * i] = u.x; dv[4 * i + 1] = u.y; dv[4 * i + 2] = u.z; dv[4 * i + 3] = u.w;
        }
        if (tail) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!((shown >> i) & 1u))
#pragma unroll
              for (int b = 0; b < NB / 2; ++b) dv[i * (NB / 2) + b] = 0u;
        }
        // The weights p and, by block, their products with the scales, rounded to f16.  They are
        // relative to the row's m and c as they stand, unless one would come near f16's end
        // (or a scale is NaN): then those of the rows that need it follow, and all is done again.
        float2 p[NT][2];
        float sum[NT];
        uint32_t w[NB][NT][2];
#pragma unroll 1
        for (bool again = false;; again = true) {
          bool grow = false;
          __half2 top = __float2half2_rn(0.f);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float2 x = fma2(s[nt][h], make_float2(sscale[nt], sscale[nt]), make_float2(-m[nt], -m[nt]));
              p[nt][h] = make_float2(fast_exp2(x.x), fast_exp2(x.y));
            }
            sum[nt] = (p[nt][0].x + p[nt][0].y) + (p[nt][1].x + p[nt][1].y);
            grow |= sum[nt] > 0x1p60f;  // (far from f32's end, for l too)
          }
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const __half* hv = reinterpret_cast<const __half*>(dv) + 2 * h * NB + b;
              const float2 d = make_float2(__half2float(hv[0]), __half2float(hv[NB]));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const float2 x = mul2(mul2(p[nt][h], make_float2(c[nt][b], c[nt][b])), d);
                w[b][nt][h] = MmaOp<__half>::pack(x.x, x.y);
                top = __hmax2_nan(top, __habs2(*reinterpret_cast<const __half2*>(&w[b][nt][h])));
              }
            }
          grow |= ((*reinterpret_cast<const uint32_t*>(&top) + 0x07ff07ffu) & 0x80008000u) != 0u;  // above 2^15, NaN
          if (again || !__any_sync(0xffffffffu, grow)) break;
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
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            // m follows where a score is more than 2^8 above it, by whole exponents (the weight
            // of a row's only key is exact)
            float mx = fmaxf(fmaxf(s[nt][0].x, s[nt][0].y), fmaxf(s[nt][1].x, s[nt][1].y)) * sscale[nt];
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float before = m[nt];
            int step = 0;
            if (mx > before + 8.f) {
              const float up = ceilf(mx - before);
              step = up < 300.f ? static_cast<int>(up) : 300;
              m[nt] = up < 300.f ? before + up : mx;
            }
            const float alpha = fast_exp2(before - m[nt]);
            l[nt] *= alpha;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float2 x = fma2(s[nt][h], make_float2(sscale[nt], sscale[nt]), make_float2(-m[nt], -m[nt]));
              p[nt][h] = make_float2(fast_exp2(x.x), fast_exp2(x.y));
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              // the block's largest product, and the power of two that brings it under 1;
              // what is there already keeps its place, or goes down with it
              float most = 0.f;
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const __half* hv = reinterpret_cast<const __half*>(dv) + 2 * h * NB + b;
                const float2 x = mul2(p[nt][h], make_float2(__half2float(hv[0]), __half2float(hv[NB])));
                most = fmaxf(most, fmaxf(fabsf(x.x), fabsf(x.y)));
              }
              most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
              most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
              const int e = exponent_of(c[nt][b]), to = max(min(min(e + step, 126 - exponent_bits(most)), kQ4Top), -kQ4Top);
              c[nt][b] = power_of_two(to);
              const float f = alpha * (to - e < -126 ? 0.f : power_of_two(to - e));
              const float a0 = __shfl_sync(0xffffffffu, f, 8 * t), a1 = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
              for (int i = 2 * b; i < 2 * b + 2; ++i) {
                o[i][nt][0] *= a0;
                o[i][nt][1] *= a1;
                o[i][nt][2] *= a0;
                o[i][nt][3] *= a1;
              }
              if (g == b) {
                ws[nt][0] *= a0;
                ws[nt][1] *= a1;
              }
            }
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) l[nt] += sum[nt];
        // ---- output -----------------------------------------------------------------
        const uint8_t* vb = base + 8 * D + (g & 3) * 64 + t * 16;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint4 u = *reinterpret_cast<const uint4*>(vb + b * 256);
          const uint32_t lo = __byte_perm(u.x, u.y, sel), hi = __byte_perm(u.z, u.w, sel);
          const uint32_t lo8 = lo >> 8, hi8 = hi >> 8;
          const uint32_t a0[4] = {lo & 0x000f000fu, lo & 0x00f000f0u, hi & 0x000f000fu, hi & 0x00f000f0u};
          const uint32_t a1[4] = {lo8 & 0x000f000fu, lo8 & 0x00f000f0u, hi8 & 0x000f000fu, hi8 & 0x00f000f0u};
          const uint32_t one = g == b ? 0x3c003c00u : 0u;
          const uint32_t ones[4] = {one, one, one, one};  // (rows 8 to 15 are not used)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_f16(o[2 * b][nt], a0, w[b][nt][0], w[b][nt][1], o[2 * b][nt]);
            mma_f16(o[2 * b + 1][nt], a1, w[b][nt][0], w[b][nt][1], o[2 * b + 1][nt]);
            mma_f16(ws[nt], ones, w[b][nt][0], w[b][nt][1], ws[nt]);
          }
        }
      }
      // the stage is read
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.empty[warp][stage]);
      if (++stage == C::kStages) {
        stage = 0;
        phase ^= 1;
      }
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
        const float back = power_of_two(-exponent_of(c[nt][b]));
        const float b0 = __shfl_sync(0xffffffffu, back, 8 * t), b1 = __shfl_sync(0xffffffffu, back, 8 * t + 4);
        float w0 = -8.f * __shfl_sync(0xffffffffu, ws[nt][0], b * 4 + t) * b0;
        float w1 = -8.f * __shfl_sync(0xffffffffu, ws[nt][1], b * 4 + t) * b1;
        if (seen_nan) {
          if (__shfl_sync(0xffffffffu, spoilt[nt], 8 * t) >> b & 1u) w0 = __uint_as_float(0x7fffffffu);
          if (__shfl_sync(0xffffffffu, spoilt[nt], 8 * t + 4) >> b & 1u) w1 = __uint_as_float(0x7fffffffu);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float* x = o[2 * b + i][nt];
          x[0] = fmaf(x[0], 16777216.f * b0, w0);
          x[1] = fmaf(x[1], 16777216.f * b1, w1);
          x[2] = fmaf(x[2], 1048576.f * b0, w0);
          x[3] = fmaf(x[3], 1048576.f * b1, w1);
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
        const float now = fmaxf(m[nt], m2);
        const float a = fast_exp2(m[nt] - now), a2 = fast_exp2(m2 - now);
        m[nt] = now;
        l[nt] = l[nt] * a + l2 * a2;
        const float a0 = __shfl_sync(0xffffffffu, a, 8 * t), a1 = __shfl_sync(0xffffffffu, a, 8 * t + 4);
        const float c0 = __shfl_sync(0xffffffffu, a2, 8 * t), c1 = __shfl_sync(0xffffffffu, a2, 8 * t + 4);
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
    const int slot = part_slot(it, blockIdx.x);
    const int live = min(RB, R - row_lo);
    // warps that had no step have m = -FLT_MAX and l = 0
    for (int i = threadIdx.x; i < live * (D / 8); i += W * 32) {
      const int r = i / (D / 8), d = (i - r * (D / 8)) * 8;
      float M = -FLT_MAX;
#pragma unroll
      for (int w = 0; w < H; ++w) M = fmaxf(M, merge_ml[(w * RB + r) * 2]);
      float L = 0.f, x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 0.f;
#pragma unroll 4
      for (int w = 0; w < H; ++w) {
        const float f = fast_exp2(merge_ml[(w * RB + r) * 2] - M);
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
        const float f = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= f;
        paged::store8(out + row * D + d, x);
        if (lse && d == 0) lse[row] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
      }
    }
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(&sh.read);
      mbar_arrive(&sh.item_empty[items % kQ4Queue]);
    }
    ++items;
  }
  zero_unwritten<T, D>(bt, end == 2, out, lse, warp, W);
}

}  // namespace tree
}  // namespace b2a
