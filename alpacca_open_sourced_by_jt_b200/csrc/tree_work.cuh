// Work division of the tree attention over a cache (tree_decode.cu,
// tree_wide.cu): what every kernel of it shares.
//
// The grid is teams of CTAs that read the same cache rows side by side:
// either a CTA per KV head (a page holds all heads of a token behind one
// another), for one block of query rows per request, or a CTA per block of
// query rows of one KV head, so that the blocks' second and later reads of a
// tile hit L2.  What a team works on is a list of items, each as long as its
// request's key tiles.  Lengths live on the device, so the division is made
// there: the list's tiles are numbered through and team i takes tiles
// [i * chunk, (i + 1) * chunk), chunk = ceil(total / teams) or a least number
// of tiles where that is more.  Every CTA so streams the same number of tiles
// whatever the lengths, and at most one item is cut at each boundary.  An item
// wholly inside one range is finished there; the parts of a cut item go to the
// workspace and tree_merge_kernel joins them.  CTA c writes at most two parts:
// slot 2c for an item that began before its range and ends in it, slot 2c + 1
// for one that goes on past its range.
#pragma once

#include <type_traits>

#include "b2a_common.cuh"

namespace b2a {
namespace tree {

constexpr int kMaxNodes = B2A_TREE_MAX_NODES;  // nodes of one request's tree
constexpr int kWords = kMaxNodes / 32;         // words of an ancestor mask
static_assert(kWords == 4, "add_special takes a mask as four words");
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

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

// The requests, as the kernels see them.
struct Batch {
  const int* lens;     // cached rows before the tree
  const int* cu;       // [B + 1] first node of each request
  const int* parents;  // [n_tok] or null: a chain
  const int* table;    // [B][table_stride] pages, or null: request b's block is page b
  long long table_stride;
  int B, n_tok, max_nodes, max_len, n_pages, page_shift;
  int H, KV, group;
  int rows_per_block;  // query rows of an item
  int tile;            // keys per tile
  int by_item;         // CTAs take whole items (no parts)
  int min_units;       // least tiles of a range
  int teams;           // ranges the list is cut into
  int m_heads;         // KV heads side by side in a team: KV or 1
  int m_blks;          // blocks of query rows side by side
};

// Nodes and cache rows of request b; false for a request that is left out (no
// nodes and no rows): its numbers are out of bounds (recorded), or its last row
// has no page, -1 in the table, where the plan could not serve it (no error).
// Where it is known that no request is left out (Start), `check` false spares
// the look-up in the table.
__device__ __forceinline__ bool request(const Batch& bt, int b, int& n, int& len,
                                        bool check = true) {
  const int c0 = bt.cu[b], c1 = bt.cu[b + 1];
  len = bt.lens[b];
  n = c1 - c0;
  if (n < 0 || n > bt.max_nodes || c0 < 0 || c1 > bt.n_tok || len < 0 ||
      len > bt.max_len - n) {
    set_dev_error(B2A_ERR_POSITION, b);
  } else if (!check || n == 0 || !bt.table ||
             __ldg(bt.table + b * bt.table_stride + ((len + n - 1) >> bt.page_shift)) != -1) {
    return true;
  }
  n = 0;
  len = 0;
  return false;
}

__device__ __forceinline__ int blocks_of(const Batch& bt, int n) {
  return (n * bt.group + bt.rows_per_block - 1) / bt.rows_per_block;
}

__device__ __forceinline__ long long units_of(const Batch& bt, int n, int len) {
  if (n == 0) return 0;
  const long long items = static_cast<long long>(bt.KV / bt.m_heads) *
                          ((blocks_of(bt, n) + bt.m_blks - 1) / bt.m_blks);
  return bt.by_item ? items : items * ((len + n + bt.tile - 1) / bt.tile);
}

// Start of a team's range.
struct Start {
  long long off;    // units into request b
  long long left;   // units of this team
  long long chunk;  // units per team
  int b;
  bool left_out;  // some request is left out
};

// Warp-collective: the range of one team.
__device__ __forceinline__ Start locate(const Batch& bt, int team) {
  const int lane = threadIdx.x & 31;
  long long total = 0;
  bool out = false;
  for (int b = lane; b < bt.B; b += 32) {
    int n, len;
    out |= !request(bt, b, n, len);
    total += units_of(bt, n, len);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  Start s;
  s.left_out = __any_sync(0xffffffffu, out) != 0;
  s.chunk = (total + bt.teams - 1) / bt.teams;
  if (s.chunk < bt.min_units) s.chunk = bt.min_units;
  const long long first = s.chunk * team;
  s.left = total - first;
  if (s.left > s.chunk) s.left = s.chunk;
  s.b = bt.B;
  s.off = 0;
  if (s.left <= 0) {
    s.left = 0;
    return s;
  }
  long long run = 0;
  for (int b0 = 0; b0 < bt.B; b0 += 32) {
    int n = 0, len = 0;
    if (b0 + lane < bt.B) request(bt, b0 + lane, n, len, s.left_out);
    const long long u = units_of(bt, n, len);
    long long inc = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    const long long lo = run + inc - u;
    const unsigned hit = __ballot_sync(0xffffffffu, first >= lo && first < lo + u);
    if (hit) {
      const int src = __ffs(hit) - 1;
      s.b = b0 + src;
      s.off = first - __shfl_sync(0xffffffffu, lo, src);
      return s;
    }
    run += __shfl_sync(0xffffffffu, inc, 31);
  }
  s.left = 0;  // not reached
  return s;
}

struct Item {
  int b, kvh, blk;
  int n, len;     // the request's nodes and cached rows
  int t0, t1;     // this CTA's key tiles of the item
  int tiles;      // the item's key tiles
  int node0;      // row of the request's node 0 in q and out
};

// KV head and block of a team's item `idx` of a request with `blks` blocks,
// for CTA c of the grid; false if this CTA has no block in it.
__device__ __forceinline__ bool member_item(const Batch& bt, int c, int idx, int blks, int& kvh,
                                            int& blk) {
  const int member = c % (bt.m_heads * bt.m_blks);
  const int hm = member % bt.m_heads, bm = member / bt.m_heads;
  const int rounds = (blks + bt.m_blks - 1) / bt.m_blks;
  const int hl = idx / rounds;
  kvh = bt.m_heads > 1 ? hm : hl;
  blk = (idx - hl * rounds) * bt.m_blks + bm;
  return blk < blks;
}

__device__ __forceinline__ int team_of(const Batch& bt, int c) {
  return c / (bt.m_heads * bt.m_blks);
}

// Walks the items of a CTA's range; every role of a CTA walks the same ones.
struct Walker {
  long long off, left;
  int b, n, len;
  bool check;
  __device__ __forceinline__ void start(const Batch& bt, const Start& s) {
    off = s.off;
    left = s.left;
    b = s.b;
    check = s.left_out;
    if (left > 0) request(bt, b, n, len, check);
  }
  __device__ __forceinline__ bool next(const Batch& bt, Item& it) {
    while (left > 0) {
      const long long u = units_of(bt, n, len);
      if (off >= u) {
        off -= u;
        if (++b >= bt.B) return false;
        request(bt, b, n, len, check);
        continue;
      }
      it.b = b;
      it.n = n;
      it.len = len;
      it.tiles = (len + n + bt.tile - 1) / bt.tile;
      const int per = bt.by_item ? 1 : it.tiles;
      const int idx = static_cast<int>(off / per);
      const int at = static_cast<int>(off - static_cast<long long>(idx) * per);
      int take = per - at;
      if (take > left) take = static_cast<int>(left);
      it.t0 = bt.by_item ? 0 : at;
      it.t1 = bt.by_item ? it.tiles : at + take;
      it.node0 = bt.cu[b];
      off += take;
      left -= take;
      if (member_item(bt, blockIdx.x, idx, blocks_of(bt, n), it.kvh, it.blk)) return true;
    }
    return false;
  }
};

// Rows [lo, hi) of out become zeros, their lse -inf, by thread i0 of step.
template <typename T, int D>
__device__ __forceinline__ void zero_rows(T* out, float* lse, long long lo, long long hi,
                                          long long i0, long long step) {
  constexpr int kGroups = D * sizeof(T) / 16;
  for (long long i = lo * kGroups + i0; i < hi * kGroups; i += step)
    reinterpret_cast<uint4*>(out)[i] = make_uint4(0u, 0u, 0u, 0u);
  if (lse)
    for (long long i = lo + i0; i < hi; i += step) lse[i] = -INFINITY;
}

// The rows that no item writes become zeros: those past the last node (the
// padding of a captured step) and those of requests left out.  Called by warp
// `warp` of `warps` of every CTA.
template <typename T, int D>
__device__ __forceinline__ void zero_unwritten(const Batch& bt, bool left_out, T* out, float* lse,
                                               int warp, int warps) {
  const int lane = threadIdx.x & 31;
  const long long i0 = (static_cast<long long>(blockIdx.x) * warps + warp) * 32 + lane;
  const long long step = static_cast<long long>(gridDim.x) * warps * 32;
  zero_rows<T, D>(out, lse, static_cast<long long>(max(bt.cu[bt.B], 0)) * bt.H,
                  static_cast<long long>(bt.n_tok) * bt.H, i0, step);
  if (!left_out) return;
  for (int b0 = 0; b0 < bt.B; b0 += 32) {
    int n, len;
    unsigned out_here = __ballot_sync(0xffffffffu, b0 + lane < bt.B && !request(bt, b0 + lane, n, len));
    for (; out_here; out_here &= out_here - 1) {
      const int b = b0 + __ffs(out_here) - 1;
      zero_rows<T, D>(out, lse, static_cast<long long>(max(bt.cu[b], 0)) * bt.H,
                      static_cast<long long>(min(bt.cu[b + 1], bt.n_tok)) * bt.H, i0, step);
    }
  }
}

// Ancestor masks of a request's nodes (bit j of node i's: i sees node j),
// written by threads tid of nt to anc[node][kWords]; par holds the parents
// (synchronise before and after).  A parent that is not an earlier node is
// recorded and ends the path.
__device__ __forceinline__ void ancestor_masks(const int* par, bool chain, int n,
                                               uint32_t (*anc)[kWords], int tid, int nt,
                                               int where) {
  for (int i = tid; i < n; i += nt) {
    uint32_t m[kWords];
#pragma unroll
    for (int w = 0; w < kWords; ++w) m[w] = 0u;
    if (chain) {
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        const int k = i + 1 - w * 32;  // bits of this word
        m[w] = k >= 32 ? 0xffffffffu : (k > 0 ? (1u << k) - 1u : 0u);
      }
    } else {
      int p = i;
      while (true) {
#pragma unroll
        for (int w = 0; w < kWords; ++w)
          if ((p >> 5) == w) m[w] |= 1u << (p & 31);
        const int up = par[p];
        if (up < 0 || up >= p) {
          if (up != -1) set_dev_error(B2A_ERR_POSITION, where);
          break;
        }
        p = up;
      }
    }
#pragma unroll
    for (int w = 0; w < kWords; ++w) anc[i][w] = m[w];
  }
}

// Page (outer tensor-map coordinate) that holds cache row `row` of request b,
// as the table has it.  The check is apart from the load, so that a producer
// can look a page up one tile ahead without waiting for it.
__device__ __forceinline__ int table_entry(const Batch& bt, int b, int row) {
  return bt.table ? __ldg(bt.table + b * bt.table_stride + (row >> bt.page_shift)) : b;
}

// A page outside the pool is recorded and answered with n_pages, which TMA
// reads as zeros.
__device__ __forceinline__ int checked_page(const Batch& bt, int b, int pg) {
  if (pg >= 0 && pg < bt.n_pages) return pg;
  set_dev_error(B2A_ERR_POSITION, b);
  return bt.n_pages;
}

// Infinities and NaN in the V rows of nodes.  A hidden row has weight 0 in the
// product P.V, but 0 * inf is NaN: where a request has several nodes, the kernels
// take such elements out of a tile's tree rows (clear_special), and an item that
// had some adds them at its end to the rows whose node sees them (add_special), as
// the sum over the visible rows alone has them.

// Clears the infinities and NaN among 16 bytes of T; true if there were any.
template <typename T>
__device__ __forceinline__ bool clear_special(uint4& u) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&u);
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t keep = 0xffffffffu;
    if constexpr (sizeof(T) == 4) {
      if ((w[i] & 0x7f800000u) == 0x7f800000u) keep = 0u;
    } else {
      constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
      if ((w[i] & kExp) == kExp) keep &= 0xffff0000u;
      if ((w[i] >> 16 & kExp) == kExp) keep &= 0x0000ffffu;
    }
    any |= keep != 0xffffffffu;
    w[i] &= keep;
  }
  return any;
}

// Adds the infinities and NaN in columns d0 .. d0 + nd - 1 of a node's V rows to
// dst (a row of out, or of a part): tree rows [lo, hi) among the bits of anc.
template <typename T, typename TO>
__device__ __noinline__ void add_special(const Batch& bt, const T* v, long long page_stride, int b,
                                         int kvh, int len, int lo, int hi, uint4 anc, TO* dst,
                                         int D, int d0, int nd) {
  for (int j = lo; j < hi; ++j) {
    const uint32_t word = j < 32 ? anc.x : j < 64 ? anc.y : j < 96 ? anc.z : anc.w;
    if (!((word >> (j & 31)) & 1u)) continue;
    const int row = len + j;
    const int pg = checked_page(bt, b, table_entry(bt, b, row));
    if (pg >= bt.n_pages) continue;
    const int in_page = bt.table ? row & ((1 << bt.page_shift) - 1) : row;
    const T* src = v + pg * page_stride + (static_cast<long long>(in_page) * bt.KV + kvh) * D + d0;
    for (int e = 0; e < nd; ++e) {
      const float x = ld_elem(src + e);
      if (!(fabsf(x) < INFINITY)) st_elem(dst + e, ld_elem(dst + e) + x);
    }
  }
}

// Part slot of an item in CTA c's range, or -1 if the item is whole in it.
__device__ __forceinline__ int part_slot(const Item& it, int c) {
  if (it.t0 == 0 && it.t1 == it.tiles) return -1;
  return 2 * c + (it.t1 < it.tiles ? 1 : 0);
}

}  // namespace tree
}  // namespace b2a
